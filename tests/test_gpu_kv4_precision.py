"""How exact the attention over the 4-bit cache is, where a bound relative to the largest values would not show it: 16-bit outputs
are the roundings of numbers within f32's errors of float64's, f32 rows of values of any size relative to those."""
import numpy as np
import pytest
import torch

from ops_reference import TYPES, attention, stored
from test_gpu_kv4 import cache, f64, ints, rows

pytestmark = pytest.mark.gpu


def is_rounding(got, want, off, t):
    """Whether each of got (values of type t) is the rounding of a number within off of want."""
    lo, hi = (torch.from_numpy(x).to(TYPES[t]).double().numpy() for x in (want - 1.01 * off, want + 1.01 * off))
    return (lo <= got) & (got <= hi)


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("dim,kv,group,tokens", [(64, 1, 2, 1), (128, 2, 4, 5), (256, 1, 3, 7), (64, 16, 16, 33), (128, 8, 4, 160)])
def test_outputs_of_16_bits_are_rounded_once(gpu, dim, kv, group, tokens, t):
    """Small scores (sum |q k| scale below 1.2), few positions: the scores are off by at most (dim + 8) 2^-24 1.2, weights by twice
    that (an exponential's own 2^-22 too), a weight times its scale in two f16 parts by 2^-22 and 2^-25 absolute: 2^-20 together; sums of n terms by n 2^-24 each, and the joins of
    records of at most 16 steps, all relative to the mean |v|."""
    n = 33 if tokens == 1 else 40 + tokens
    c = cache(1, kv, dim, n + 1000 * (tokens > 100))
    k, v = rows(1, (1, n, kv, dim)), rows(2, (1, n, kv, dim))
    c.append(k, v, ints(0))
    q = (rows(3, (1, tokens, kv * group, dim)) * (0.5 * dim ** -0.5)).to(TYPES[t])
    print(f"case rounded once dim {dim} tokens {tokens} {t}", flush=True)
    got = f64(c.attend(q, ints(n - tokens)))[0]
    kk, vv, qq = stored(f64(k))[0], stored(f64(v))[0], f64(q)[0]
    last = n - tokens + np.arange(tokens)
    for h in range(kv * group):
        want, size = attention(qq[:, h], kk[:, h // group], vv[:, h // group], last, dim ** -0.5)
        mean, _ = attention(qq[:, h], kk[:, h // group], np.abs(vv[:, h // group]), last, dim ** -0.5)
        assert size.max() < 1.2
        off = mean * (2 * (dim + 8) * 2.0 ** -24 * size[:, None] + 2 * (n + 16) * 2.0 ** -24 + 2.0 ** -20)
        ok = is_rounding(got[:, h], want, off, t)
        assert ok.all(), (h, (~ok).sum(), ok.size, np.abs(got[:, h] - want).max())
    c.close()


@pytest.mark.parametrize("t", ["f16", "bf16"])
@pytest.mark.parametrize("dim,kv,group,tokens,n", [(64, 2, 1, 1, 700), (128, 2, 4, 9, 5000), (256, 1, 3, 5, 1300), (128, 8, 8, 160, 2100), (64, 8, 4, 64, 33000)])
def test_16_bit_rows_are_the_f32_rows_rounded(gpu, dim, kv, group, tokens, n, t):
    """Queries of 16 bits are exact in the f16 part that f32 queries have too, and every step after that is the same: the outputs are
    the roundings of the f32 ones, bit for bit. Also keys with a few channels much larger than the rest."""
    c = cache(1, kv, dim, n)
    for spread in (0.5, 1.5):
        k, v = rows(7, (1, n, kv, dim), spread=spread), rows(8, (1, n, kv, dim))
        c.append(k, v, ints(0))
        q = (rows(9, (1, tokens, kv * group, dim)) * 4).to(TYPES[t])
        print(f"case rounded f32 dim {dim} tokens {tokens} {t} spread {spread}", flush=True)
        for first in (0, n - tokens):
            got, want = c.attend(q, ints(first)), c.attend(q.float(), ints(first))
            assert torch.isfinite(got).all() and (got == want.to(TYPES[t])).all()
    c.close()


def whole_scores(dim, kv, group, n, tokens, t, seed):
    """Keys in blocks of scale 1 and queries of whole numbers, and a scale: every product and sum of a score is a whole number below
    2^24, so that its order does not matter, over a range of some 10 after the scale. The products are up to 200 times what their
    sums come to."""
    g = torch.Generator().manual_seed(seed)
    k = torch.randint(-7, 8, (1, n, kv, dim), generator=g).float()
    k[..., ::32] = -8.0
    q = torch.randint(-250, 251, (1, tokens, kv * group, dim), generator=g).float()
    return k.cuda(), q.to(TYPES[t]).cuda(), 2.0 ** -12 * (64 / dim) ** 0.5


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("magnitude", [1e-1, 3e-2, 1e-2, 1e-3, 1e-4, 1e-5, 1e-6, "mixed", "one"])
@pytest.mark.parametrize("dim,tokens,group", [(64, 1, 2), (128, 9, 4), (256, 3, 1), (128, 300, 8)])
def test_small_values_keep_their_bits(gpu, dim, tokens, group, magnitude, t):
    """Values of a size, of another size in every block of 32, and one position a thousand times the others. With the largest value
    scale of a span's block raised to 2^-5 at least and the largest weight 8, a weight times its scale is off by 2^-25 and 2^-22 of
    itself, at a code of at most 8, over 64 positions whose weights sum to 8 or more: 2^-17 of the block's largest value. Whole scores,
    and f32 sums of spans (64 terms) and their folds (some 40), relative to the mean |v|."""
    kv, n = (2, 1000) if tokens > 100 else (1, 1000)
    k, q, scale = whole_scores(dim, kv, group, n, tokens, t, dim + tokens)
    v = rows(52, (1, n, kv, dim))
    if magnitude == "mixed":
        v = v * (10.0 ** -(torch.arange(dim // 32) * 5 % 7)).repeat_interleave(32).cuda()
    elif magnitude == "one":
        v *= 1e-4
        v[:, 777] *= 1e3
    else:
        v *= magnitude
    c = cache(1, kv, dim, n + 2000 * (tokens > 100))
    c.append(k, v, ints(0))
    print(f"case small values {magnitude} dim {dim} tokens {tokens} {t}", flush=True)
    got = f64(c.attend(q, ints(n - tokens), scale=scale))[0]
    kk, vv, qq = stored(f64(k))[0], stored(f64(v))[0], f64(q)[0]
    last = n - tokens + np.arange(tokens)
    worst = 0.0
    for h in range(kv * group):
        x, y = kk[:, h // group], vv[:, h // group]
        want, _ = attention(qq[:, h], x, y, last, scale)
        mean, _ = attention(qq[:, h], x, np.abs(y), last, scale)
        top = np.abs(x @ qq[:, h].T).max() * scale
        assert top < 20
        big = np.repeat(np.abs(y).reshape(n, -1, 32).max((0, 2)), 32)
        off = mean * (4 * top * 2.0 ** -22 + 2 * 128 * 2.0 ** -24 + 2.0 ** -20) + big * 2.0 ** -17
        ok = is_rounding(got[:, h], want, off, t)
        assert ok.all(), (h, (~ok).sum(), ok.size, (np.abs(got[:, h] - want) / off).max())
        worst = max(worst, (np.abs(got[:, h] - want) / off).max())
    print(f"worst error / bound {worst:.3f}", flush=True)
    c.close()


@pytest.mark.parametrize("t", ["f32", "f16"])
@pytest.mark.parametrize("dim,kv,group,tokens", [(64, 2, 4, 40), (128, 8, 4, 300), (256, 1, 2, 70)])
def test_small_values_have_the_same_bits_in_every_batch(gpu, dim, kv, group, tokens, t):
    """Rows of one tile that see, in the same span, small values alone and a large one among them; blocks of either kind side by side."""
    n = 700
    c = cache(1, kv, dim, n)
    k, v = rows(21, (1, n, kv, dim)), rows(22, (1, n, kv, dim)) * 1e-4
    for p in (n - tokens + 5, n - 30, n - 3):
        v[:, p, :, 32:64] *= 1e4
    v[..., :16] *= 0.01
    c.append(k, v, ints(0))
    q = rows(23, (1, tokens, kv * group, dim)).to(TYPES[t])
    print(f"case small bits dim {dim} {t}", flush=True)
    got = c.attend(q, ints(n - tokens))
    assert torch.isfinite(got).all() and (got != 0).any()
    for m in (1, 3, 16):
        for j in (0, 4, 5, 6, tokens - 31, tokens - 29, tokens - m):
            m = min(m, tokens - j)
            assert (c.attend(q[:, j:j + m], ints(n - tokens + j)) == got[:, j:j + m]).all(), (m, j)
    c.close()
