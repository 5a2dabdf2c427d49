"""How exact the attention over the 4-bit cache is, where a bound relative to the largest values would not show it: 16-bit outputs
are the roundings of numbers within f32's errors of float64's."""
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
