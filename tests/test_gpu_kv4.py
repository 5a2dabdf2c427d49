"""The 4-bit KV cache and the attention over it (zerollm_amd.ops.KVCacheQ4) against plain float64."""
import numpy as np
import pytest
import torch

from ops_reference import TYPES, attention, attention_bound, half_step, quantise, stored
from oracle import oracle as O

pytestmark = pytest.mark.gpu


def cache(*a):
    from zerollm_amd.ops import KVCacheQ4
    return KVCacheQ4(*a)


def rows(seed, shape, t="f32", layout="token", spread=0.5):
    """[sequence, token, head, dim] values with a few large channels, on the GPU, in a memory layout of its own."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g) * torch.exp(spread * torch.randn(shape[2:], generator=g))
    x = x.to(TYPES[t])
    if layout == "head":    # [sequence, head, token, dim] seen as [sequence, token, head, dim]
        return x.transpose(1, 2).contiguous().cuda().transpose(1, 2)
    if layout == "padded":  # rows that start at odd values of a wider buffer
        s = list(shape)
        s[3] += 3
        w = torch.full(s, float("nan"), dtype=TYPES[t], device="cuda")
        w[..., 1:-2] = x.cuda()
        return w[..., 1:-2]
    return x.cuda()


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def f64(x):
    return x.double().cpu().numpy()


def read(c, pos, n_tok, slot=None, t="f32"):
    shape = (len(pos), n_tok, c.n_head_kv, c.head_dim)
    k, v = (torch.zeros(shape, dtype=TYPES[t], device="cuda") for _ in range(2))
    c.read(k, v, ints(*pos), slot=None if slot is None else ints(*slot))
    return f64(k), f64(v)


@pytest.mark.parametrize("layout", ["token", "head", "padded"])
@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,heads", [(64, 3), (128, 2), (256, 1)])
def test_append_then_read_is_the_q4_0_of_the_values(gpu, dim, heads, t, layout):
    """Windows of every phase against the 32-position records, with tokens around them that must stay."""
    n = 97
    c = cache(1, heads, dim, 150)
    k, v = rows(1, (1, n, heads, dim), t, layout), rows(2, (1, n, heads, dim), t, layout)
    k[0, 5, 0, :32] = 0.0
    k[0, 6, 0, 3], k[0, 6, 0, 9] = 8.0, -8.0  # two of the largest magnitude: the first gives the sign
    v[0, 7, 0, 20], v[0, 7, 0, 21] = -9.0, 9.0
    want_k, want_v = stored(f64(k)), stored(f64(v))
    at = 0
    for m in (1, 3, 27, 1, 1, 32, 31, 1):
        print(f"case append dim {dim} {t} {layout} at {at} + {m}", flush=True)
        c.append(k[:, at:at + m], v[:, at:at + m], ints(at))
        at += m
        got_k, got_v = read(c, [0], at)
        assert (got_k == want_k[:, :at]).all() and (got_v == want_v[:, :at]).all()
    # positions in the middle again, other values: their neighbours stay
    k2, v2 = rows(3, (1, 5, heads, dim), t, layout), rows(4, (1, 5, heads, dim), t, layout)
    c.append(k2, v2, ints(30))
    want_k[:, 30:35], want_v[:, 30:35] = stored(f64(k2)), stored(f64(v2))
    got_k, got_v = read(c, [0], n)
    assert (got_k == want_k).all() and (got_v == want_v).all()
    got_k, got_v = read(c, [0], n, t="bf16")
    for got, want in ((got_k, want_k), (got_v, want_v)):
        assert (np.abs(got - want) <= half_step(torch.bfloat16) * np.abs(want)).all()
    c.close()


def test_codes_are_the_oracles(gpu):
    """d and codes against the Q4_0 blocks of the oracle's quantiser, recovered from what it writes."""
    c = cache(1, 1, 64, 64)
    k = rows(9, (1, 40, 1, 64))
    c.append(k, k, ints(0))
    want = O.dequant(2, O.quantize_q4_0(k.cpu().numpy().reshape(-1)), 40, 64)
    got, got_v = read(c, [0], 40)
    assert (got[0, :, 0] == want).all() and (got_v[0, :, 0] == want).all()
    c.close()


def test_sequences_counts_slots_and_places_that_do_not_exist(gpu):
    dim, heads, cap = 128, 2, 70
    c = cache(4, heads, dim, cap)
    k, v = rows(5, (5, 40, heads, dim)), rows(6, (5, 40, heads, dim))
    # slot 1 twice (the later sequence wins where they meet), a slot that does not exist, positions before 0 and past the end
    pos, count, slot = [3, 20, -7, 60, 0], [40, 30, 40, 40, 99], [1, 1, 3, 0, 4]
    c.append(k, v, ints(*pos), ints(*count), ints(*slot))
    want = [np.zeros((2, cap, heads, dim)) for _ in range(4)]
    kv = np.stack([stored(f64(k)), stored(f64(v))])
    for s in range(4):
        for j in range(min(40, count[s])):
            if 0 <= pos[s] + j < cap:
                want[slot[s]][:, pos[s] + j] = kv[:, s, j]
    for s in range(4):
        got = np.stack(read(c, [0], cap, [s]))
        assert (got[:, 0] == want[s]).all(), s
    got = np.stack(read(c, [68, -1, 0], 4, [0, 0, 7]))
    assert np.isnan(got[:, 0, 2:]).all() and np.isfinite(got[:, 0, :2]).all()
    assert np.isnan(got[:, 1, 0]).all() and (got[:, 1, 1:] == want[0][:, :3]).all() and np.isnan(got[:, 2]).all()
    # rows behind a count are left as they were
    ko, vo = torch.full((4, 9, heads, dim), 7.0, device="cuda"), torch.full((4, 9, heads, dim), 7.0, device="cuda")
    c.read(ko, vo, ints(0, 0, 0, 0), ints(9, 2, 0, -5))
    assert (ko[0] != 7).all() and (ko[1, 2:] == 7).all() and (ko[2:] == 7).all() and (vo[2:] == 7).all()
    # nothing to do
    c.append(k[:0], v[:0], ints())
    c.append(k[:, :0], v[:, :0], ints(*pos))
    c.close()


def test_values_that_do_not_fit_read_as_nan(gpu):
    c = cache(1, 1, 64, 64)
    k = torch.ones((1, 4, 1, 64), device="cuda")
    k[0, 0, 0, 3], k[0, 1, 0, 40], k[0, 2, 0, 0], k[0, 3, 0, 0] = float("inf"), float("nan"), 65505.0, 65504.0
    c.append(k, k, ints(0))
    for got in read(c, [0], 4):
        bad = np.isnan(got[0, :, 0])
        assert bad[0, :32].all() and not bad[0, 32:].any() and bad[1, 32:].all() and not bad[1, :32].any()
        assert bad[2, :32].all() and not bad[3].any() and got[0, 3, 0, 0] == 65504.0
    c.close()


def check(c, q, pos, count=None, slot=None, k=None, v=None, scale=None, t="f32", **kw):
    """attend() against float64 over what the cache holds. k, v: [slot, position, head, dim] float64 values it stands for."""
    S, T, H, D = q.shape
    got = c.attend(q, ints(*pos), count=None if count is None else ints(*count), slot=None if slot is None else ints(*slot),
                   scale=scale, **kw)
    g = f64(got)
    q = f64(q)
    G = H // c.n_head_kv
    worst = 0.0
    for s in range(S):
        n = T if count is None else max(0, min(T, count[s]))
        sl = s if slot is None else slot[s]
        for h in range(H):
            last = pos[s] + np.arange(n)
            want, size = attention(q[s, :n, h], k[sl, :, h // G], v[sl, :, h // G], last, scale or D ** -0.5)
            lim = attention_bound(size, D, np.abs(v[sl, :max(1, last.max(initial=0) + 1), h // G]).max(), want, TYPES[t])
            err = np.abs(g[s, :n, h] - want)
            assert (err <= lim).all(), (s, h, np.argwhere(err > lim)[:3], err.max(), lim.min())
            worst = max(worst, (err / lim).max(initial=0))
    return got, worst


LENGTHS = [1, 2, 31, 32, 33, 63, 64, 65, 255, 256, 257, 511, 512, 513, 1023, 1024, 1025, 2047, 2048, 2049, 4100]


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,kv,group", [(64, 2, 1), (128, 1, 4), (128, 2, 7), (256, 1, 3)])
def test_single_tokens_of_every_length(gpu, dim, kv, group, t):
    """One token each of sequences around the borders of records, spans and chunks, the shorter ones with stale values,
    NaN among them, behind their last position."""
    n = max(LENGTHS)
    c = cache(len(LENGTHS), kv, dim, n + 3)
    k, v = rows(11, (1, n, kv, dim), "f16"), rows(12, (1, n, kv, dim), "f16")
    every = (len(LENGTHS), n, kv, dim)
    c.append(k.expand(every), v.expand(every), ints(*[0] * len(LENGTHS)))
    kk, vv = (np.repeat(stored(f64(x)), len(LENGTHS), 0) for x in (k, v))
    bad = torch.full((len(LENGTHS), 40, kv, dim), float("nan"), device="cuda")
    c.append(bad, bad, ints(*LENGTHS))
    q = rows(13, (len(LENGTHS), 1, kv * group, dim), t)
    print(f"case single tokens dim {dim} kv {kv} group {group} {t}", flush=True)
    _, worst = check(c, q, [x - 1 for x in LENGTHS], k=kk, v=vv, t=t)
    print(f"worst error / bound {worst:.3f}", flush=True)
    c.close()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("dim,kv,group,tokens", [(64, 4, 2, 9), (128, 2, 4, 5), (128, 1, 5, 70), (256, 2, 1, 33), (128, 1, 8, 300)])
def test_windows_of_several_sequences(gpu, dim, kv, group, tokens, t):
    """Ragged windows: causal rows, counts, slots in another order, rows behind a count left alone."""
    pre = [0, 1, 500, 2040, 700]
    S, n = len(pre), max(pre) + tokens
    c = cache(S + 1, kv, dim, n)
    slot = [3, 0, 5, 1, 2]
    k, v = rows(21, (S, n, kv, dim), "f32", "head"), rows(22, (S, n, kv, dim), "f32", "head")
    c.append(k, v, ints(*[0] * S), slot=ints(*slot))
    kk, vv = np.zeros((S + 1, n, kv, dim)), np.zeros((S + 1, n, kv, dim))
    kk[slot], vv[slot] = stored(f64(k)), stored(f64(v))
    q = rows(23, (S, tokens, kv * group, dim), t, "head")
    count = [tokens, tokens - 1, 1, 0, tokens + 7]
    out = torch.full((S, kv * group, tokens, dim), 5.0, dtype=TYPES[t], device="cuda").transpose(1, 2)
    print(f"case windows dim {dim} kv {kv} group {group} tokens {tokens} {t}", flush=True)
    got, worst = check(c, q, pre, count, slot, kk, vv, t=t, out=out)
    print(f"worst error / bound {worst:.3f}", flush=True)
    for s in range(S):
        assert (got[s, max(0, count[s]):] == 5.0).all(), s
    c.close()


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_rows_that_see_nothing_and_rows_that_do_not_exist(gpu, t):
    c = cache(2, 2, 128, 600)
    k = rows(31, (2, 600, 2, 128))
    c.append(k, k, ints(0, 0))
    q = rows(32, (5, 3, 4, 128), t)
    got = f64(c.attend(q, ints(-2, 598, 0, -9, 2 ** 31 - 1), slot=ints(0, 1, 2, 1, 0)))
    assert (got[0, :2] == 0).all() and np.isfinite(got[0, 2]).all() and (got[0, 2] != 0).any()
    assert np.isfinite(got[1, :2]).all() and np.isnan(got[1, 2]).all()
    assert np.isnan(got[2]).all() and (got[3] == 0).all() and np.isnan(got[4]).all()
    c.close()


def test_nan_and_large_scores(gpu):
    """A NaN key makes the rows that see it NaN, a NaN value its block of 32 alone; scores far apart; a query of zeros, of
    huge and of tiny values; infinite queries."""
    D = 128
    c = cache(1, 1, D, 700)
    k, v = rows(41, (1, 700, 1, D)), rows(42, (1, 700, 1, D))
    v[0, 300, 0, 40] = float("inf")
    k[0, 600, 0, 0] = float("nan")
    k[0, 100] *= 40
    c.append(k, v, ints(0))
    q = rows(43, (1, 700, 2, D))
    q[0, 1], q[0, 2], q[0, 3] = 0.0, q[0, 2] * 1e30, q[0, 3] * 1e-30
    q[0, 4, 0, 5], q[0, 5, 1, 6] = float("inf"), float("nan")
    got = f64(c.attend(q, ints(0)))[0]
    assert np.isnan(got[600:]).all()
    assert np.isnan(got[300:600, :, 32:64]).all() and np.isfinite(got[300:600, :, :32]).all() and np.isfinite(got[300:600, :, 64:]).all()
    bad = np.isnan(got).any(-1)
    assert bad[4, 0] and not bad[4, 1] and bad[5, 1] and not bad[5, 0] and not bad[6:300].any() and not bad[:4].any()
    kk, vv = stored(f64(k))[0, :, 0], stored(f64(v))[0, :, 0]
    for h in range(2):
        r = np.r_[0:2, 3, 6:300]
        want, size = attention(f64(q)[0, r, h], kk, vv, r, D ** -0.5)
        lim = attention_bound(size, D, np.abs(vv[:300]).max(), want, torch.float32)
        assert (np.abs(got[r, h] - want) <= lim).all()
        # one score lies 1e29 above the others
        s = kk[:3] @ f64(q)[0, 2, h]
        assert (np.abs(got[2, h] - vv[s.argmax()]) <= 2.0 ** -20 * np.abs(vv[s.argmax()]).max()).all()
    c.close()


@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_queries_near_the_end_of_their_type(gpu, t):
    """Scores of 1e37, within float32's range: the largest takes all of the weight (an output off by its own rounding, and by two
    f16 parts of weights, one for bf16)."""
    D = 64
    c = cache(1, 1, D, 40)
    k, v = rows(45, (1, 40, 1, D)), rows(46, (1, 40, 1, D))
    c.append(k, v, ints(0))
    q = rows(47, (1, 40, 1, D), t)
    q *= 1e38 / float(q.abs().max())
    got = f64(c.attend(q, ints(0)))[0, :, 0]
    kk, vv = stored(f64(k))[0, :, 0], stored(f64(v))[0, :, 0]
    for r in range(40):
        want = vv[(kk[:r + 1] @ f64(q)[0, r, 0]).argmax()]
        assert (np.abs(got[r] - want) <= (half_step(TYPES[t]) + (2.0 ** -11 if t == "bf16" else 2.0 ** -20)) * np.abs(want).max()).all()
    c.close()


@pytest.mark.parametrize("magnitude", [1e-6, 1e-3, 1.0, 2000.0])
def test_values_of_every_magnitude(gpu, magnitude):
    """Values far below and above 1: weights are held in two f16 parts, which end at 2^-25 of a scale of 8."""
    c = cache(1, 1, 64, 1000)
    k, v = rows(51, (1, 1000, 1, 64)), rows(52, (1, 1000, 1, 64)) * magnitude
    c.append(k, v, ints(0))
    q = rows(53, (1, 1, 2, 64))
    got = f64(c.attend(q, ints(999)))[0, 0]
    want, size = attention(f64(q)[0, 0], stored(f64(k))[0, :, 0], stored(f64(v))[0, :, 0], [999, 999], 64 ** -0.5)
    # (a weight of at most 8 times its scale, error 2^-26, codes up to 8, over a sum of weights of at least 8)
    lim = attention_bound(size, 64, np.abs(f64(v)).max(), want, torch.float32) - 2.0 ** -20 + 2.0 ** -26 * 8 * 1000 / 8
    err = np.abs(got - want)
    print(f"magnitude {magnitude}: error {err.max() / np.abs(want).max():.2e} of the largest output", flush=True)
    assert (err <= lim).all()
    c.close()


@pytest.mark.parametrize("dim,kv,group", [(64, 2, 2), (128, 1, 4), (256, 1, 2)])
def test_a_row_has_the_same_bits_in_every_batch(gpu, dim, kv, group):
    n = 4200
    c = cache(1, kv, dim, n)
    k = rows(61, (1, n, kv, dim))
    c.append(k, k, ints(0))
    big = cache(2, kv, dim, 9000)
    big.append(k, k, ints(0), slot=ints(1))
    q = rows(62, (1, 300, kv * group, dim))
    for first in (0, 480, 2000, n - 300):
        print(f"case same bits dim {dim} first {first}", flush=True)
        want = c.attend(q, ints(first))
        assert (big.attend(q, ints(first), slot=ints(1)) == want).all()
        for m in (1, 2, 5, 16, 64):
            for j in (0, 31, 130, 299 - m + 1):
                got = c.attend(q[:, j:j + m], ints(first + j))
                assert (got == want[:, j:j + m]).all(), (m, j)
    c.close()
    big.close()


@pytest.mark.parametrize("kv,group,tokens,n,dim,t", [(8, 4, 16, 40000, 64, "f32"), (8, 4, 256, 9000, 64, "f32"), (1, 8, 64, 140000, 64, "f32"),
                                                     (8, 4, 256, 5000, 128, "f16"), (4, 2, 300, 3000, 256, "bf16"), (4, 2, 300, 2100, 256, "f32"),
                                                     (4, 2, 260, 700, 256, "f16"), (2, 7, 300, 1500, 128, "bf16")])
def test_long_calls_have_the_bits_of_single_tokens(gpu, kv, group, tokens, n, dim, t):
    """Calls that take a record per part of 1024 (several parts a wave, more than 128 of them, a single one) against single tokens and
    float64; the cache behind the tokens holds NaN."""
    c = cache(1, kv, dim, n + 324)
    nan = torch.full((1, 324, kv, dim), float("nan"), device="cuda")
    c.append(nan, nan, ints(n))
    k, v = rows(63, (1, n, kv, dim), t), rows(64, (1, n, kv, dim), t)
    c.append(k, v, ints(0))
    q = rows(65, (1, tokens, kv * group, dim), t)
    for first in (n - tokens, n // 2 - 100, 3):
        print(f"case long {tokens} tokens at {first}", flush=True)
        got = c.attend(q, ints(first))
        assert torch.isfinite(got).all()
        for j in (0, tokens // 2, tokens - 1):
            assert (c.attend(q[:, j:j + 1], ints(first + j)) == got[:, j:j + 1]).all(), j
    got = f64(c.attend(q, ints(n - tokens)))[0]
    h = kv * group - 1
    kk, vv = stored(f64(k[0, :, -1])), stored(f64(v[0, :, -1]))
    for j in (0, tokens // 3, tokens - 1):
        p = n - tokens + j
        want, size = attention(f64(q)[0, j, h][None], kk[:p + 1], vv[:p + 1], [p], dim ** -0.5)
        assert (np.abs(got[j, h] - want[0]) <= attention_bound(size, dim, np.abs(vv).max(), want, TYPES[t])[0]).all()
    c.close()


def test_offsets_beyond_32_bits(gpu):
    """The last slot, head and positions of a cache of 6 GB."""
    c = cache(20, 8, 256, 131072)
    assert c.nbytes > 2 ** 32
    k, v, q = rows(66, (1, 72, 8, 256)), rows(67, (1, 72, 8, 256)), rows(68, (1, 2, 8, 256))
    c.append(k, v, ints(131000), slot=ints(19))
    rk, rv = read(c, [131000], 72, slot=[19])
    assert (rk == stored(f64(k))).all() and (rv == stored(f64(v))).all()
    got = f64(c.attend(q, ints(131070), slot=ints(19)))[0]
    for h in (0, 7):  # the positions before hold zeros
        kk, vv = (np.concatenate([np.zeros((131000, 256)), x[0, :, h]]) for x in (rk, rv))
        want, size = attention(f64(q)[0, :, h], kk, vv, [131070, 131071], 1 / 16)
        assert (np.abs(got[:, h] - want) <= attention_bound(size, 256, np.abs(vv).max(), want, torch.float32)).all()
    assert (read(c, [131000], 72, slot=[18])[0] == 0).all()
    c.close()


def test_unaligned_rows_scales_and_output_in_place(gpu):
    D, kv, H = 128, 2, 6
    c = cache(3, kv, D, 900)
    k, v = rows(71, (3, 800, kv, D), "f16", "padded"), rows(72, (3, 800, kv, D), "f16", "padded")
    c.append(k, v, ints(0, 0, 0))
    kk, vv = stored(f64(k)), stored(f64(v))
    pos = [3, 400, 790]
    for t in ("f32", "f16", "bf16"):
        q = rows(73, (3, 10, H, D), t, "padded")
        print(f"case unaligned {t}", flush=True)
        check(c, q, pos, k=kk, v=vv, t=t, out=rows(74, (3, 10, H, D), t, "padded"))
        got, _ = check(c, q, pos, k=kk, v=vv, t=t, scale=0.3)
        same = q.clone()
        assert c.attend(same, ints(*pos), scale=0.3, out=same) is same and (same == got).all()
        wide = torch.zeros((3, 10, H, 2, D), dtype=TYPES[t], device="cuda")
        c.attend(q, ints(*pos), scale=0.3, out=wide[:, :, :, 1])  # every second head of a wider buffer
        assert (wide[:, :, :, 1] == got).all() and (wide[:, :, :, 0] == 0).all()
    # one token each as [sequence, head, dim]
    q3 = rows(75, (3, 1, H, D))
    assert (c.attend(q3[:, 0], ints(*pos)) == c.attend(q3, ints(*pos))[:, 0]).all()
    c.close()


def test_graphs_replay_at_new_positions_and_two_at_once(gpu):
    """A captured step (append, attend) replayed with other inputs and positions, between eager calls; two graphs with work
    spaces of their own, replayed side by side on two streams."""
    D, kv, H, S = 128, 2, 8, 2
    c = cache(S, kv, D, 3000)
    k0, v0 = rows(81, (S, 3000, kv, D)), rows(82, (S, 3000, kv, D))
    c.append(k0[:, :2500], v0[:, :2500], ints(0, 0))
    pos = ints(0, 0)
    parts = []
    for i in range(2):
        st = dict(k=torch.empty((S, 3, kv, D), device="cuda"), v=torch.empty((S, 3, kv, D), device="cuda"),
                  q=torch.empty((S, 3, H, D), device="cuda"), out=torch.empty((S, 3, H, D), device="cuda"),
                  work=torch.empty(c.work_bytes(S, 3, H), dtype=torch.uint8, device="cuda"), stream=torch.cuda.Stream())
        st["graph"] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(st["graph"], stream=st["stream"]):
            if i == 0:
                c.append(st["k"], st["v"], pos)
            c.attend(st["q"], pos, out=st["out"], work=st["work"])
        parts.append(st)
    a, b = parts
    for step, p in enumerate((0, 509, 2044, 2490)):
        print(f"case graphs at {p}", flush=True)
        pos.copy_(ints(p, p + 3))
        x = p + torch.arange(3, device="cuda")
        a["k"].copy_(torch.stack([k0[0, x], k0[1, x + 3]]))
        a["v"].copy_(torch.stack([v0[0, x], v0[1, x + 3]]))
        for j, st in enumerate(parts):
            st["q"].copy_(rows(90 + 2 * step + j, (S, 3, H, D)))
            st["out"].zero_()
        torch.cuda.synchronize()
        a["graph"].replay()
        torch.cuda.synchronize()
        first = a["out"].clone()
        for _ in range(3):  # the second graph and another replay of the first (the same values again) overlap
            with torch.cuda.stream(a["stream"]):
                a["graph"].replay()
            with torch.cuda.stream(b["stream"]):
                b["graph"].replay()
            torch.cuda.synchronize()
            assert (a["out"] == first).all()
            assert (c.attend(a["q"], pos) == first).all()
            assert (c.attend(b["q"], pos) == b["out"]).all()
    c.close()


def test_work_on_another_stream(gpu):
    c = cache(1, 1, 64, 400)
    k = rows(95, (1, 400, 1, 64))
    q = rows(96, (1, 2, 4, 64))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c.append(k, k, ints(0))
        got = c.attend(q, ints(300))
    s.synchronize()
    assert (c.attend(q, ints(300)) == got).all()
    c.close()


def test_refusals(gpu):
    from zerollm_amd._lib import ZLError
    c = cache(2, 2, 64, 100)
    k, q = rows(97, (2, 3, 2, 64)), rows(98, (2, 3, 4, 64))
    p = ints(0, 0)
    for bad, msg in ((lambda: c.append(k[..., :32], k[..., :32], p), "2 heads of 64 values"),
                     (lambda: c.append(k, k[:, :2], p), "v must be"),
                     (lambda: c.append(k, k.half(), p), "type of the other rows"),
                     (lambda: c.append(k.double(), k.double(), p), "float32, float16 or bfloat16"),
                     (lambda: c.append(k, k, p.long()), "int32"),
                     (lambda: c.append(k, k, ints(0)), "2 contiguous int32"),
                     (lambda: c.append(k.cpu(), k, p), "tensor on GPU"),
                     (lambda: c.append(k, k, p.cpu()), "tensor on GPU"),
                     (lambda: c.append(k, k, None), "positions missing"),
                     (lambda: c.attend(q[..., :32], p), "heads of 64 values"),
                     (lambda: c.attend(q, p, scale=-1.0), "scale must be positive"),
                     (lambda: c.attend(q, p, scale=float("nan")), "scale must be positive"),
                     (lambda: c.attend(q, p, out=q[:, :, :2]), "out must be"),
                     (lambda: c.attend(q, p, out=q[:, :1].expand(2, 3, 4, 64)), "must not share memory"),
                     (lambda: c.attend(q.transpose(2, 3).contiguous().transpose(2, 3), p), "must be contiguous"),
                     (lambda: c.attend(q, p, work=torch.empty(3, dtype=torch.uint8, device="cuda")), "bytes or more"),
                     (lambda: c.attend(q[0, 0], p), "must be .sequence, token, head, dim.")):
        with pytest.raises(ValueError, match=msg):
            bad()
    for bad, msg in ((lambda: c.attend(q[:, :, :3], p), "3 query heads over 2 KV heads"),
                     (lambda: c.attend(q, p, scale=float("inf")), "finite"),
                     (lambda: c.work_bytes(60000, 60000, 4), "query rows a call"),
                     (lambda: c.append(k[:, :1].expand(2, 2 ** 26, 2, 64), k[:, :1].expand(2, 2 ** 26, 2, 64), p), "tokens a call"),
                     (lambda: c.append(k.repeat(2, 1, 1, 1), k.repeat(2, 1, 1, 1), ints(0, 0, 0, 0)), "4 sequences in a cache of 2 slots")):
        with pytest.raises(ZLError, match=msg):
            bad()
    assert c.nbytes == 2 * 2 * 4 * 36 * 64
    c.close()
    c.close()
    with pytest.raises(ZLError, match="cache is closed"):
        c.append(k, k, p)
