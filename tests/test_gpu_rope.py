"""Rotary positions (zerollm_amd.ops.Rope) against plain float64."""
import numpy as np
import pytest
import torch

from ops_reference import TYPES, angles, half_step, rotate

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def make(seed, shape, t):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(TYPES[t]).cuda()


def check(got, x, pos, th, gain, half, t):
    """Each output is two f32 products with cos and sin of 2^-22 (their own rounding, the rounding of the reduced angle, the
    polynomials, the factor), the sum and its rounding to the type; the reduced angle itself is off by 2^-52 of the turns."""
    x64 = x.double().cpu().numpy()
    want = rotate(x64, pos, th, gain, half)
    n = len(th)
    pair = np.abs(x64).copy()
    i0, i1 = (slice(0, n), slice(n, 2 * n)) if half else (slice(0, 2 * n, 2), slice(1, 2 * n, 2))
    both = gain * (np.abs(x64[..., i0]) + np.abs(x64[..., i1]))
    far = 2.0 ** -21 + 4 * 2.0 ** -52 * np.abs(np.asarray(pos, np.float64))[..., None] * th
    pair[..., i0] = pair[..., i1] = both * far[..., None, :]
    pair[..., 2 * n:] = 0.0
    g = got.double().cpu().numpy()
    lim = pair + half_step(TYPES[t]) * np.abs(want) * (1 + 2.0 ** -10)
    err = np.abs(g - want)
    assert (err <= lim).all(), (err.max(), np.argwhere(err > lim)[:3])
    assert (got[..., 2 * n:] == x[..., 2 * n:]).all()  # values that pass through
    return (err / np.maximum(lim, 1e-300))[..., :2 * n].max()


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("dim,rot", [(64, 64), (128, 128), (256, 64), (128, 2), (256, 250), (128, 98), (65, 6), (256, 256)])
def test_layouts_parts_of_the_head_and_far_positions(gpu, dim, rot, half, t):
    from zerollm_amd.ops import Rope
    pos = [[0, 1, 2, 3, 4], [131071 - 2, 131071 - 1, 131071, 131072, 131073], [-3, -2, -1, 0, 1], [2 ** 31 - 9 + i for i in range(5)]]
    th, gain = angles(rot, 10000.0)
    r = Rope(rot, neox=half)
    q, k = make(1, (4, 5, 6, dim), t), make(2, (4, 5, 2, dim), t)
    print(f"case rope dim {dim} rot {rot} half {half} {t}", flush=True)
    qo, ko = r.apply(q, k, ints([p[0] for p in pos]))
    worst = max(check(a, b, np.array(pos), th, gain, half, t) for a, b in ((qo, q), (ko, k)))
    print(f"worst error / bound {worst:.3f}", flush=True)
    r.close()


@pytest.mark.parametrize("kw", [dict(scaling="linear", factor=4.0), dict(scaling="yarn", factor=4.0, orig=4096),
                                dict(scaling="yarn", factor=8.5, orig=32768), dict(scaling="yarn", factor=2.0, orig=2048, fast=20.0, slow=2.0, gain=1.25),
                                dict(scaling="yarn", factor=1.0, orig=64), dict(freq=True), dict(scaling="linear", factor=3.0, freq=True)])
@pytest.mark.parametrize("base,rot", [(10000.0, 64), (1000000.0, 128), (500000.0, 20)])
def test_scalings(gpu, base, rot, kw):
    from zerollm_amd.ops import Rope
    kw = dict(kw)
    if kw.get("freq"):
        kw["freq"] = np.linspace(1.0, 9.0, rot // 2).astype(np.float32)
    th, gain = angles(rot, base, **kw)
    r = Rope(rot, base=base, scaling=kw.get("scaling"), factor=kw.get("factor", 1.0), orig_ctx=kw.get("orig", 0),
             beta_fast=kw.get("fast", 0), beta_slow=kw.get("slow", 0), attn_factor=kw.get("gain", 0), freq_factors=kw.get("freq"))
    pos = np.array([[7], [5000], [131000]])
    q = make(3, (3, 1, 4, 128), "f32")
    check(r.apply(q, None, ints([7, 5000, 131000]))[0], q, pos, th, gain, True, "f32")
    r.close()


def test_the_yarn_ramp_known_answers(gpu):
    """64 pairs of base 10^6 over 32768 positions: pairs up to 23 turn more than 32 times and keep their angle, pairs from 40
    on turn less than once and have it quartered."""
    from zerollm_amd.ops import Rope
    r, plain = Rope(128, base=1e6, scaling="yarn", factor=4.0, orig_ctx=32768), Rope(128, base=1e6)
    x = make(4, (1, 1, 1, 128), "f32")
    m = 1 + 0.1 * np.log(4.0)
    a = r.apply(x, None, ints([4000]))[0].double().cpu().numpy()[0, 0, 0] / m
    b = plain.apply(x, None, ints([4000]))[0].double().cpu().numpy()[0, 0, 0]
    c = plain.apply(x, None, ints([1000]))[0].double().cpu().numpy()[0, 0, 0]
    lo, hi = np.r_[:24, 64:88], np.r_[40:64, 104:128]
    assert np.abs(a[lo] - b[lo]).max() < 1e-5 and np.abs(a[hi] - c[hi]).max() < 1e-5
    mid = np.r_[25:39, 89:103]
    assert np.abs(a[mid] - b[mid]).max() > 0.01 and np.abs(a[mid] - c[mid]).max() > 0.01


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("half", [True, False])
def test_in_place_strides_counts_and_single_tokens(gpu, half, t):
    from zerollm_amd.ops import Rope
    rot, dim = 32, 64
    th, gain = angles(rot, 10000.0)
    r = Rope(rot, neox=half)
    # heads of a fused projection [token, (q | k | v), dim], each sequence's tokens strided, rotated in place
    x = make(5, (3, 4, 9, dim), t)
    want = x.clone()
    fused = x.clone()
    q, k = fused[:, :, :5], fused[:, :, 5:7]
    r.apply(q, k, ints([10, 20, 30]), count=ints([4, 0, 2]), out=(q, k))
    full = r.apply(x[:, :, :5].contiguous(), x[:, :, 5:7].contiguous(), ints([10, 20, 30]))
    for s, n in enumerate((4, 0, 2)):
        want[s, :n, :5], want[s, :n, 5:7] = full[0][s, :n], full[1][s, :n]
    assert (fused == want).all()
    check(full[0], x[:, :, :5], np.array([[10, 11, 12, 13], [20, 21, 22, 23], [30, 31, 32, 33]]), th, gain, half, t)
    # rows at odd values, head-major outputs
    wide = make(6, (3, 4, 5, dim + 1), t)
    y = torch.empty((3, 5, 4, dim), dtype=TYPES[t], device="cuda").transpose(1, 2)
    got = r.apply(wide[..., 1:], None, ints([10, 20, 30]), out=(y, None))[0]
    assert (got == r.apply(wide[..., 1:].contiguous(), None, ints([10, 20, 30]))[0]).all()
    # [sequence, head, dim]: one token each
    assert (r.apply(x[:, 1], None, ints([11, 21, 31]))[0] == r.apply(x, None, ints([10, 20, 30]))[0][:, 1]).all()
    assert r.apply(x[:0], None, ints([]))[0].shape == (0, 4, 9, dim)
    r.close()


def test_many_tokens_have_the_bits_of_few(gpu):
    from zerollm_amd.ops import Rope
    r = Rope(128, base=1e6, scaling="yarn", factor=4.0, orig_ctx=32768)
    q, k = make(7, (1, 1500, 8, 128), "bf16"), make(8, (1, 1500, 2, 128), "bf16")
    qo, ko = r.apply(q, k, ints([70000]))
    each = torch.arange(70000, 71500, dtype=torch.int32, device="cuda")
    q1, k1 = r.apply(q[0], k[0], each)
    assert (q1 == qo[0]).all() and (k1 == ko[0]).all()
    for i in (0, 3, 777, 1499):
        a = r.apply(q[:, i:i + 1], k[:, i:i + 1], ints([70000 + i]))
        assert (a[0] == qo[:, i:i + 1]).all() and (a[1] == ko[:, i:i + 1]).all()
    r.close()


def test_rope_in_a_graph(gpu):
    from zerollm_amd.ops import Rope
    r = Rope(64)
    q, k, pos = make(9, (2, 3, 4, 64), "f32"), make(10, (2, 3, 1, 64), "f32"), ints([0, 0])
    out = torch.empty_like(q), torch.empty_like(k)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r.apply(q, k, pos, out=out)
    for p in ([3, 5], [1000, 9], [0, 123456]):
        pos.copy_(ints(p))
        q.mul_(1.5)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = r.apply(q, k, ints(p))
        assert (out[0] == want[0]).all() and (out[1] == want[1]).all()
    r.close()


def test_refusals(gpu):
    from zerollm_amd._lib import ZLError
    from zerollm_amd.ops import Rope
    r = Rope(64)
    q, k, p = make(11, (2, 3, 4, 64), "f32"), make(12, (2, 3, 2, 64), "f32"), ints([0, 0])
    for bad, msg in ((lambda: r.apply(q, k[:, :2], p), "k must be"), (lambda: r.apply(q, k.half(), p), "type of the other rows"),
                     (lambda: r.apply(q, k, p, out=(q, k.half())), "type of the other rows"),
                     (lambda: r.apply(q, k, ints([0])), "2 contiguous int32"),
                     (lambda: r.apply(q, k, p, out=(q[:, :, :1].expand_as(q), k)), "must not share memory")):
        with pytest.raises(ValueError, match=msg):
            bad()
    with pytest.raises(ZLError, match="below the 64 rotated values"):
        r.apply(q[..., :32], None, p)
    r.close()
    with pytest.raises(ZLError, match="rope is closed"):
        r.apply(q, k, p)
