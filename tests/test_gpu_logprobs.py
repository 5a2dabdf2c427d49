"""Log probabilities of logits rows (zerollm_amd.ops.logprobs) against plain float64."""
import numpy as np
import pytest
import torch

from ops_reference import TYPES, logprobs

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def check(x, tokens, top, **kw):
    """Ids exactly. An exponent x - m rounded to f32 and scaled to base 2 is off by 2^-23 of itself at most, so its
    exponential by |x - m| 2^-23 + 2^-22 of itself, which the terms e^-(m - x) make at most 2^-21 of the sum; the sums of
    a row (f32 partial sums of at most a few hundred terms, f64 beyond) 2^-20 at most; the logarithm and the difference to
    f32: half a step of the result and of x - m, at most 2^-23 of |x - m|. The entropy's sum has the same, relative to
    sum p |x - m|."""
    from zerollm_amd.ops import logprobs as own
    r = own(x, None if tokens is None else ints(tokens), top=top, **kw)
    x64 = x.double().cpu().numpy()
    lp, ent, ids, top_lp = logprobs(x64, np.zeros(len(x64), int) if tokens is None else np.asarray(tokens), top)
    with np.errstate(all="ignore"):
        m = x64.max(-1, keepdims=True)
        p = np.exp(x64 - m)
        spread = np.where(p > 0, p * (m - x64), 0).sum(-1) / p.sum(-1)

    def near(got, want, size):
        got = got.double().cpu().numpy()
        same = (got == want) | (np.isnan(got) & np.isnan(want))
        with np.errstate(all="ignore"):
            lim = 2.0 ** -19 + 2.0 ** -22 * np.abs(size)
            err = np.abs(got - want)
        ok = same | (np.isfinite(want) & (err <= lim))
        assert ok.all(), (got[~ok][:4], want[~ok][:4])

    if tokens is not None:
        near(r.logprobs, lp, lp)
    else:
        assert r.logprobs is None
    near(r.entropy, ent, np.abs(ent) + 4 * spread)
    if top:
        assert (r.top_ids.cpu().numpy() == ids).all()
        near(r.top_logprobs, top_lp, top_lp)
    else:
        assert r.top_ids is None and r.top_logprobs is None
    return r


@pytest.mark.parametrize("t", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (1, 2, 2), (3, 63, 5), (2, 64, 64), (5, 151936, 20), (1, 151936, 64),
                                            (70, 1000, 1), (300, 4099, 7), (2, 32003, 0), (1100, 257, 20)])
def test_rows_of_every_size(gpu, rows, vocab, top, t):
    g = torch.Generator().manual_seed(rows * 31 + vocab)
    x = (torch.randn((rows, vocab), generator=g) * 3).to(TYPES[t]).cuda()
    tokens = torch.randint(0, vocab, (rows,), generator=g).tolist()
    print(f"case logprobs {rows} x {vocab} top {top} {t}", flush=True)
    check(x, tokens, top)
    check(x, None, top)


@pytest.mark.parametrize("t", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [500, 40000])
def test_orders_that_fill_the_candidate_lists(gpu, vocab, t):
    """Ascending, descending and constant rows, rows of two values, large values at the ends, equal values everywhere."""
    i = torch.arange(vocab, dtype=torch.float32)
    g = torch.Generator().manual_seed(2)
    x = torch.stack([i * 1e-3, -i * 1e-3, torch.zeros(vocab), (i % 2), torch.where(i == vocab - 1, 50.0, 0.0),
                     torch.where(i < 100, 3.0, -torch.rand(vocab, generator=g)), (torch.rand(vocab, generator=g) * 8).floor(),
                     torch.where(i % 97 == 0, 0.0, -0.0), torch.where(i % 64 == 5, 9.0 + i / vocab, -5.0)]).to(TYPES[t]).cuda()
    for top in (1, 20, 64):
        print(f"case orders vocab {vocab} {t} top {top}", flush=True)
        check(x, [0, 1, 2, 3, vocab - 1, 99, 7, 8, 9], top)


def test_masked_infinite_and_nan_logits(gpu):
    inf, nan = float("inf"), float("nan")
    x = torch.randn((8, 3000), generator=torch.Generator().manual_seed(3)).cuda()
    x[0, 5:] = -inf            # five ids left
    x[1, 1:] = -inf            # one
    x[2] = -inf                # none
    x[3, 7] = inf
    x[4, 2900] = nan
    x[5, 0], x[5, 1] = nan, inf
    x[6, ::2] = -inf
    x[7] = 3e38
    x[7, ::3] = -3e38
    r = check(x, [2, 0, 0, 7, 5, 1, 3, 1], 20)
    lp = r.logprobs.cpu().numpy()
    assert np.isfinite(lp[[0, 1, 6, 7]]).all() and np.isnan(lp[[2, 3, 4, 5]]).all()
    assert lp[1] == 0.0 and r.entropy[1].item() == 0.0
    assert r.top_ids[0, :7].sort().values[-2:].tolist() == [5, 6]  # masked ids after the others, in order
    check(x[:2], [9, 1], 20)   # a given token that is masked
    assert np.isneginf(check(x[:1], [9], 0).logprobs.cpu().numpy()).all()
    assert np.isnan(check(x[6:], [-1, 3000], 3).logprobs.cpu().numpy()).all()


def test_many_rows_of_ties_and_masks(gpu):
    """Rows that one block takes whole, tile by tile, against the same rows a few at a time (twice the bound of one)."""
    from zerollm_amd.ops import logprobs as own
    inf, vocab = float("inf"), 40000
    x = torch.randn((8, vocab), generator=torch.Generator().manual_seed(4)).cuda()
    x[0] = 0.0
    x[1, 3:] = -inf
    x[2, :-2] = -inf
    x[3] = x[3].round()
    x[4, 30000:] = x[4, 0]
    x[5] = -inf
    x[6] = torch.where(torch.arange(vocab) % 3 == 0, 0.0, -0.0).cuda()
    few = check(x, list(range(8)), 20)
    print("case many rows", flush=True)
    many = own(x.repeat(1300, 1), ints(list(range(8)) * 1300), top=20)
    assert (many.top_ids.view(1300, 8, 20) == few.top_ids).all()
    for a, b in ((many.logprobs.view(1300, 8), few.logprobs), (many.entropy.view(1300, 8), few.entropy), (many.top_logprobs.view(1300, 8, 20), few.top_logprobs)):
        same = (a == b) | (a.isnan() & b.isnan())
        assert (same | ((a - b).abs() <= 2 * (2.0 ** -19 + 2.0 ** -22 * 5 * 16))).all()


def test_row_strides_outputs_and_work_of_the_caller(gpu):
    from zerollm_amd.ops import LogProbs, logprobs as own, logprobs_work_bytes
    w = torch.full((40, 1001), 1e30, device="cuda")
    w[:, 1:-7] = torch.randn((40, 993), generator=torch.Generator().manual_seed(4)).cuda()
    check(w[:, 1:-7], list(range(40)), 9)
    check(w[::3, 1:-7], list(range(14)), 9)
    x = w[:, 1:-7].contiguous()
    out = LogProbs(torch.empty(40, device="cuda"), None, torch.empty((40, 9), dtype=torch.int32, device="cuda"), None)
    work = torch.empty(logprobs_work_bytes(40, 993, 9), dtype=torch.uint8, device="cuda")
    r = own(x, ints(list(range(40))), top=9, out=out, work=work)
    full = own(x, ints(list(range(40))), top=9)
    assert r is out and (out.logprobs == full.logprobs).all() and (out.top_ids == full.top_ids).all()
    e = own(x[:0], ints([]), top=3)
    assert e.logprobs.shape == (0,) and e.top_ids.shape == (0, 3)


def test_logprobs_in_a_graph(gpu):
    from zerollm_amd.ops import LogProbs, logprobs as own, logprobs_work_bytes
    x, tok = torch.zeros((3, 50000), device="cuda"), ints([1, 2, 3])
    out = LogProbs(torch.empty(3, device="cuda"), torch.empty(3, device="cuda"), torch.empty((3, 5), dtype=torch.int32, device="cuda"),
                   torch.empty((3, 5), device="cuda"))
    work = torch.empty(logprobs_work_bytes(3, 50000, 5), dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        own(x, tok, top=5, out=out, work=work)
    for seed in range(4):
        x.copy_(torch.randn((3, 50000), generator=torch.Generator().manual_seed(seed)))
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = own(x, tok, top=5)
        assert (out.logprobs == want.logprobs).all() and (out.entropy == want.entropy).all()
        assert (out.top_ids == want.top_ids).all() and (out.top_logprobs == want.top_logprobs).all()


def test_refusals(gpu):
    from zerollm_amd._lib import ZLError
    from zerollm_amd.ops import logprobs as own
    x = torch.zeros((3, 100), device="cuda")
    for bad, msg in ((lambda: own(x[0]), "must be .rows, vocab."), (lambda: own(x.t()), "contiguous rows"),
                     (lambda: own(x, ints([1, 2])), "3 contiguous int32"), (lambda: own(x.double()), "float32"),
                     (lambda: own(x, work=torch.empty(1, dtype=torch.uint8, device="cuda")), "bytes or more")):
        with pytest.raises(ValueError, match=msg):
            bad()
    for top in (65, 101, -1):
        with pytest.raises(ZLError, match="n_top must be"):
            own(x, top=top)
