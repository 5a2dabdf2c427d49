"""Models on the long-context operators: a KV cache in 4 bits, positions scaled beyond the trained context, log probabilities
of passes; and the operators as a program strings them together."""
import numpy as np
import pytest

from ops_reference import angles, attention, logprobs as plain_logprobs, rotate, stored
from zerollm_amd import gguf, synth
from zerollm_amd import model as Mdl
from zerollm_amd.generate import generate, score
from zerollm_amd.speculative import generate_speculative

pytestmark = pytest.mark.gpu

YARN = dict(scaling="yarn", factor=4.0, beta_fast=24.0)


def prompt(n, seed, vocab):
    return [int(x) for x in np.random.default_rng(seed).integers(0, vocab, n)]


def rms(x, w, eps):
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w


def edge(x):
    """How near the values' x / d + 8.5 come to a whole number, above which the next code starts (values at the ends apart, where
    either side is the same code)."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    d = np.take_along_axis(b, np.abs(b).argmax(-1)[..., None], -1) / -8.0
    y = b / d + 8.5
    y = y[(y > 0.9) & (y < 15.5)]  # (0.5 and 16.5 are the largest values themselves)
    return np.abs(y - np.round(y)).min()


def plain_logits(spec, tokens, rope=None):
    """Every position's logits in float64 from float32 weights, keys and values as a cache in 4 bits holds them; and how near
    any of them came to another code. A qwen35 spec of interval 1 has gated attention in every layer."""
    w = {t.name: synth.tensor_bytes(t).view(np.float32).astype(np.float64).reshape(t.rows, t.cols) for t in spec.tensors}
    eps, hd, nh, nkv = float(np.float32(spec.rms_eps)), spec.head_dim, spec.n_head, spec.n_head_kv
    n, near = len(tokens), 1.0
    n_rot = spec.n_rot or hd
    kw = dict(scaling=None) if rope is None else dict(scaling=rope["scaling"], factor=rope["factor"], orig=rope.get("orig_ctx", spec.ctx_train),
                                                      fast=rope.get("beta_fast", 32.0), slow=rope.get("beta_slow", 1.0))
    th, gain = angles(n_rot, float(np.float32(spec.rope_base)), **kw)
    x = w["token_embd.weight"][tokens]
    for l in range(spec.n_layer):
        def W(name):
            return w[f"blk.{l}.{name}.weight"]

        h = rms(x, W("attn_norm"), eps)
        q = (h @ W("attn_q").T).reshape(n, nh, -1)
        q, gate = q[..., :hd], q[..., hd:]
        k, v = ((h @ W(s).T).reshape(n, nkv, hd) for s in ("attn_k", "attn_v"))
        if spec.arch != "llama":
            q, k = rms(q, W("attn_q_norm"), eps), rms(k, W("attn_k_norm"), eps)
        half = spec.arch != "llama"
        q, k = rotate(q, np.arange(n), th, gain, half), rotate(k, np.arange(n), th, gain, half)
        near = min(near, edge(k), edge(v))
        k, v = stored(k), stored(v)
        o = np.stack([attention(q[:, i], k[:, i * nkv // nh], v[:, i * nkv // nh], np.arange(n), hd ** -0.5)[0] for i in range(nh)], 1)
        if spec.hybrid:
            o = o / (1 + np.exp(-gate))
        x = x + o.reshape(n, -1) @ W("attn_output").T
        h = rms(x, W("post_attention_norm" if spec.hybrid else "ffn_norm"), eps)
        g = h @ W("ffn_gate").T
        x = x + (g / (1 + np.exp(-g)) * (h @ W("ffn_up").T)) @ W("ffn_down").T
    return rms(x, w["output_norm.weight"], eps) @ w.get("output.weight", w["token_embd.weight"]).T, near


def float_spec(kind, seed):
    if kind == "gated":
        return synth.build_qwen35_spec(256, 2, 4, 1, 256, 64, 512, 512, 32, synth.qwen35_types(gguf.F32), seed, interval=1, std=0.06)
    nh, nkv, hd = {"qwen3": (6, 2, 64), "llama": (4, 1, 128)}[kind]
    return synth.build_spec(kind, 256, 2, nh, nkv, hd, 512, 512, 32, synth.all_type(gguf.F32), seed, std=0.06)


CASES = [("qwen3", 3, None), ("llama", 4, None), ("gated", 5, None), ("qwen3", 6, YARN), ("gated", 7, dict(scaling="linear", factor=3.0)),
         ("llama", 28, dict(scaling="yarn", factor=2.0, orig_ctx=20))]


@pytest.mark.parametrize("kind,seed,rope", CASES)
def test_logits_of_a_cache_in_4_bits(gpu, kind, seed, rope):
    """Against float64. Every float32 vector that a layer stores (some 12 of them) is off by 2^-24 of its largest values, up to 8
    times its typical ones, and the attention by 2^-18: 2^-15 of the largest logit covers two layers of both. A value whose code
    may be another one by such an error (2^-16 of the largest value of a block: 1e-4 of a code) would be off by more: the inputs
    have none."""
    spec = float_spec(kind, seed)
    n = 30 if rope is None else 44  # (trained on 32)
    toks = prompt(n, seed, spec.vocab)
    want, near = plain_logits(spec, toks, rope)
    assert near > 1e-5
    print(f"case {kind} {rope}", flush=True)
    m = synth.build_on_device(spec, ctx=1000, kv="q4_0", rope=rope)
    assert m.kv == "q4_0" and m.ctx == 32 * (rope["factor"] if rope else 1)
    one = np.stack([m.forward(t).copy() for t in toks])
    assert np.abs(one - want).max() <= 2.0 ** -15 * np.abs(want).max()
    # passes of several tokens: the same bits
    m.truncate(0)
    cuts = [0, 2, 7, 8, 24, min(40, n)] + ([n] if n > 40 else [])
    got = np.concatenate([m.forward_batch(toks[a:b], logits="all").copy() for a, b in zip(cuts, cuts[1:])])
    assert (got.view(np.uint32) == one.view(np.uint32)).all()
    m.close()


@pytest.mark.parametrize("heads", [8, 32])
def test_long_prompts_rollbacks_and_fresh_runs(gpu, heads):
    """1300 positions in passes of 64 (of 32 heads: the attention of many rows), of 7 and of 1 give the same bits, also after
    rollbacks to the middle of a record, of a span and to nothing."""
    spec = synth.build_spec("qwen3", 256, 2, heads, 4, 64, 512, 2048, 4096, synth.all_type(gguf.Q8_0), 9)
    toks = prompt(1300, 2, spec.vocab)
    print(f"case heads {heads}", flush=True)
    m = synth.build_on_device(spec, ctx=2048, kv="q4_0", max_batch=64, logits_batch=64)

    def feed(step, start=0, end=len(toks)):
        last = None
        for i in range(start, end, step):
            last = m.forward_batch(toks[i:min(i + step, end)], logits="last").copy()
        return last

    want = feed(64)
    m.truncate(0)
    assert (feed(7).view(np.uint32) == want.view(np.uint32)).all()
    for back in (1299, 1237, 1024, 705, 1):
        m.truncate(back)
        m.forward_batch(prompt(9, back, spec.vocab), logits=False)  # what a rejected draft leaves behind
        m.truncate(back)
        assert (feed(1 if back > 1200 else 64, back).view(np.uint32) == want.view(np.uint32)).all(), back
    m.reset()
    assert (feed(33).view(np.uint32) == want.view(np.uint32)).all()
    m.close()


def test_speculative_greedy_equals_plain_greedy(gpu, close_files):
    p = prompt(60, 3, 32000)
    plain = Mdl.HipModel.load(close_files[0], ctx=256, kv="q4_0")
    want = list(generate(plain, p, max_tokens=40))
    T = Mdl.HipModel.load(close_files[0], ctx=256, kv="q4_0")
    D = Mdl.HipModel.load(close_files[1], ctx=256, kv="q4_0")
    for k in (1, 4, 8):
        print(f"case speculative k={k}", flush=True)
        st = {}
        assert list(generate_speculative(T, D, p, k=k, max_tokens=40, stats=st)) == want
        assert st["speculative"]["cycles"] > 0
    for m in (plain, T, D):
        m.close()


def test_a_hybrid_model_rolls_back(gpu):
    spec = synth.tiny_qwen35(seed=51)
    p = [3, 70, 5, 200, 12, 9]
    plain = synth.build_on_device(spec, ctx=96, kv="q4_0")
    want = list(generate(plain, p, max_tokens=24))
    T = synth.build_on_device(spec, ctx=96, max_batch=8, kv="q4_0")
    D = synth.build_on_device(synth.tiny_qwen35(seed=52, n_layer=2, interval=2), ctx=96, kv="q4_0")
    print("case hybrid", flush=True)
    for k in (1, 4):
        assert list(generate_speculative(T, D, p, k=k, max_tokens=24)) == want
    for m in (plain, T, D):
        m.close()


def test_the_cache_takes_its_size(gpu):
    spec = synth.build_spec("qwen3", 256, 2, 8, 4, 64, 512, 2048, 65536, synth.all_type(gguf.Q8_0), 9)
    size = {}
    for kv in ("f16", "q4_0"):
        m = synth.build_on_device(spec, ctx=65536, kv=kv, max_batch=1)
        size[kv] = m.device_bytes
        m.close()
    assert size["f16"] - size["q4_0"] >= 65536 * 2 * 4 * 64 * (4 - 1.125)  # (and the scores of a pass)


@pytest.mark.parametrize("kv", ["f16", "q4_0"])
def test_log_probabilities_of_a_pass(gpu, tiny_files, kv):
    """Against float64 of the returned logits; the bound is that of the operator's own tests."""
    toks = prompt(12, 4, 32000)
    m = Mdl.HipModel.load(tiny_files[0], ctx=64, kv=kv)
    x = m.forward_batch(toks, logits="all").copy()
    for n, row0, top in ((12, 0, 5), (3, 7, 0), (1, 11, 64), (0, 0, 1)):
        given = prompt(n, 5 + n, 32000)
        print(f"case rows {row0} + {n} top {top}", flush=True)
        r = m.logprobs(n, row0, tokens=given, top=top)
        lp, ent, ids, best = plain_logprobs(x[row0:row0 + n].astype(np.float64), np.array(given, int), top) if n else (np.zeros(0),) * 4
        assert np.abs(r.logprobs - lp).max(initial=0) <= 2.0 ** -19 + 2.0 ** -22 * np.abs(lp).max(initial=0)
        assert np.abs(r.entropy - ent).max(initial=0) <= 2.0 ** -19 + 2.0 ** -22 * 5 * 32
        if top and n:
            assert (r.top_ids == ids).all() and np.abs(r.top_logprobs - best).max() <= 2.0 ** -19 + 2.0 ** -22 * np.abs(best).max()
        else:
            assert r.top_ids is None or r.top_ids.shape == (n, top)
    assert m.logprobs(2).logprobs is None
    last = m.forward(toks[0]).copy()
    one = m.logprobs(tokens=[7], top=3)
    assert one.top_ids[0, 0] == last.argmax()
    m.close()


def test_scores_of_a_text(gpu, tiny_files):
    """Passes of any width give the single tokens' bits; a longer text starts from the shared context."""
    ids = prompt(50, 6, 32000)
    m = Mdl.HipModel.load(tiny_files[0], ctx=64, kv="q4_0")
    one = []
    for i in range(49):
        m.forward_batch([ids[i]], logits="last", copy=False)
        one.append(m.logprobs(tokens=[ids[i + 1]], top=2))
    want = np.concatenate([o.logprobs for o in one])
    print("case score", flush=True)
    for start in (1, 2, 17, 49):
        r = score(m, ids, start=start, top=2)
        assert (r.logprobs.view(np.uint32) == want[start - 1:].view(np.uint32)).all() and m.tokens == ids[:-1]
        assert (r.top_ids == np.concatenate([o.top_ids for o in one])[start - 1:]).all()
    m.reset()
    assert (score(m, ids).logprobs.view(np.uint32) == want.view(np.uint32)).all()
    for bad in (0, 50):
        with pytest.raises(ValueError, match="start must be"):
            score(m, ids, start=bad)
    with pytest.raises(ValueError, match="do not fit"):
        score(m, prompt(66, 1, 32000))
    m.close()


def test_refusals_of_models(gpu, tiny_files):
    from zerollm_amd._lib import ZLError
    with pytest.raises(ValueError, match="kv must be"):
        Mdl.HipModel.load(tiny_files[0], kv="q8_0")
    with pytest.raises(ValueError, match="scaling must be"):
        Mdl.HipModel.load(tiny_files[0], rope=dict(scaling="ntk", factor=2.0))
    with pytest.raises(ValueError, match="rope does not take base, n_rot"):
        Mdl.HipModel.load(tiny_files[0], rope=dict(scaling="linear", factor=2.0, base=1e4, n_rot=64))
    with pytest.raises(ZLError, match="factor"):
        Mdl.HipModel.load(tiny_files[0], rope=dict(scaling="linear", factor=0.5))
    m = Mdl.HipModel.load(tiny_files[0], ctx=64, kv="q4_0")
    m.forward_batch([1, 2, 3], logits="all")
    for a in (dict(n=17), dict(n=1, row0=16), dict(n=1, row0=-1)):
        with pytest.raises(ZLError, match="out of range"):
            m.logprobs(**a)
    for a in (dict(n=-1), dict(top=65), dict(top=-1), dict(n=2, tokens=[1])):
        with pytest.raises(ValueError):
            m.logprobs(**a)
    with pytest.raises(ZLError, match="context full"):
        for _ in range(5):
            m.forward_batch(list(range(16)))
    m.close()
    with pytest.raises(ZLError, match="closed"):
        m.logprobs()


def test_the_operators_together(gpu):
    """A layer of a user's own program: rotary positions, the cache, its attention and the log probabilities of a head, for a prompt,
    then for single tokens in a captured graph whose positions advance on the device, against float64."""
    import torch
    from zerollm_amd.ops import KVCacheQ4, Rope, logprobs, logprobs_work_bytes
    g = torch.Generator(device="cpu").manual_seed(11)
    seqs, nh, nkv, hd, vocab, n0, steps = 3, 8, 2, 64, 700, 33, 4

    def rand(*shape):
        return torch.randn(*shape, generator=g).cuda()

    q, k, v = rand(seqs, n0 + steps, nh, hd), rand(seqs, n0 + steps, nkv, hd), rand(seqs, n0 + steps, nkv, hd)
    head = rand(nh * hd, vocab) * 0.1
    start = [0, 5, 60]
    tokens = torch.tensor([1, 2, 699], dtype=torch.int32).cuda()
    rope, cache = Rope(hd, base=1e6, scaling="yarn", factor=4.0, orig_ctx=64), KVCacheQ4(seqs, nkv, hd, 128)
    pos = torch.tensor(start, dtype=torch.int32).cuda()
    junk = rand(seqs, 60, nkv, hd)  # what earlier turns left in the cache
    cache.append(junk, junk, torch.zeros(seqs, dtype=torch.int32).cuda())

    def run(q, k, v, work, out):
        rope.apply(q, k, pos, out=(q, k))
        cache.append(k, v, pos)
        o = cache.attend(q, pos, out=q, work=work[0])
        torch.mm(o[:, -1].reshape(seqs, nh * hd), head, out=out[0])
        logprobs(out[0], tokens, top=4, out=out[1], work=work[1])

    def buffers(n):
        lg = torch.empty(seqs, vocab, device="cuda")
        work = [torch.empty(b, dtype=torch.uint8, device="cuda") for b in (cache.work_bytes(seqs, n, nh), logprobs_work_bytes(seqs, vocab, 4))]
        return work, (lg, logprobs(lg.zero_(), tokens, top=4))

    got = []
    work, out = buffers(n0)
    run(q[:, :n0].clone(), k[:, :n0].clone(), v[:, :n0], work, out)
    got.append([x.clone() for x in (out[1].logprobs, out[1].entropy, out[1].top_ids, out[1].top_logprobs)])
    pos += n0
    q1, k1, v1 = torch.empty(seqs, 1, nh, hd, device="cuda"), torch.empty(seqs, 1, nkv, hd, device="cuda"), torch.empty(seqs, 1, nkv, hd, device="cuda")
    work, out = buffers(1)
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    keep = pos.clone()
    with torch.cuda.stream(side):  # once before the capture; what it writes is written again
        q1.copy_(q[:, n0:n0 + 1]), k1.copy_(k[:, n0:n0 + 1]), v1.copy_(v[:, n0:n0 + 1])
        run(q1, k1, v1, work, out)
    side.synchronize()
    print("case capture", flush=True)
    with torch.cuda.graph(graph, stream=side):
        run(q1, k1, v1, work, out)
        pos += 1
    assert (pos == keep).all()
    for s in range(steps):
        q1.copy_(q[:, n0 + s:n0 + s + 1]), k1.copy_(k[:, n0 + s:n0 + s + 1]), v1.copy_(v[:, n0 + s:n0 + s + 1])
        graph.replay()
        torch.cuda.synchronize()
        got.append([x.clone() for x in (out[1].logprobs, out[1].entropy, out[1].top_ids, out[1].top_logprobs)])
    # float64: the junk stays where no sequence has written
    th, gain = angles(hd, 1e6, scaling="yarn", factor=4.0, orig=64)
    f = [x.double().cpu().numpy() for x in (q, k, v, junk, head)]
    for i, s in enumerate(start):
        at = s + np.arange(n0 + steps)
        qr, kr = rotate(f[0][i], at, th, gain, True), rotate(f[1][i], at, th, gain, True)
        # (rows rotated in f32: a value within 2^-20 of a code's edge could take the other one)
        near = min(edge(kr), edge(f[2][i]))
        assert near > 2.0 ** -18
        kk, vv = (np.concatenate([stored(f[3][i])[:s], stored(x)]) for x in (kr, f[2][i]))
        for j, t in enumerate([n0 - 1] + list(range(n0, n0 + steps))):
            o = np.concatenate([attention(qr[t:t + 1, h], kk[:, h * nkv // nh], vv[:, h * nkv // nh], [s + t], hd ** -0.5)[0] for h in range(nh)])
            lg = o.reshape(1, -1) @ f[4]
            lp, ent, ids, best = plain_logprobs(lg, np.array([int(tokens[i])]), 4)
            # logits off by the attention's 2^-17 of values up to 4 over sums of 512 factors of 0.1 (rms: 23 times 0.1), and f32 sums
            lim = 2.0 ** -17 * 4 * 2.3 * 4
            a = [x[i].cpu().numpy() for x in got[j]]
            assert abs(a[0] - lp[0]) <= 2 * lim and abs(a[1] - ent[0]) <= 20 * lim
            assert (a[2] == ids[0]).all() and np.abs(a[3] - best[0]).max() <= 2 * lim
