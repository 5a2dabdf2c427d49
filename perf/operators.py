"""The operators of long contexts, through the package's entry points (zerollm_amd.ops): attention over a 4-bit KV cache,
rotary positions, log probabilities.

Kinds of case:
- "attend"   a step of several sequences: their new keys and values are appended to the cache (KVCacheQ4.append), then the
             new tokens' queries attend over it (KVCacheQ4.attend);
- "store"    keys and values into the cache (append) and what they stand for back out of it (read);
- "rope"     queries and keys rotated to their positions (Rope.apply);
- "logprobs" log probability of a given token, entropy and the top alternatives of logits rows (logprobs).
With `own` unset, run() computes the same in elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a drafted token of a small model at an ordinary length: launch latency
        {"name": "decode_700", "kind": "attend", "seqs": 1, "tokens": 1, "heads": 16, "kv_heads": 8, "dim": 128, "prefix": 700,
         "ragged": False, "capacity": 1024, "type": "f32", "head_major": False},
        # many short conversations of unequal length decoded together
        {"name": "decode_batch", "kind": "attend", "seqs": 24, "tokens": 1, "heads": 8, "kv_heads": 4, "dim": 64, "prefix": 2017,
         "ragged": True, "capacity": 4096, "type": "bf16", "head_major": False},
        # checking k = 8 drafts deep in a long conversation
        {"name": "verify_16k", "kind": "attend", "seqs": 1, "tokens": 9, "heads": 32, "kv_heads": 8, "dim": 128, "prefix": 16384,
         "ragged": False, "capacity": 16658, "type": "f32", "head_major": False},
        # the next turn of a long conversation: a piece of prompt over a long cached prefix (the most arithmetic)
        {"name": "prompt_12k", "kind": "attend", "seqs": 1, "tokens": 256, "heads": 32, "kv_heads": 8, "dim": 128, "prefix": 12000,
         "ragged": False, "capacity": 16384, "type": "f16", "head_major": True},
        # one token over a cache four times the trained context (the most bytes)
        {"name": "decode_131k", "kind": "attend", "seqs": 1, "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "prefix": 131000,
         "ragged": False, "capacity": 131072, "type": "f16", "head_major": False},
        # a prompt's keys and values into the cache, and out again as another cache would take them
        {"name": "store_prompt", "kind": "store", "seqs": 1, "tokens": 2048, "kv_heads": 8, "dim": 128, "prefix": 0,
         "ragged": False, "capacity": 2048, "type": "bf16", "head_major": False},
        # verification windows of several sequences at odd positions, wide heads, unequal counts
        {"name": "store_windows", "kind": "store", "seqs": 16, "tokens": 5, "kv_heads": 4, "dim": 256, "prefix": 2048,
         "ragged": True, "capacity": 2304, "type": "f32", "head_major": False},
        # the queries and keys of a verification pass: launch latency
        {"name": "rope_verify", "kind": "rope", "tokens": 9, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128, "half": True,
         "base": 1000000.0, "scaling": "none", "factor": 1.0, "orig": 32768, "first": 16384, "type": "f32"},
        # a long document's, four times the trained context, adjacent pairs in part of the head
        {"name": "rope_document", "kind": "rope", "tokens": 16384, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 64, "half": False,
         "base": 10000.0, "scaling": "yarn", "factor": 4.0, "orig": 32768, "first": 114600, "type": "bf16"},
        # the rows of a verification pass with the alternatives a client shows
        {"name": "logprobs_verify", "kind": "logprobs", "rows": 5, "vocab": 151936, "top": 20, "type": "f32"},
        # one full batch of a text whose likelihood is measured
        {"name": "logprobs_score", "kind": "logprobs", "rows": 64, "vocab": 151936, "top": 0, "type": "f32"},
        # many answers' tokens at once, logits of 16 bits (many equal values)
        {"name": "logprobs_answers", "kind": "logprobs", "rows": 2048, "vocab": 32000, "top": 5, "type": "bf16"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    r, ty = rng.random(), rng.choice(["f32", "f16", "bf16"])
    if r < 0.45:
        dim, kv, g = rng.choice([64, 128, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 5, 7, 8])
        s = rng.choice([1, 1, 1, _log(rng, 2, 32)])
        t = rng.choice([1, 1, 2, 5, 9, _log(rng, 10, 300)])
        top = min(131000, 60e6 / (s * kv * dim), 4.5e10 / (4 * s * t * kv * g * dim), 2e8 / (s * t * kv * g))
        p = _log(rng, 1, max(2, top))
        return {"kind": "attend", "seqs": s, "tokens": t, "heads": kv * g, "kv_heads": kv, "dim": dim, "prefix": p,
                "ragged": s > 1 and rng.random() < 0.7, "capacity": p + t + rng.randint(0, 300), "type": ty,
                "head_major": rng.random() < 0.3}
    if r < 0.6:
        dim, kv, s = rng.choice([64, 128, 256]), rng.choice([1, 2, 4, 8]), _log(rng, 1, 24)
        t, p = _log(rng, 1, max(1, 2048 * 8 * 128 // (s * kv * dim))), _log(rng, 1, 4000) - 1
        return {"kind": "store", "seqs": s, "tokens": t, "kv_heads": kv, "dim": dim, "prefix": p, "ragged": s > 1 and rng.random() < 0.7,
                "capacity": p + t + rng.randint(0, 300), "type": ty, "head_major": rng.random() < 0.3}
    if r < 0.8:
        dim, kv, g = rng.choice([64, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 3, 4, 8])
        n = _log(rng, 1, min(16384, 16384 * 40 * 128 // (kv * (g + 1) * dim)))
        return {"kind": "rope", "tokens": n, "heads": kv * g, "kv_heads": kv, "dim": dim, "rot": 2 * rng.randint(1, dim // 2),
                "half": rng.random() < 0.6, "base": rng.choice([10000.0, 500000.0, 1000000.0]),
                "scaling": rng.choice(["none", "linear", "yarn"]), "factor": rng.choice([2.0, 4.0, 8.5]),
                "orig": rng.choice([4096, 32768]), "first": _log(rng, 1, 1000000) - 1, "type": ty}
    n = _log(rng, 1, 2048)
    v = _log(rng, 300, min(152000, 64e6 / n))
    return {"kind": "logprobs", "rows": n, "vocab": v, "top": rng.choice([0, 1, 5, 20, 50]), "type": ty}


# ---------------------------------------------------------------------------------------------- inputs
def _positions(case):
    """The first new position of each sequence: all after the prefix, or after lengths spread up to it."""
    n, p = case["seqs"], case["prefix"]
    return [p * (1 + 7 * s % n) // n if case["ragged"] else p for s in range(n)]


def _counts(case):
    """Tokens of each sequence of a ragged window: all of them, one less, ..., one, and from the start again."""
    return [case["tokens"] - s % min(case["tokens"], 5) if case["ragged"] else case["tokens"] for s in range(case["seqs"])]


def _rows(g, shape, ty, head_major, channels=None):
    """[sequence, token, head, dim] values; head_major: as a view of [sequence, head, token, dim]."""
    s, t, h, d = shape
    x = torch.empty((s, h, t, d) if head_major else shape, device=DEV).normal_(0, 1, generator=g)
    if channels is not None:
        x *= channels[:, None] if head_major else channels
    x = x.to(TYPES[ty])
    return x.transpose(1, 2) if head_major else x


def _inputs(case, seed):
    """The tensors of a call. Keys have a few large channels, as rotated keys have, and the first one attracts weight."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    d = {}
    if case["kind"] in ("attend", "store"):
        s, t, kv, dim, ty = case["seqs"], case["tokens"], case["kv_heads"], case["dim"], case["type"]
        ch = torch.empty((kv, dim), device=DEV).normal_(0, 0.5, generator=g).exp()
        d["k"] = _rows(g, (s, t, kv, dim), ty, case["head_major"], ch)
        d["v"] = _rows(g, (s, t, kv, dim), ty, case["head_major"])
        d["pos"] = torch.tensor(_positions(case), dtype=torch.int32, device=DEV)
        if case["kind"] == "attend":
            d["q"] = _rows(g, (s, t, case["heads"], dim), ty, case["head_major"])
            p = max(_positions(case))
            d["k0"] = _rows(g, (s, p, kv, dim), "f16", False, ch)
            d["k0"][:, :1] *= 2
            d["v0"] = _rows(g, (s, p, kv, dim), "f16", False)
        else:
            d["count"] = torch.tensor(_counts(case), dtype=torch.int32, device=DEV) if case["ragged"] else None
    elif case["kind"] == "rope":
        d["q"], d["k"] = (_rows(g, (case["tokens"], 1, h, case["dim"]), case["type"], False)[:, 0]
                          for h in (case["heads"], case["kv_heads"]))
        d["pos"] = torch.arange(case["first"], case["first"] + case["tokens"], dtype=torch.int32, device=DEV)
    else:
        x = torch.empty((case["rows"], case["vocab"]), device=DEV).normal_(0, 2.5, generator=g)
        d["logits"] = x.to(TYPES[case["type"]])
        d["tokens"] = torch.randint(0, case["vocab"], (case["rows"],), device=DEV, dtype=torch.int32, generator=g)
    return d


class _State:
    def __init__(self, **kw):
        self.cache = None
        self.__dict__.update(kw)

    def __del__(self):
        if self.cache is not None:
            self.cache.close()


def prepare(case, seed):
    s = _State(case=case, **_inputs(case, seed))
    kind = case["kind"]
    if kind in ("attend", "store"):
        n, kv, dim, cap = case["seqs"], case["kv_heads"], case["dim"], case["capacity"]
        if kind == "store":
            s.ko, s.vo = torch.zeros_like(s.k), torch.zeros_like(s.v)
        if own:
            from zerollm_amd import model, ops
            model.init(0)
            s.cache = ops.KVCacheQ4(n, kv, dim, cap)
            if kind == "attend":
                # (sequences shorter than the longest hold a longer prefix's keys behind them, which nothing sees)
                s.cache.append(s.k0, s.v0, torch.zeros_like(s.pos))
                s.out = torch.empty((n, case["tokens"], case["heads"], dim), dtype=TYPES[case["type"]], device=DEV)
                s.work = torch.empty(s.cache.work_bytes(n, case["tokens"], case["heads"]), dtype=torch.uint8, device=DEV)
        else:
            shape = (n, kv, cap)
            s.kn, s.vn = (torch.zeros((*shape, dim), dtype=torch.uint8, device=DEV) for _ in range(2))
            s.kd, s.vd = (torch.zeros((*shape, dim // 32), dtype=torch.float16, device=DEV) for _ in range(2))
            s.sid = torch.arange(n, device=DEV)[:, None]
            if kind == "attend":
                _put(s.kn, s.kd, s.k0, s.sid, torch.zeros_like(s.pos))
                _put(s.vn, s.vd, s.v0, s.sid, torch.zeros_like(s.pos))
        if kind == "attend":
            del s.k0, s.v0
    elif kind == "rope" and own:
        from zerollm_amd import model, ops
        model.init(0)
        s.rope = ops.Rope(case["rot"], neox=case["half"], base=case["base"], scaling=case["scaling"], factor=case["factor"],
                          orig_ctx=case["orig"])
        s.outs = torch.empty_like(s.q), torch.empty_like(s.k)
    elif kind == "logprobs" and own:
        from zerollm_amd import model, ops
        model.init(0)
        s.work = torch.empty(ops.logprobs_work_bytes(case["rows"], case["vocab"], case["top"]), dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------------------------------------- a pass
def run(s):
    c = s.case
    if own:
        from zerollm_amd import ops
        if c["kind"] == "attend":
            s.cache.append(s.k, s.v, s.pos)
            return s.cache.attend(s.q, s.pos, out=s.out, work=s.work)
        if c["kind"] == "store":
            s.cache.append(s.k, s.v, s.pos, count=s.count)
            return s.cache.read(s.ko, s.vo, s.pos, count=s.count)
        if c["kind"] == "rope":
            return s.rope.apply(s.q, s.k, s.pos, out=s.outs)
        r = ops.logprobs(s.logits, s.tokens, top=c["top"], work=s.work)
        return {"lp": r.logprobs, "entropy": r.entropy, "ids": r.top_ids, "top": r.top_logprobs}
    if c["kind"] == "attend":
        _put(s.kn, s.kd, s.k, s.sid, s.pos)
        _put(s.vn, s.vd, s.v, s.sid, s.pos)
        return _attend(s)
    if c["kind"] == "store":
        _put(s.kn, s.kd, s.k, s.sid, s.pos, s.count)
        _put(s.vn, s.vd, s.v, s.sid, s.pos, s.count)
        return [_get(n, d, o, s.sid, s.pos, s.count) for n, d, o in ((s.kn, s.kd, s.ko), (s.vn, s.vd, s.vo))]
    if c["kind"] == "rope":
        return _rope(s)
    return _logprobs(s)


def _quantise(x):
    """(codes, scales) of blocks of 32: the value of largest magnitude (the first of equals) maps to code 0."""
    b = x.double().unflatten(-1, (-1, 32))
    a = b.abs()
    i = torch.arange(32, device=DEV)
    first = torch.where(a == a.amax(-1, keepdim=True), i, 32).amin(-1, keepdim=True)
    d = b.gather(-1, first) / -8
    inv = torch.where(d != 0, 1 / d, 0)
    return (b * inv + 8.5).trunc().clamp(0, 15).to(torch.uint8).flatten(-2), d[..., 0].float().half()


def _places(n, sid, pos, tokens, count):
    """The cache places of tokens [sequence, token], those of tokens behind a sequence's count outside."""
    j = torch.arange(tokens, device=DEV)
    p = pos.long()[:, None] + j
    return sid.expand_as(p), p, None if count is None else j < count[:, None]


def _put(codes, scales, x, sid, pos, count=None):
    n, d = _quantise(x)
    at, p, used = _places(codes, sid, pos, x.shape[1], count)
    if used is not None:
        n = torch.where(used[..., None, None], n, codes[at, :, p])
        d = torch.where(used[..., None, None], d, scales[at, :, p])
    codes[at, :, p] = n
    scales[at, :, p] = d


def _values(codes, scales):
    return ((codes.float() - 8).unflatten(-1, (-1, 32)) * scales.float()[..., None]).flatten(-2)


def _get(codes, scales, out, sid, pos, count):
    at, p, used = _places(codes, sid, pos, out.shape[1], count)
    x = _values(codes[at, :, p], scales[at, :, p]).to(out.dtype)
    return x if used is None else torch.where(used[..., None, None], x, out)


def _attend(s):
    c = s.case
    t, kv, g, dim = c["tokens"], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    n = max(_positions(c)) + t
    k, v = _values(s.kn[:, :, :n], s.kd[:, :, :n]), _values(s.vn[:, :, :n], s.vd[:, :, :n])
    q = s.q.float().unflatten(2, (kv, g)).permute(0, 2, 1, 3, 4).reshape(-1, kv, t * g, dim)
    x = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(dim)
    last = (s.pos[:, None] + torch.arange(t, device=DEV)).repeat_interleave(g, 1)
    x.masked_fill_((torch.arange(n, device=DEV) > last[..., None])[:, None], -math.inf)
    x = (x - x.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(x, v) / x.sum(-1, keepdim=True)
    return o.unflatten(2, (t, g)).permute(0, 2, 1, 3, 4).flatten(2, 3).to(s.q.dtype)


def _frequencies(c):
    """(radians a position of each pair, the factor of cos and sin)."""
    n = c["rot"]
    i = torch.arange(n // 2, dtype=torch.float64, device=DEV)
    th = c["base"] ** (-2 * i / n)
    if c["scaling"] == "linear":
        return th / c["factor"], 1.0
    if c["scaling"] == "yarn":
        lo, hi = (n * math.log(c["orig"] / (2 * math.pi * b)) / (2 * math.log(c["base"])) for b in (32.0, 1.0))
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), n - 1)
        r = ((i - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return th * (1 - r) + th / c["factor"] * r, 0.1 * math.log(c["factor"]) + 1.0
    return th, 1.0


def _rope(s):
    c = s.case
    th, m = _frequencies(c)
    a = s.pos.double()[:, None] * th
    cs, sn = (a.cos() * m).float()[:, None], (a.sin() * m).float()[:, None]
    out = []
    for x in (s.q, s.k):
        r, rest = x[..., :c["rot"]].float(), x[..., c["rot"]:]
        x0, x1 = r.chunk(2, -1) if c["half"] else (r[..., 0::2], r[..., 1::2])
        y0, y1 = x0 * cs - x1 * sn, x0 * sn + x1 * cs
        y = torch.cat([y0, y1], -1) if c["half"] else torch.stack([y0, y1], -1).flatten(-2)
        out.append(torch.cat([y.to(x.dtype), rest], -1))
    return out


def _logprobs(s):
    x = s.logits.float()
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    z = e.sum(-1)
    lz = z.log()
    lp = x.gather(-1, s.tokens.long()[:, None])[:, 0] - m[:, 0] - lz
    r = {"lp": lp, "entropy": lz - (e * (x - m)).sum(-1) / z, "ids": None, "top": None}
    if s.case["top"]:
        v, i = torch.sort(x, dim=-1, descending=True, stable=True)
        k = s.case["top"]
        r["ids"], r["top"] = i[:, :k].int(), v[:, :k] - m - lz[:, None]
    return r


# ---------------------------------------------------------------------------------------------- what a pass needs
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case.get("type")]
    if case["kind"] == "attend":
        pos, t, h, kv, dim = _positions(case), case["tokens"], case["heads"], case["kv_heads"], case["dim"]
        seen = sum((p + 1) * t + t * (t - 1) // 2 for p in pos)  # (token, position) pairs
        held = sum(p + t for p in pos)
        n = case["seqs"] * t
        return {"bytes": held * kv * dim * 9 // 8 + size * n * dim * (2 * h + 2 * kv), "flops": 4 * seen * h * dim}
    if case["kind"] == "store":
        n = sum(_counts(case)) * case["kv_heads"] * case["dim"]
        return {"bytes": n * 4 * size + n * 9 // 4, "flops": 6 * n}
    if case["kind"] == "rope":
        n = case["tokens"] * (case["heads"] + case["kv_heads"])
        return {"bytes": 2 * size * n * case["dim"] + 4 * case["tokens"], "flops": 3 * n * case["rot"]}
    n = case["rows"] * case["vocab"]
    return {"bytes": size * n + case["rows"] * (12 + 8 * case["top"]), "flops": 5 * n}


# ---------------------------------------------------------------------------------------------- 64-bit answers
def _stored(x):
    """What blocks of 32 values of x stand for in the cache, in float64."""
    x = x.to(torch.float64)
    b = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    order = torch.sort(b.abs(), dim=-1, descending=True, stable=True).indices
    step = torch.take_along_dim(b, order[..., :1], -1) * -0.125
    code = torch.floor(b * torch.where(step == 0, torch.zeros_like(step), step.reciprocal()) + 8.5).clamp(max=15.0)
    return (step.to(torch.float16).to(torch.float64) * (code - 8)).reshape(x.shape)


def exact(case, seed):
    d = _inputs(case, seed)
    if case["kind"] == "store":
        out = []
        for x in (d["k"], d["v"]):
            y = _stored(x)
            for i, n in enumerate(_counts(case)):
                y[i, n:] = 0.0
            out.append(y)
        return out
    if case["kind"] == "attend":
        t, h, kv = case["tokens"], case["heads"], case["kv_heads"]
        out = torch.empty((case["seqs"], t, h, case["dim"]), dtype=torch.float64, device=DEV)
        for s, p in enumerate(_positions(case)):
            for j in range(h):
                i = j // (h // kv)
                k, v = (_stored(torch.cat([d[x + "0"][s, :p, i].double(), d[x][s, :, i].double()])) for x in "kv")
                w = d["q"][s, :, j].double() @ k.T * case["dim"] ** -0.5
                w = torch.softmax(w + torch.full_like(w, -math.inf).triu(p + 1), -1)
                out[s, :, j] = w @ v
        return out
    if case["kind"] == "rope":
        n, out = case["rot"], []
        pair = np.arange(n // 2)
        w = np.power(case["base"], -pair / (n / 2.0))
        gain = 1.0
        if case["scaling"] == "linear":
            w = w / case["factor"]
        elif case["scaling"] == "yarn":
            at = [n / 2.0 * np.log(case["orig"] / (turns * 2.0 * np.pi)) / np.log(case["base"]) for turns in (32.0, 1.0)]
            a, b = max(np.floor(at[0]), 0.0), min(np.ceil(at[1]), n - 1.0)
            mix = np.clip((pair - a) / max(b - a, 0.001), 0.0, 1.0)
            w, gain = w * ((1.0 - mix) + mix / case["factor"]), 1.0 + np.log(case["factor"]) / 10.0
        turn = torch.polar(torch.tensor(gain, dtype=torch.float64, device=DEV), d["pos"].double()[:, None] * torch.tensor(w, device=DEV))
        for x in (d["q"], d["k"]):
            y = x.double()
            r = y[..., :n]
            z = torch.complex(r[..., :n // 2], r[..., n // 2:]) if case["half"] else torch.view_as_complex(r.reshape(*r.shape[:-1], -1, 2).contiguous())
            z = z * turn[:, None]
            y[..., :n] = torch.cat([z.real, z.imag], -1) if case["half"] else torch.view_as_real(z).flatten(-2)
            out.append(y)
        return out
    k = case["top"]
    r = {"lp": [], "entropy": [], "ids": [], "top": []}
    for i in range(0, case["rows"], 256):
        lp = torch.log_softmax(d["logits"][i:i + 256].double(), -1)
        r["lp"].append(lp[torch.arange(len(lp), device=DEV), d["tokens"][i:i + 256].long()])
        r["entropy"].append(-(lp.exp() * lp).sum(-1))
        if k:
            o = torch.sort(d["logits"][i:i + 256].double(), dim=-1, descending=True, stable=True).indices[:, :k]
            r["ids"].append(o.int())
            r["top"].append(torch.take_along_dim(lp, o, -1))
    return {name: torch.cat(x) if x else None for name, x in r.items()}
