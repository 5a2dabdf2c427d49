"""Operators of long contexts on device tensors: a KV cache held in 4 bits with the attention over it, rotary positions
scaled beyond the trained context, log probabilities of logits rows (the C ABI's zl_kv4_*, zl_rope_*, zl_logprobs).

Tensors are torch's (this module imports no torch of its own: it takes any tensor with torch's interface), on the library's
GPU, float32, float16 or bfloat16, with any strides as long as the values of a head (of a logits row) are contiguous. Rows of
several sequences are [sequence, token, head, dim], or [sequence, head, dim] for one token each. Positions, counts and slots
are int32 tensors on the GPU, one entry per sequence, read when the work runs. Calls are enqueued on torch's current stream
and return at once; with `out` and `work` given they allocate nothing and may be captured into a graph. They have no gradients: a
tensor that requires one is refused while gradients are recorded. Wrong shapes, types or places raise ValueError, what the library
refuses ZLError.
"""
from __future__ import annotations

import ctypes as C
import sys
from dataclasses import dataclass

import numpy as np

from . import _lib
from ._lib import call

_TYPES = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 30}
_type_of = {}  # by torch's type objects, filled as they come: a call on few rows is as long as its checks


def _elsewhere(x, name):
    return ValueError(f"{name} must be a tensor on GPU {_lib.DEVICE} (got {getattr(x, 'device', None)})")


def _place(x, name):
    if not hasattr(x, "get_device") or x.get_device() != _lib.DEVICE:  # (-1 for a tensor in host memory)
        raise _elsewhere(x, name)


def _type(x, name):
    try:
        if x.get_device() == _lib.DEVICE:
            return _type_of[x.dtype]
    except (AttributeError, KeyError):
        pass
    _place(x, name)
    t = _TYPES.get(str(x.dtype))
    if t is None:
        raise ValueError(f"{name} must be float32, float16 or bfloat16 (got {x.dtype})")
    _type_of[x.dtype] = t
    return t


def _no_gradient(x, name):
    if x.requires_grad and _torch().is_grad_enabled():
        raise ValueError(f"{name} requires a gradient, which these operators do not give: detach it, or call under torch.no_grad()")


def _ints(x, n, name):
    if x is None:
        return None
    _place(x, name)
    if x.dtype != _torch().int32 or x.shape != (n,) or not x.is_contiguous():
        raise ValueError(f"{name} must be {n} contiguous int32 values (got {x.dtype} {tuple(x.shape)})")
    return x.data_ptr()


def _rows(x, name, shape=None, type_=None, written=False):
    """(zl_rows, type, shape as (sequence, token, head, dim)) of a tensor."""
    t = _type(x, name)
    _no_gradient(x, name)
    s = tuple(x.shape)
    if len(s) == 4:
        a, b, c, d = x.stride()
    elif len(s) == 3:
        a, c, d = x.stride()
        b, s = 0, (s[0], 1, s[1], s[2])
    else:
        raise ValueError(f"{name} must be [sequence, token, head, dim] or [sequence, head, dim] (got {s})")
    if d != 1 and s[3] > 1:
        raise ValueError(f"the values of a head of {name} must be contiguous (stride {d})")
    if shape is not None and s != shape:
        raise ValueError(f"{name} must be {shape} (got {s})")
    if type_ is not None and t != type_:
        raise ValueError(f"{name} must have the type of the other rows (got {x.dtype})")
    if written and ((a == 0 and s[0] > 1) or (b == 0 and s[1] > 1) or (c == 0 and s[2] > 1)):
        raise ValueError(f"{name} is written, so its rows must not share memory")
    return _lib.zl_rows(x.data_ptr(), a, b, c), t, s


def _batch(n_seq, n_tok, pos, count, slot=None):
    if pos is None:
        raise ValueError("positions missing")
    return _lib.zl_batch(n_seq, n_tok, _ints(pos, n_seq, "pos"), count if count is None else _ints(count, n_seq, "count"),
                         slot if slot is None else _ints(slot, n_seq, "slot"))


def _torch():
    t = sys.modules.get("torch")
    if t is None:
        raise ValueError("these calls take torch tensors: import torch first")
    return t


def _stream():
    return _torch().cuda.current_stream(_lib.DEVICE).cuda_stream


def _work(work, nbytes, like):
    """A work space of at least nbytes: the caller's, or one of torch's for this call."""
    if work is None:
        return _torch().empty(nbytes, dtype=_torch().uint8, device=like.device)
    _place(work, "work")
    if not work.is_contiguous() or work.numel() * work.element_size() < nbytes:
        raise ValueError(f"work must be contiguous, {nbytes} bytes or more")
    return work


def _capturing():
    t = sys.modules.get("torch")
    return t is not None and t.cuda.is_initialized() and t.cuda.is_current_stream_capturing()


class _Handle:
    """An object of the library's. Making and freeing one allocates and waits for the GPU, which would break a graph that is being
    captured on the current stream: refused there; an object that goes in the meantime (a garbage collection) is freed later, when
    the next one is made or goes."""

    _gone = []  # of those: (entry point, handle)

    def _make(self, name, *args):
        if _capturing():
            raise _lib.ZLError(5, f"{name}: a graph is being captured")
        self._free_later()
        self._h = C.c_void_p()
        call(name, *args, C.byref(self._h))
        self.closed, self._device = False, _lib.DEVICE

    def _handle(self):
        if self.closed:
            raise _lib.ZLError(5, f"{self._what} is closed")
        if self._device != _lib.DEVICE:  # (its memory is there, the call's tensors and stream here)
            raise _lib.ZLError(5, f"{self._what} is on GPU {self._device}, the library on GPU {_lib.DEVICE} by now")
        return self._h

    @classmethod
    def _free_later(cls):
        while cls._gone:
            call(*cls._gone.pop())

    def close(self):
        """Release it once the GPU is done with it (idempotent)."""
        if self.closed:
            return
        if _capturing():
            raise _lib.ZLError(5, f"{self._free}: a graph is being captured")
        self.closed = True
        call(self._free, self._h)

    def __del__(self):
        try:
            if not _capturing():
                self.close()
                self._free_later()
            elif not self.closed:
                self.closed = True
                self._gone.append((self._free, self._h))
        except Exception:
            pass


class KVCacheQ4(_Handle):
    """A KV cache of n_slot sequences of up to `capacity` positions, held as Q4_0 blocks: 1.125 bytes per (position, KV head,
    dimension) for key and value together, where float16 takes 4."""

    _what, _free, closed = "cache", "zl_kv4_free", True

    def __init__(self, n_slot: int, n_head_kv: int, head_dim: int, capacity: int):
        self._make("zl_kv4_create", int(n_slot), int(n_head_kv), int(head_dim), int(capacity))
        self.n_slot, self.n_head_kv, self.head_dim, self.capacity = int(n_slot), int(n_head_kv), int(head_dim), int(capacity)
        self._sized = None, 0  # the last queries' shape and its work space

    @property
    def nbytes(self) -> int:
        n = C.c_int64()
        call("zl_kv4_bytes", self._handle(), C.byref(n))
        return n.value

    def _kv(self, k, v, written):
        kr, t, s = _rows(k, "k", written=written)
        if s[2:] != (self.n_head_kv, self.head_dim):
            raise ValueError(f"k must hold {self.n_head_kv} heads of {self.head_dim} values (got {s[2:]})")
        return kr, _rows(v, "v", s, t, written)[0], t, s

    def append(self, k, v, pos, count=None, slot=None):
        """Put k and v at positions pos[s], pos[s] + 1, ... of each sequence s (of its slot: s itself without `slot`); only
        the first count[s] tokens where `count` is given."""
        kr, vr, t, s = self._kv(k, v, False)
        call("zl_kv4_append", self._handle(), _batch(s[0], s[1], pos, count, slot), t, kr, vr, _stream())

    def read(self, k, v, pos, count=None, slot=None):
        """Fill k and v with what the cache holds at those positions; returns (k, v)."""
        kr, vr, t, s = self._kv(k, v, True)
        call("zl_kv4_read", self._handle(), _batch(s[0], s[1], pos, count, slot), t, kr, vr, _stream())
        return k, v

    def work_bytes(self, n_seq: int, n_tok: int, n_head: int) -> int:
        n = C.c_int64()
        call("zl_kv4_attention_work", self._handle(), int(n_seq), int(n_tok), int(n_head), C.byref(n))
        return n.value

    def attend(self, q, pos, count=None, slot=None, scale=None, out=None, work=None):
        """Causal attention of the queries over the cache: token j of sequence s sees positions 0 .. pos[s] + j, which must
        have been appended, its own key and value among them. scale None: 1/sqrt(head_dim). A token at a negative position
        gets zeros, one past the capacity or of a slot that does not exist NaN. Returns `out` (may be q itself)."""
        qr, t, s = _rows(q, "q")
        if s[3] != self.head_dim:
            raise ValueError(f"q must have heads of {self.head_dim} values (got {s[3]})")
        if scale is not None and not (scale > 0 and C.c_float(scale).value > 0):
            raise ValueError(f"scale must be positive in float32 (got {scale})")
        b = _batch(s[0], s[1], pos, count, slot)
        if out is None:
            out = _torch().empty(tuple(q.shape), dtype=q.dtype, device=q.device)
        o = _rows(out, "out", s, t, True)[0]
        sized = self._sized
        if s != sized[0]:
            sized = self._sized = s, self.work_bytes(s[0], s[1], s[2])
        w = _work(work, sized[1], q)
        call("zl_kv4_attention", self._handle(), b, t, qr, s[2], scale or 0.0, o, w.data_ptr(), w.numel() * w.element_size(), _stream())
        return out


SCALINGS = {None: 0, "none": 0, "linear": 1, "yarn": 2}


def rope_opts(n_rot=0, neox=True, base=10000.0, scaling=None, factor=1.0, orig_ctx=0, beta_fast=0.0, beta_slow=0.0,
              attn_factor=0.0, freq_factors=None):
    """zl_rope_opts from names (the meanings are Rope's)."""
    if scaling not in SCALINGS:
        raise ValueError(f'scaling must be none, linear or yarn (got "{scaling}")')
    ff = None
    if freq_factors is not None:
        ff = np.ascontiguousarray(freq_factors, np.float32)
        if ff.shape != (n_rot // 2,):
            raise ValueError(f"freq_factors must be {n_rot // 2} values (got {ff.shape})")
    o = _lib.zl_rope_opts(n_rot=int(n_rot), neox=1 if neox else 0, base=float(base), scaling=SCALINGS[scaling],
                          orig_ctx=int(orig_ctx), factor=float(factor), beta_fast=float(beta_fast or 0.0),
                          beta_slow=float(beta_slow or 0.0), attn_factor=float(attn_factor or 0.0),
                          freq_factors=_lib.ptr(ff, C.c_float) if ff is not None else None)
    o._keep = ff
    return o


class Rope(_Handle):
    """Rotary positions of the first n_rot values of a head: pairs (i, i + n_rot/2) (neox) or (2i, 2i + 1), by
    pos * base^(-2i/n_rot) / freq_factors[i] radians. scaling "linear": angles divided by factor; "yarn": by parts, between
    pairs that turn beta_fast (32) and beta_slow (1) times within orig_ctx positions, and everything times attn_factor
    (0.1 ln factor + 1)."""

    _what, _free, closed = "rope", "zl_rope_free", True

    def __init__(self, n_rot, neox=True, base=10000.0, scaling=None, factor=1.0, orig_ctx=0, beta_fast=0.0, beta_slow=0.0,
                 attn_factor=0.0, freq_factors=None):
        o = rope_opts(n_rot, neox, base, scaling, factor, orig_ctx, beta_fast, beta_slow, attn_factor, freq_factors)
        self._make("zl_rope_create", C.byref(o))
        self.n_rot = int(n_rot)

    def apply(self, q, k, pos, count=None, out=None):
        """q and k (or None) rotated to positions pos[s], pos[s] + 1, ... of each sequence, in one launch. out: (q', k'), which
        may be q and k themselves; new tensors without it. Returns (q', k')."""
        handle = self._handle()
        qr, t, s = _rows(q, "q")
        if out is None:
            out = tuple(None if x is None else _torch().empty(tuple(x.shape), dtype=x.dtype, device=x.device) for x in (q, k))
        qo = _rows(out[0], "out[0]", s, t, True)[0]
        kr = ko = None
        nk = 0
        if k is not None:
            nk = k.shape[-2] if len(k.shape) >= 3 else 0
            ks = (s[0], s[1], nk, s[3])
            kr, ko = _rows(k, "k", ks, t)[0], _rows(out[1], "out[1]", ks, t, True)[0]
        call("zl_rope_apply", handle, _batch(s[0], s[1], pos, count), t, s[3], qr, qo, s[2], kr, ko, nk, _stream())
        return out


@dataclass
class LogProbs:
    """Of each row: the log probability of its given token (None without tokens), the entropy in nats, and the ids and log
    probabilities of the largest logits, largest first, the lowest id first among equals (None with top 0)."""
    logprobs: object
    entropy: object
    top_ids: object
    top_logprobs: object


def logprobs_work_bytes(rows: int, vocab: int, top: int = 0) -> int:
    n = C.c_int64()
    call("zl_logprobs_work", int(rows), int(vocab), int(top), C.byref(n))
    return n.value


def logprobs(logits, tokens=None, top: int = 0, out=None, work=None) -> LogProbs:
    """LogProbs of logits rows [rows, vocab] (any row stride of at least vocab). tokens: int32 [rows]; an id outside the vocabulary gives NaN.
    top: 0 to 64 alternatives. Logits of -inf have probability 0; a row with NaN or +inf, or with nothing above -inf, is NaN."""
    t = _type(logits, "logits")
    _no_gradient(logits, "logits")
    if len(logits.shape) != 2 or (logits.shape[1] > 1 and logits.stride(1) != 1):
        raise ValueError("logits must be [rows, vocab] with contiguous rows")
    rows, vocab = logits.shape
    tok = _ints(tokens, rows, "tokens")
    torch = _torch()
    n = C.c_int64()
    call("zl_logprobs_work", rows, vocab, int(top), C.byref(n))
    if out is None:
        def new(shape, dtype):
            return torch.empty(shape, dtype=dtype, device=logits.device)

        out = LogProbs(new(rows, torch.float32) if tokens is not None else None, new(rows, torch.float32),
                       new((rows, top), torch.int32) if top else None, new((rows, top), torch.float32) if top else None)
    p = []
    for x, shape, dtype in ((out.logprobs, (rows,), torch.float32), (out.entropy, (rows,), torch.float32),
                            (out.top_ids, (rows, top), torch.int32), (out.top_logprobs, (rows, top), torch.float32)):
        if x is None:
            p.append(None)
            continue
        _place(x, "out")
        if tuple(x.shape) != shape or x.dtype != dtype or not x.is_contiguous():
            raise ValueError(f"out must be contiguous {dtype} {shape} (got {x.dtype} {tuple(x.shape)})")
        p.append(x.data_ptr())
    w = _work(work, n.value, logits)
    call("zl_logprobs", logits.data_ptr(), t, logits.stride(0) if rows > 1 else vocab, rows, vocab, tok, int(top), *p,
         w.data_ptr(), w.numel() * w.element_size(), _stream())
    return out
