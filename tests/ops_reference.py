"""Plain 64-bit forms of the long-context operators, for their tests."""
import math

import numpy as np
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(t):
    """The largest relative error of one rounding to the type."""
    return torch.finfo(t).eps / 2


def quantise(x):
    """(codes, float64 scales after their rounding to f16) of float64 [..., dim] values in blocks of 32: x / d + 8.5
    truncated, d = -1/8 of the value of largest magnitude, the first of equals. A block with a value that is not finite or
    above 65504 stands for NaN."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        bad = ~(np.abs(b) <= 65504).all(-1)
        b = np.where(bad[..., None], 0.0, b)
        first = np.abs(b).argmax(-1)
        d = np.take_along_axis(b, first[..., None], -1)[..., 0] / -8.0
        inv = np.where(d != 0, 1.0 / d, 0.0)
        n = np.clip(np.trunc(b * inv[..., None] + 8.5), 0, 15)
        d = d.astype(np.float32).astype(np.float16).astype(np.float64)
    return n.reshape(x.shape), np.where(bad, np.nan, d)


def stored(x):
    """What the cache holds for float64 values: scale times (code - 8)."""
    n, d = quantise(x)
    return (n - 8) * np.repeat(d, 32, -1)


def attention(q, k, v, last, scale):
    """q [rows, dim] at positions last [rows] over k, v [positions, dim], all float64. Returns the outputs and, for each row,
    the largest sum of |q k| scale over the positions it sees (what the scores' roundings are relative to)."""
    out, size = np.zeros_like(q), np.zeros(len(q))
    for r, p in enumerate(last):
        if p < 0:
            continue
        with np.errstate(all="ignore"):
            s = k[:p + 1] @ q[r] * scale
            e = np.exp(s - s.max())
            out[r] = (e @ v[:p + 1]) / e.sum()
            size[r] = (np.abs(k[:p + 1]) @ np.abs(q[r])).max() * scale
    return out, size


def attention_bound(size, dim, vmax, out, t):
    """How far an output may be from float64's: scores summed in f32 are off by at most (dim + 8) 2^-24 size (the products of
    a block and its scale, the blocks' sum, the factor), which moves a weight relative to the sum of them by twice that; the
    exponential, the weight times its value's scale in two f16 parts (2^-22, and 2^-25 absolute below the weight's own
    f16 range, at a code of 8), and the sums of a span, chunk and row in f32 (64, 8, 4 and some 64 terms, errors that add up
    like a random walk of at most 256 steps: 2^-20) come to 2^-18 of the largest value; the output's own rounding on top.
    With 16-bit outputs that are rounded further (bf16) the weights have one f16 part: 2^-11 of each."""
    b = vmax * (2 * (dim + 8) * 2.0 ** -24 * size[:, None] + 2.0 ** -18 + (2.0 ** -11 if t == torch.bfloat16 else 0.0)) + 2.0 ** -20
    return b + half_step(t) * np.abs(out)


def angles(n_rot, base, scaling=None, factor=1.0, orig=0, fast=32.0, slow=1.0, gain=None, freq=None):
    """(radians per position of each pair, factor of cos and sin), in float64."""
    th = [base ** (-2.0 * i / n_rot) / (1.0 if freq is None else float(freq[i])) for i in range(n_rot // 2)]
    if scaling == "linear":
        return np.array(th) / factor, 1.0
    if scaling == "yarn":
        def pair(b):
            return n_rot * math.log(orig / (2 * math.pi * b)) / (2 * math.log(base))

        low, high = max(math.floor(pair(fast)), 0), min(math.ceil(pair(slow)), n_rot - 1)
        mix = [min(1.0, max(0.0, (i - low) / max(high - low, 0.001))) for i in range(n_rot // 2)]
        return np.array([t * (1 - m) + t / factor * m for t, m in zip(th, mix)]), gain or 0.1 * math.log(factor) + 1.0
    return np.array(th), 1.0


def rotate(x, pos, th, gain, half):
    """x [..., token, head, dim] float64 rotated to pos [..., token]."""
    n = 2 * len(th)
    a = np.asarray(pos, np.float64)[..., None] * th
    c, s = np.cos(a)[..., None, :] * gain, np.sin(a)[..., None, :] * gain
    y = x.copy()
    i0, i1 = (slice(0, n // 2), slice(n // 2, n)) if half else (slice(0, n, 2), slice(1, n, 2))
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i0] * s + x[..., i1] * c
    return y


def logprobs(x, tokens, top):
    """(log probabilities of tokens, entropies, ids, log probabilities of the top alternatives) of float64 rows."""
    with np.errstate(all="ignore"):
        m = x.max(-1, keepdims=True)  # NaN wins
        e = np.exp(x - m)
        z = e.sum(-1)
        lp = x - m - np.log(z)[:, None]
        ent = np.log(z) - np.where(e > 0, e * (x - m), e).sum(-1) / z
    key = np.where(np.isnan(x), -np.inf, x)
    ids = np.lexsort((np.broadcast_to(np.arange(x.shape[1]), x.shape), np.isnan(x), -key), axis=-1)[:, :top]
    ok = (tokens >= 0) & (tokens < x.shape[1])
    given = np.where(ok, lp[np.arange(len(x)), np.where(ok, tokens, 0)], np.nan)
    return given, ent, ids, np.take_along_axis(lp, ids, -1)
