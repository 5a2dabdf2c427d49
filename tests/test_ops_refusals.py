"""What the long-context entry points refuse before they touch a GPU."""
import ctypes as C
import math

import numpy as np
import pytest

from ops_reference import angles, logprobs, quantise, stored
from oracle import oracle as O
from zerollm_amd import _lib, ops
from zerollm_amd._lib import ZLError, call


@pytest.mark.parametrize("args,msg", [((1, 2, 96, 100), "head_dim must be 64, 128 or 256"), ((0, 2, 64, 100), "bad slot count"),
                                      ((1, 0, 64, 100), "bad slot count"), ((1, 2, 64, 0), "bad slot count"),
                                      ((1, 2, 64, 2 ** 31), "bad slot count"), ((70000, 2, 64, 10), "bad slot count")])
def test_cache_shapes(args, msg):
    with pytest.raises(ZLError, match=msg):
        ops.KVCacheQ4(*args)


@pytest.mark.parametrize("kw,msg", [(dict(n_rot=7), "n_rot must be even"), (dict(n_rot=0), "n_rot must be even"), (dict(n_rot=258), "n_rot must be even"),
                                    (dict(base=0.0), "base must be positive"), (dict(base=math.inf), "base must be positive"),
                                    (dict(base=math.nan), "base must be positive"), (dict(scaling="linear", factor=0.5), "at least 1"),
                                    (dict(scaling="linear", factor=math.nan), "at least 1"),
                                    (dict(scaling="yarn", factor=2.0), "trained context"),
                                    (dict(scaling="yarn", factor=2.0, orig_ctx=64, base=1.0), "base above 1"),
                                    (dict(scaling="yarn", factor=2.0, orig_ctx=64, beta_fast=1.0, beta_slow=2.0), "beta_fast"),
                                    (dict(scaling="yarn", factor=2.0, orig_ctx=64, attn_factor=-1.0), "attention factor"),
                                    (dict(freq_factors=np.zeros(32)), "frequency factors must be positive")])
def test_rope_options(kw, msg):
    with pytest.raises(ZLError, match=msg):
        ops.Rope(**{"n_rot": 64, **kw})


def test_rope_names():
    with pytest.raises(ValueError, match="none, linear or yarn"):
        ops.Rope(64, scaling="ntk")
    with pytest.raises(ValueError, match="32 values"):
        ops.Rope(64, freq_factors=np.ones(31))


def test_null_arguments_and_bad_types():
    b = _lib.zl_batch(1, 1, None, None, None)
    r = _lib.zl_rows(16, 0, 0, 0)
    for name, args in (("zl_kv4_append", (None, b, 0, r, r, None)), ("zl_kv4_read", (None, b, 0, r, r, None)),
                       ("zl_kv4_attention", (None, b, 0, r, 1, 0.0, r, None, 0, None)),
                       ("zl_rope_apply", (None, b, 0, 64, r, r, 1, None, None, 0, None)),
                       ("zl_model_logprobs", (None, 0, 1, None, 0, None, None, None, None))):
        with pytest.raises(ZLError, match="null argument"):
            call(name, *args)
    call("zl_kv4_free", None)
    call("zl_rope_free", None)
    with pytest.raises(ZLError, match="must be F32, F16 or BF16"):
        call("zl_logprobs", None, 8, 10, 0, 10, None, 0, None, None, None, None, None, 0, None)


@pytest.mark.parametrize("args,msg", [((1, 10, 11), "n_top must be"), ((1, 100, 65), "n_top must be"), ((-1, 10, 1), "bad row count"), ((1 << 24, 10, 1), "bad row count"),
                                      ((1, 0, 0), "bad row count")])
def test_logprobs_sizes(args, msg):
    with pytest.raises(ZLError, match=msg):
        call("zl_logprobs_work", *args, C.byref(C.c_int64()))


def test_logprobs_arguments():
    call("zl_logprobs", None, 0, 10, 0, 10, None, 0, None, None, None, None, None, 0, None)  # no rows
    for args, msg in (((None, 0, 10, 1, 10, None, 0, None, None, None, None, None, 0, None), "logits missing"),
                      ((16, 0, 9, 1, 10, None, 0, None, None, None, None, None, 0, None), "row stride"),
                      ((17, 0, 10, 1, 10, None, 0, None, None, None, None, None, 0, None), "not aligned"),
                      ((16, 0, 10, 1, 10, None, 0, 16, None, None, None, None, 0, None), "need the tokens"),
                      ((16, 0, 10, 1, 10, None, 0, None, None, None, None, None, 0, None), "work space of")):
        with pytest.raises(ZLError, match=msg):
            call("zl_logprobs", *args)


# ---------------------------------------------------------------------------------------------- the plain forms themselves
def test_the_plain_quantiser_is_the_oracles():
    x = np.random.default_rng(1).normal(0, 1, (50, 64)).astype(np.float32)
    x[3, :4] = 2.0, -2.0, 2.0, -2.0
    x[4, 32:] = 0.0
    want = O.dequant(2, O.quantize_q4_0(x.reshape(-1)), 50, 64)
    assert (stored(x.astype(np.float64)) == want).all()
    n, d = quantise(x.astype(np.float64))
    assert n.min() >= 0 and n.max() <= 15 and d.shape == (50, 2)


def test_the_plain_yarn_ramp_known_answer():
    """Pair i of 64 with base 10^6 turns 32768 / (2 pi 10^(6 i / 64)) times in 32768 positions: 32 times at i = 23.6, once at
    i = 39.6."""
    th, m = angles(128, 1e6, "yarn", 4.0, 32768)
    plain = 1e6 ** (-np.arange(64) / 64)
    assert np.allclose(th[:24], plain[:24], rtol=1e-15) and np.allclose(th[40:], plain[40:] / 4, rtol=1e-15)
    assert np.allclose(th[24], plain[24] * (1 - 1 / 17 * 0.75), rtol=1e-14) and m == 0.1 * math.log(4) + 1


def test_the_plain_logprobs_known_answers():
    x = np.log(np.array([[0.5, 0.25, 0.25, 0.0]] * 2) + [[0], [1e-300]])
    lp, h, ids, top = logprobs(x, np.array([1, 3]), 3)
    assert np.allclose(lp[0], math.log(0.25)) and np.allclose(h, 1.5 * math.log(2)) and ids.tolist() == [[0, 1, 2]] * 2
    assert np.allclose(top[0], np.log([0.5, 0.25, 0.25]))
