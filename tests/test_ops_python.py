"""What the Python calls of the long-context operators refuse, on tensors in host memory that stand for the GPU's."""
import gc

import pytest
import torch

from zerollm_amd import _lib, ops


@pytest.fixture
def host(monkeypatch):
    """Host tensors pass for tensors on the library's GPU; a call that would reach the library fails the test."""
    monkeypatch.setattr(_lib, "DEVICE", -1)

    def reached(name, *a):
        raise AssertionError(f"{name} was called")

    monkeypatch.setattr(ops, "call", reached)


def bare(cls, **kw):
    x = object.__new__(cls)
    x.__dict__.update(closed=True, _h=None, _device=-1, **kw)  # (nothing to free)
    return x


def test_tensors_that_require_gradients(host):
    q = torch.zeros((1, 2, 4, 64), requires_grad=True)
    plain, pos = torch.zeros((1, 2, 4, 64)), torch.zeros(1, dtype=torch.int32)
    c = bare(ops.KVCacheQ4, n_head_kv=4, head_dim=64)
    r = bare(ops.Rope)
    r.closed = False
    for call, name in ((lambda: c.attend(q, pos), "q"), (lambda: c.attend(plain, pos, out=q), "out"), (lambda: c.append(q, plain, pos), "k"),
                       (lambda: c.append(plain, q, pos), "v"), (lambda: r.apply(q, None, pos), "q"), (lambda: r.apply(plain, q * 2, pos), "k"),
                       (lambda: ops.logprobs(q[0, 0]), "logits")):
        with pytest.raises(ValueError, match=f"^{name} requires a gradient"):
            call()
    with torch.no_grad():
        assert ops._rows(q, "q")[2] == (1, 2, 4, 64)
    assert ops._rows(q.detach(), "q")[2] == (1, 2, 4, 64)
    r.closed = True


def test_position_scaling_of_models_says_which():
    from zerollm_amd import model
    for kw in (dict(factor=4.0), dict(scaling=None, factor=4.0, orig_ctx=32768), dict(attn_factor=1.0)):
        with pytest.raises(ValueError, match="rope needs a scaling"):
            model.HipModel.load("none.gguf", rope=kw)
    assert model._ext("f16", dict(scaling="linear", factor=4.0)).rope.contents.factor == 4.0
    assert model._ext("f16", dict(scaling="none", factor=4.0)).rope.contents.scaling == 0
    assert model._ext("q4_0", dict()).kv_q4 == 1 and model._ext("f16", None) is None


def test_scales_that_float32_rounds_to_nothing(host):
    """0 means 1 / sqrt(head_dim) to the library."""
    q, pos = torch.zeros((1, 2, 4, 64)), torch.zeros(1, dtype=torch.int32)
    c = bare(ops.KVCacheQ4, n_head_kv=4, head_dim=64)
    for scale in (1e-50, 0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="scale must be positive"):
            c.attend(q, pos, scale=scale)


def test_handles_that_come_and_go_while_a_graph_is_captured(monkeypatch):
    """Nothing is allocated or freed then: making and closing one is refused, one that is collected is freed later."""
    done, capturing = [], [False]
    monkeypatch.setattr(ops, "call", lambda name, *a: done.append(name))
    monkeypatch.setattr(ops, "_capturing", lambda: capturing[0])
    r, c = ops.Rope(64), ops.KVCacheQ4(1, 2, 64, 100)
    assert done == ["zl_rope_create", "zl_kv4_create"]
    done.clear()
    capturing[0] = True
    for bad in (lambda: ops.Rope(64), lambda: ops.KVCacheQ4(1, 2, 64, 100), r.close, c.close):
        with pytest.raises(_lib.ZLError, match="a graph is being captured"):
            bad()
    del r
    gc.collect()
    assert done == [] and not c.closed
    capturing[0] = False
    c.close()
    c.close()
    assert done == ["zl_kv4_free"]
    with pytest.raises(_lib.ZLError, match="cache is closed"):
        c.work_bytes(1, 1, 2)
    done.clear()
    r = ops.Rope(64)
    assert done == ["zl_rope_free", "zl_rope_create"]
    del r
    gc.collect()
    assert done[2:] == ["zl_rope_free"]


def test_handles_of_another_gpu(monkeypatch):
    """model.init of another GPU moves the calls' tensors and streams there."""
    monkeypatch.setattr(ops, "call", lambda name, *a: None)
    r, c = ops.Rope(64), ops.KVCacheQ4(1, 2, 64, 100)
    c.work_bytes(1, 1, 2)
    q, pos = torch.zeros((1, 2, 2, 64)), torch.zeros(1, dtype=torch.int32)
    monkeypatch.setattr(_lib, "DEVICE", -1)  # (host tensors stand for that GPU's)
    monkeypatch.setattr(ops, "_stream", lambda: None)
    for bad in (lambda: c.attend(q, pos), lambda: c.append(q, q, pos), lambda: c.read(q, q, pos), lambda: c.work_bytes(1, 1, 2), lambda: r.apply(q, None, pos)):
        with pytest.raises(_lib.ZLError, match="is on GPU 0, the library on GPU -1"):
            bad()
    c.close()
    r.close()
