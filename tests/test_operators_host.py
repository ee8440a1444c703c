"""Refusals and host logic of the training and serving operators (no kernel launches)."""

import ctypes
import pickle
import math

import pytest
import torch

import mamba3_b200 as m
from mamba3_b200 import _lib


def test_entry_points_reject_bad_arguments():
    L = _lib.lib()
    for fn in (L.m3b_gated_ffn_fwd, L.m3b_gated_ffn_bwd, L.m3b_linear_xent_fwd, L.m3b_linear_xent_bwd, L.m3b_grad_clip):
        assert fn(None, None, 0, None) == 1 and b"null" in L.m3b_last_error()
    a = _lib.GatedFfnArgs(4, 64, 0, 64, 64, 128, 1)
    assert L.m3b_gated_ffn_fwd(ctypes.byref(a), None, 0, None) == 1 and b"null" in L.m3b_last_error()
    assert L.m3b_gated_ffn_act_bytes(ctypes.byref(a)) == 4 * 128 * 2
    assert L.m3b_gated_ffn_gu_bytes(ctypes.byref(a)) == 256 * 128 * 6
    for bad in (_lib.GatedFfnArgs(-1, 64, 0, 64, 64, 128, 1), _lib.GatedFfnArgs(4, 64, 0, 64, 0, 128, 1),
                _lib.GatedFfnArgs(4, 64, 0, 64, 64, 128, 9)):
        assert L.m3b_gated_ffn_fwd(ctypes.byref(bad), None, 0, None) == 1
        assert L.m3b_gated_ffn_fwd_workspace(ctypes.byref(bad)) == 0
    x = _lib.LinearXentArgs(4, 64, -100, 64, 1000, 1, 1)
    assert L.m3b_linear_xent_fwd(ctypes.byref(x), None, 0, None) == 1 and b"null" in L.m3b_last_error()
    assert L.m3b_linear_xent_saved(ctypes.byref(x)) >= 4 * 64 * 4 + 4 * 1000 * 4  # few rows: in fp32, and the logits
    x.rows = 40
    assert L.m3b_linear_xent_saved(ctypes.byref(x)) >= 256 * 64 * 2 + 3 * 256 * 4
    x.reduction = 3
    assert L.m3b_linear_xent_fwd(ctypes.byref(x), None, 0, None) == 1 and b"reduction" in L.m3b_last_error()
    c = _lib.GradClipArgs(3)
    assert L.m3b_grad_clip(ctypes.byref(c), None, 0, None) == 1


def test_short_workspace_is_refused():
    """Checked before any launch, so plain addresses stand in for device pointers."""
    L = _lib.lib()
    buf = ctypes.create_string_buffer(1 << 16)
    p = (ctypes.addressof(buf) + 255) // 256 * 256
    a = _lib.GatedFfnArgs(40, 63, 0, 63, 63, 128, 1, 1.0, p, p, p, p, None, None, None, None, p, None, p)
    need = L.m3b_gated_ffn_fwd_workspace(ctypes.byref(a))
    assert need >= 40 * 64 * 2 + 2 * 128 * 64 * 2  # x, w_gate and w_up laid out with rows of 64
    assert L.m3b_gated_ffn_fwd(ctypes.byref(a), p, need - 1, None) == 6
    assert L.m3b_gated_ffn_fwd(ctypes.byref(a), p + 4, need, None) == 4
    a.saved_act = p + 2
    assert L.m3b_gated_ffn_fwd(ctypes.byref(a), p, need, None) == 4
    x = _lib.LinearXentArgs(4, 64, -100, 64, 1000, 1, 1, p, p, p, p, p)
    assert L.m3b_linear_xent_fwd(ctypes.byref(x), None, 0, None) == 6
    need = L.m3b_linear_xent_fwd_workspace(ctypes.byref(x))
    assert L.m3b_linear_xent_fwd(ctypes.byref(x), p, need - 1, None) == 6
    x.dloss = x.dhidden = x.dweight = p
    need = L.m3b_linear_xent_bwd_workspace(ctypes.byref(x))
    assert need >= 4 * 64 * 4 and L.m3b_linear_xent_bwd(ctypes.byref(x), p, need - 1, None) == 6
    one = (ctypes.c_void_p * 1)(p)
    num, dt = (ctypes.c_int64 * 1)(10), (ctypes.c_int32 * 1)(0)
    c = _lib.GradClipArgs(1, ctypes.addressof(one), ctypes.addressof(one), ctypes.addressof(num), ctypes.addressof(dt),
                          ctypes.addressof(dt), 2, 1.0, p)
    assert L.m3b_grad_clip(ctypes.byref(c), None, 0, None) == 6
    c.norm_type = 1
    assert L.m3b_grad_clip(ctypes.byref(c), p, 1 << 12, None) == 1 and b"norm_type" in L.m3b_last_error()


@pytest.mark.parametrize("dtype,code", [(torch.float32, 0), (torch.bfloat16, 1), (torch.float16, 2)])
def test_saved_sizes_agree_with_the_library(dtype, code):
    L = _lib.lib()
    for rows, f in ((0, 8), (1, 1), (7, 33), (8, 64), (9, 64), (256, 2112), (257, 100)):
        a = _lib.GatedFfnArgs(rows, 64, 0, 64, 64, f, code)
        want = L.m3b_gated_ffn_act_bytes(ctypes.byref(a)), L.m3b_gated_ffn_gu_bytes(ctypes.byref(a))
        assert _lib.ffn_saved_bytes(torch.empty(rows, 64, dtype=dtype), f) == want
        for d in (64, 33):
            x = _lib.LinearXentArgs(rows, d, -100, d, 1003, code, 1)
            assert _lib.xent_saved_bytes(torch.empty(rows, d, dtype=dtype), 1003) == L.m3b_linear_xent_saved(ctypes.byref(x))


def test_sizes_past_the_limits_are_refused():
    L = _lib.lib()
    for rows, d, f in ((1 << 31, 64, 64), (4, 1 << 22, 64), (4, 64, 1 << 22)):
        a = _lib.GatedFfnArgs(rows, d, 0, d, d, f, 1)
        assert L.m3b_gated_ffn_fwd(ctypes.byref(a), None, 0, None) == 1 and b"limits" in L.m3b_last_error()
    x = _lib.LinearXentArgs(1 << 31, 64, -100, 64, 1000, 1, 1)
    assert L.m3b_linear_xent_fwd(ctypes.byref(x), None, 0, None) == 1 and b"limits" in L.m3b_last_error()


def test_cpu_tensors_raise():
    x, w = torch.randn(3, 8), torch.randn(16, 8)
    with pytest.raises(m.M3bError, match="CUDA"):
        m.gated_ffn(x, w, w, w.t())
    with pytest.raises(m.M3bError, match="CUDA"):
        m.linear_cross_entropy(x, w, torch.zeros(3, dtype=torch.long))
    with pytest.raises(m.M3bError, match="CUDA"):
        m.clip_grads([x], 1.0)


class _Cuda(torch.Tensor):
    """A CPU tensor that says it is on a GPU: the checks run, and refuse before any launch."""

    @staticmethod
    def __new__(cls, t):
        return torch.Tensor._make_subclass(cls, t)

    is_cuda = property(lambda self: True)
    device = property(lambda self: torch.device("cuda", 0))


def fake(*shape, dtype=torch.float32):
    return _Cuda(torch.zeros(*shape, dtype=dtype))


@pytest.mark.parametrize("change,error", [
    (dict(w_up=(16, 9)), ValueError), (dict(w_down=(16, 8)), ValueError), (dict(x=(3, 9)), ValueError),
    (dict(b_gate=(16,)), ValueError), (dict(b_gate=(16,), b_up=(8,)), ValueError), (dict(b_down=(16,)), ValueError),
    (dict(residual=(1, 8)), ValueError), (dict(w_gate=(16,)), ValueError)])
def test_ffn_refuses_shapes(change, error):
    shapes = dict(x=(3, 8), w_gate=(16, 8), w_up=(16, 8), w_down=(8, 16))
    t = {k: fake(*s) for k, s in {**shapes, **change}.items()}
    with pytest.raises(error):
        m.gated_ffn(t.pop("x"), t.pop("w_gate"), t.pop("w_up"), t.pop("w_down"), **t)


def test_ffn_refuses_types():
    t = [fake(3, 8), fake(16, 8), fake(16, 8, dtype=torch.bfloat16), fake(8, 16)]
    with pytest.raises(m.M3bError, match="one dtype"):
        m.gated_ffn(*t)
    with pytest.raises(m.M3bError, match="unsupported dtype"):
        m.gated_ffn(*[fake(*s, dtype=torch.float64) for s in ((3, 8), (16, 8), (16, 8), (8, 16))])


def test_loss_refuses():
    h, w, t = fake(3, 8), fake(20, 8), fake(3, dtype=torch.int64)
    for call in (lambda: m.linear_cross_entropy(h, fake(20, 9), t),
                 lambda: m.linear_cross_entropy(h, w, fake(4, dtype=torch.int64)),
                 lambda: m.linear_cross_entropy(h, w, fake(3)),
                 lambda: m.linear_cross_entropy(h, w, t, reduction="max"),
                 lambda: m.linear_cross_entropy(h, fake(0, 8), t)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(m.M3bError, match="one dtype"):
        m.linear_cross_entropy(h, fake(20, 8, dtype=torch.float16), t)


def test_clip_refuses(monkeypatch):
    monkeypatch.setattr("mamba3_b200.clip._get_device", lambda t: 0 if t.is_cuda else -1)
    g = torch.zeros(10)
    for call in (lambda: m.clip_grads([_Cuda(g)], -1.0), lambda: m.clip_grads([_Cuda(g)], math.nan),
                 lambda: m.clip_grads([_Cuda(g)], 1.0, 1.0), lambda: m.clip_grads([_Cuda(g), _Cuda(g)], 1.0),
                 lambda: m.clip_grads([_Cuda(g)], 1.0, out=[]), lambda: m.clip_grads([_Cuda(g[::2])], 1.0),
                 lambda: m.clip_grads([_Cuda(g)], 1.0, out=[fake(11)]),
                 lambda: m.clip_grads([_Cuda(g), fake(10)], 1.0, out=[fake(10), _Cuda(g)]),
                 lambda: m.clip_grads([_Cuda(g)], 1.0, out=[_Cuda(g.view(torch.bfloat16)[:10])])):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(m.M3bError, match="unsupported dtype"):
        m.clip_grads([fake(3, dtype=torch.float64)], 1.0)
    assert m.clip_grads([], 1.0).item() == 0.0
    assert m.clip_grad_norm_([torch.nn.Parameter(g)], 1.0).item() == 0.0  # no gradient yet


def test_lm_options():
    lm = m.KulaMambaLM(vocab_size=50, d_model=64, n_layers=2, d_state=16, headdim=16, fused_mlp=True)
    assert all(blk.mlp.fused for blk in lm.layers)
    plain = m.KulaMambaLM(vocab_size=50, d_model=64, n_layers=2, d_state=16, headdim=16)
    assert not any(blk.mlp.fused for blk in plain.layers)
    assert set(lm.state_dict()) == set(plain.state_dict())
    with pytest.raises(ValueError, match="labels"):
        lm(torch.zeros(1, 4, dtype=torch.long), return_logits=False)


def test_modules_pickled_without_the_fused_attribute():
    mlp = m.SwiGLU(8, 16, fused=True)
    del mlp.__dict__["fused"]
    old = pickle.loads(pickle.dumps(mlp))
    assert old.fused is False


def test_loss_without_logits_needs_a_plain_head():
    """Only its weight is read: a head that does more is refused, before anything runs."""
    lm = m.KulaMambaLM(vocab_size=50, d_model=64, n_layers=1, d_state=16, headdim=16)
    ids = torch.zeros(1, 4, dtype=torch.long)
    with pytest.raises(ValueError, match="labels"):
        lm(ids, return_logits=False)
    for head in (torch.nn.Linear(64, 50), torch.nn.Sequential(torch.nn.Linear(64, 50, bias=False))):
        lm.lm_head = head
        with pytest.raises(ValueError, match="lm_head"):
            lm(ids, ids, return_logits=False)
