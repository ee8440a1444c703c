"""The Python side of the training and serving operators: traced forms, workspaces, modules (no kernel launches)."""

import weakref

import pytest
import torch
import torch.autograd.forward_ad as fwAD
import torch.nn.utils.parametrize
from torch._subclasses.fake_tensor import FakeTensorMode

from mamba3_b200 import _lib, block, clip, ffn, loss, ops


@pytest.mark.parametrize("reduction,per_row", [("none", True), ("mean", False), ("sum", False)])
@pytest.mark.parametrize("rows", [9, 3])
def test_traced_loss_has_the_reduction_s_shape(rows, reduction, per_row):
    with FakeTensorMode():
        h, w = torch.empty(rows, 64, dtype=torch.bfloat16), torch.empty(300, 64, dtype=torch.bfloat16)
        loss, saved = torch.ops.mamba3_b200.linear_xent_fwd(h, w, torch.empty(rows, dtype=torch.long), -100, reduction)
    assert loss.shape == ((rows,) if per_row else ()) and loss.dtype == torch.float32 and saved.dtype == torch.uint8


@pytest.fixture
def no_launches(monkeypatch):
    """The library's host side runs on CPU tensors; its launches are recorded instead."""
    calls = []
    monkeypatch.setattr(_lib, "_err_addr", lambda index: None)
    monkeypatch.setattr(_lib, "_same_gpu", lambda name, ts: -1)
    monkeypatch.setattr(_lib, "_call", lambda fn, what, index, *args: calls.append((what, args)))
    return calls


@pytest.mark.parametrize("save", [True, False])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("rows", [3, 40])
def test_traced_ffn_returns_what_the_call_returns(rows, dtype, save, no_launches):
    args = lambda: [torch.zeros(s, dtype=dtype) for s in ((rows, 40), (24, 40), (24, 40), (40, 24))]  # noqa: E731
    op = torch.ops.mamba3_b200.gated_ffn_fwd
    got = op(*args(), None, None, None, None, 1.0, save)
    with FakeTensorMode():
        want = op(*args(), None, None, None, None, 1.0, save)
    assert len(no_launches) == 1
    for a, b in zip(got, want):
        assert a.shape == b.shape and a.dtype == b.dtype and a.stride() == b.stride()


@pytest.mark.parametrize("rows", [3, 40])
@pytest.mark.parametrize("save", [True, False])
def test_workspaces_live_until_the_launches_are_made(rows, save, monkeypatch, no_launches):
    """A block that is given back before the call could be handed to another thread between its launches."""
    given, dead = [], []
    real = _lib._bytes

    def counted(n, dev):
        t = real(n, dev)
        given.append(weakref.ref(t))
        return t

    monkeypatch.setattr(_lib, "_bytes", counted)
    monkeypatch.setattr(_lib, "_call", lambda fn, what, *a: dead.append((what, sum(r() is None for r in given))))
    z = lambda *s: torch.zeros(s)  # noqa: E731
    x, wg, wu, wd = z(rows, 33), z(24, 33), z(24, 33), z(33, 24)
    out, act, gu = _lib.gated_ffn_fwd(x, wg, wu, wd, None, None, None, None, 1.0, save)
    if save:
        given.clear()
        _lib.gated_ffn_bwd(x, wg, wu, wd, None, None, None, 1.0, act, gu, x, [True] * 7)
    given.clear()
    loss, saved = _lib.linear_xent_fwd(x, wg, torch.zeros(rows, dtype=torch.long), -100, "mean", save)
    if save:
        given.clear()
        _lib.linear_xent_bwd(rows, wg, saved, loss, -100, "mean", True, True)
    given.clear()
    _lib.grad_clip([x.data_ptr()], [x.numel()], [x.dtype], [x.data_ptr()], [x.dtype], 1.0, False, x.device)
    assert len(dead) == (5 if save else 3) and not any(n for _, n in dead), dead


def test_labels_of_any_integer_type(monkeypatch):
    """The last token predicts nothing: its label is the ignored one also where the labels' type cannot hold it."""
    seen = []
    monkeypatch.setattr(block, "linear_cross_entropy", lambda h, w, t: seen.append(t) or h.sum())
    lm = block.KulaMambaLM(vocab_size=50, d_model=64, n_layers=1, d_state=16, headdim=16)
    monkeypatch.setattr(lm, "_hidden", lambda ids: torch.zeros(*ids.shape, 64))
    ids = torch.tensor([[3, 4, 5]])
    for dt in (torch.int64, torch.int32, torch.int16, torch.uint8):
        lm(ids, ids.to(dt), return_logits=False)
        assert seen.pop().tolist() == [[4, 5, -100]]


class _Adapter(torch.nn.Linear):
    def forward(self, x):
        return super().forward(x) + 1.0


def _altered(linear, how):
    """`linear` doing more than its weight and bias say."""
    if how == "subclass":
        other = _Adapter(linear.in_features, linear.out_features, bias=linear.bias is not None)
        other.load_state_dict(linear.state_dict())
        return other
    if how == "wrapped":
        return torch.nn.Sequential(linear)
    if how == "forward hook":
        linear.register_forward_hook(lambda mod, args, out: out + 1.0)
    elif how == "pre-hook":
        linear.register_forward_pre_hook(lambda mod, args: (args[0] + 1.0,))
    elif how == "backward hook":
        linear.register_full_backward_hook(lambda mod, gi, go: None)
    else:
        linear.forward = lambda x: torch.nn.functional.linear(x, linear.weight, linear.bias) + 1.0
    return linear


ALTERED = ["subclass", "wrapped", "forward hook", "pre-hook", "backward hook", "own forward"]


@pytest.mark.parametrize("how", ALTERED)
@pytest.mark.parametrize("name", ["w_gate", "w_up", "w_down"])
def test_fused_mlp_runs_projections_that_do_more_as_modules(name, how):
    """The operator reads weights only (and refuses CPU tensors, so what returns here ran as modules)."""
    mlp = block.SwiGLU(8, 16, bias=True, fused=True)
    x, r = torch.randn(3, 8), torch.randn(3, 8)
    with pytest.raises(_lib.M3bError, match="CUDA"):
        mlp(x)
    setattr(mlp, name, _altered(getattr(mlp, name), how))
    want = mlp.w_down(torch.nn.functional.silu(mlp.w_gate(x)) * mlp.w_up(x))
    assert torch.equal(mlp(x), want) and torch.allclose(mlp(x, r, 0.5), r + 0.5 * want)


@pytest.mark.parametrize("how", ALTERED)
def test_fused_mlp_with_a_parametrised_or_hooked_module(how, monkeypatch):
    """A parametrised Linear is its computed weight: the operator takes that.  A hook on the MLP itself sees the
    MLP's output, without the residual."""
    calls = []
    monkeypatch.setattr(block, "gated_ffn", lambda x, *w, residual=None, residual_scale=1.0, **b:
                        calls.append((w, residual)) or x)
    blk = block.KulaMambaBlock(64, d_state=16, headdim=16, fused_mlp=True)
    x = torch.randn(2, 3, 64)
    blk._mlp_residual(x)
    assert calls.pop()[1] is x and not calls
    torch.nn.utils.parametrize.register_parametrization(blk.mlp.w_up, "weight", _Doubled())
    blk._mlp_residual(x)
    (w, r), = calls
    assert r is x and torch.equal(w[1], blk.mlp.w_up.weight)
    calls.clear()
    if how in ("forward hook", "pre-hook", "backward hook"):
        _altered(blk.mlp, how)
        blk._mlp_residual(x)
        assert calls.pop()[1] is None and not calls


class _Doubled(torch.nn.Module):
    def forward(self, w):
        return 2 * w


@pytest.mark.parametrize("how", ALTERED)
def test_loss_without_logits_refuses_heads_that_do_more(how):
    lm = block.KulaMambaLM(vocab_size=50, d_model=64, n_layers=1, d_state=16, headdim=16)
    ids = torch.zeros(1, 4, dtype=torch.long)
    lm.lm_head = _altered(lm.lm_head, how)
    with pytest.raises(ValueError, match="lm_head"):
        lm(ids, ids, return_logits=False)


def test_forward_mode_derivatives_are_refused(monkeypatch):
    """No operator here has a forward-mode derivative: a tangent raises, also where nothing requires grad."""
    monkeypatch.setattr(_lib, "_same_gpu", lambda name, ts: 0)
    monkeypatch.setattr(ops, "gated_ffn_fwd", lambda x, *a: (x + 0.0, x.detach(), x.detach()))
    monkeypatch.setattr(ops, "linear_xent_fwd", lambda h, *a: (h.sum().detach(), h.detach()))
    x, w, wd = torch.randn(3, 8), torch.randn(16, 8), torch.randn(8, 16)
    t = torch.zeros(3, dtype=torch.long)
    calls = [lambda a: ffn.gated_ffn(a, w, w, wd), lambda a: ffn.gated_ffn(x, w, w, wd, residual=a),
             lambda a: loss.linear_cross_entropy(a, w, t)]
    for call in calls:
        call(x)
        for grad in (True, False):
            with torch.set_grad_enabled(grad), fwAD.dual_level(), pytest.raises(RuntimeError, match="jvp|forward"):
                call(fwAD.make_dual(x, torch.ones_like(x)))
            with torch.set_grad_enabled(grad), fwAD.dual_level():
                call(x)  # no tangent among the arguments


def test_forward_mode_derivatives_of_the_scans_are_refused():
    from mamba3_b200 import chunked_ssd, ssd_scan

    with fwAD.dual_level():
        a = fwAD.make_dual(torch.zeros(1, 2, 3), torch.ones(1, 2, 3))
        with pytest.raises(_lib.M3bError, match="forward-mode"):
            ssd_scan(a, torch.zeros(1, 2, 3, 4, 5))
        with pytest.raises(_lib.M3bError, match="forward-mode"):
            chunked_ssd(None, None, None, None, None, a, None, None, None)


@pytest.mark.parametrize("other", [False, True])
def test_clipping_is_a_write_that_autograd_knows_of(monkeypatch, other):
    """A tensor kept for a backward pass and then clipped: the backward pass raises, as after any write in place."""
    monkeypatch.setattr(clip, "_get_device", lambda t: 0)
    monkeypatch.setattr(_lib, "grad_clip", lambda *a: torch.zeros(()))
    w, g = torch.ones(3, requires_grad=True), torch.ones(3)
    y = (w * g).sum()
    clip.clip_grads([torch.ones(3)] if other else [g], 1.0, out=[g] if other else None)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    y = (w * g).sum()
    clip.clip_grads([g], 1.0, out=[torch.ones(3)])  # only read
    y.backward()
