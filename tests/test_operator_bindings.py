"""The Python side of the training and serving operators: traced forms, workspaces, modules (no kernel launches)."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from mamba3_b200 import _lib


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
