"""The Python side of the training and serving operators: traced forms, workspaces, modules (no kernel launches)."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import mamba3_b200 as m  # noqa: F401


@pytest.mark.parametrize("reduction,per_row", [("none", True), ("mean", False), ("sum", False)])
@pytest.mark.parametrize("rows", [9, 3])
def test_traced_loss_has_the_reduction_s_shape(rows, reduction, per_row):
    with FakeTensorMode():
        h, w = torch.empty(rows, 64, dtype=torch.bfloat16), torch.empty(300, 64, dtype=torch.bfloat16)
        loss, saved = torch.ops.mamba3_b200.linear_xent_fwd(h, w, torch.empty(rows, dtype=torch.long), -100, reduction)
    assert loss.shape == ((rows,) if per_row else ()) and loss.dtype == torch.float32 and saved.dtype == torch.uint8
