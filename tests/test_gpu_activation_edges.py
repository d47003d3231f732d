"""Calls at the edges of what the activation operators document."""
import pytest
import torch

import ark_b200 as ab

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


@pytest.mark.parametrize("itype", [torch.int32, torch.int64])
def test_positions_of_no_tokens(itype):
    """A batch without tokens gives positions without elements."""
    plan, pos = ab.RopePlan(32), torch.empty(0, dtype=itype, device="cuda")
    q, g = torch.empty(0, 4, 32, dtype=F16, device="cuda"), torch.ones(32, dtype=F16, device="cuda")
    assert ab.rope(q, q[:, :2], plan, pos)[1].shape == (0, 2, 32)
    y = ab.qk_norm_rope(q, q[:, :2], g, g, plan, pos, checkpoint="int8")
    assert y[0].shape == q.shape and y[2].rows == 0
    back = ab.qk_norm_rope_backward(q, q[:, :2], y[2], y[3], g, g, plan, pos)
    assert (back[2] == 0).all() and (back[3] == 0).all()
