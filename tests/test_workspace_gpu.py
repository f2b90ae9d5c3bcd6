"""Workspaces whose size passes 64 bits are refused when the operator is bound.
Nothing is run."""
import pytest
import torch

import momiru_b200 as mb
from momiru_b200.execution import InvalidShape, PlanError

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda_lib")]
V = mb.DeviceView.from_torch


def broadcast(dims):
    return V(torch.zeros(8, dtype=torch.bfloat16, device="cuda")).as_strided_view(dims, (0,) * len(dims))


def test_packing_more_than_64_bits_can_say():
    """Sixteen weights of 2^30 x 2^30, all one element: 2^65 bytes to pack, which 64 bits hold as 0."""
    n = 1 << 30
    lay = mb.ExpertLayout.empty(1, 1, 16, 1)
    out = torch.empty(lay.rows, n, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(InvalidShape):
        mb.BoundExpertLinear(mb.LinearNode(), lay, broadcast((lay.rows, n)), broadcast((16, n, n)), V(out))


def test_packing_more_than_the_memory():
    n = 1 << 23
    out = torch.empty(8, n, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(PlanError):  # 2^47 bytes: the allocation itself fails
        mb.BoundLinear(mb.LinearNode(), broadcast((8, n)), broadcast((n, n)), V(out))
