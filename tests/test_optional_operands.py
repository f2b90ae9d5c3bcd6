"""An optional operand that is there but of no taken rank is refused, not left
out: the layer would be computed without it."""
import ctypes

import pytest

import momiru_b200 as mb
from momiru_b200 import _abi, _ops_abi
from momiru_b200.execution import InvalidShape

pytestmark = pytest.mark.usefixtures("cuda_lib")


def at(address, dims, dtype=mb.DType.BF16):
    return mb.DeviceView.contiguous(mb.DeviceBuffer(address, 4096), dims, dtype=dtype)


LHS, RHS, OUT = at(0x100000, (4, 32)), at(0x200000, (32, 1)), at(0x300000, (4, 1))


@pytest.mark.parametrize("name", ["bias", "residual", "pre"])
def test_scalars_are_refused(name):
    with pytest.raises(InvalidShape):
        mb.BoundLinear(mb.LinearNode(), LHS, RHS, OUT, **{name: at(0x400000, ())})


def test_scalar_gradients_and_weights_are_refused():
    with pytest.raises(InvalidShape):
        mb.BoundLinearGrad(mb.LinearNode(), OUT, LHS, RHS, d_lhs=at(0x500000, (4, 32)), d_bias=at(0x400000, ()))
    rows = mb.ExpertLayout.capacity(4, 1, 2, 1)
    lay = mb.ExpertLayout(4, 1, 2, 1, *(at(0x1000000 + 4096 * i, d, mb.DType.I32) for i, d in enumerate([(4, 1), (rows,), (3,), (2,)])))
    with pytest.raises(InvalidShape):
        mb.BoundCombine(lay, at(0x600000, (rows, 8)), at(0x700000, (4, 8)), weights=at(0x400000, (), mb.DType.F32))


@pytest.mark.parametrize("rank", [-1, -8, 9])
def test_ranks_out_of_range_are_refused(rank):
    d = _ops_abi.MmrLinearDesc(lhs=LHS.to_abi_tensor(), rhs=RHS.to_abi_tensor(), out=OUT.to_abi_tensor())
    d.bias = at(0x400000, (1,)).to_abi_tensor()
    d.bias.view.rank = rank
    h = ctypes.c_void_p()
    assert _ops_abi.load().mmr_linear_bind(ctypes.byref(d), ctypes.byref(h)) == _abi.ERR_INVALID_SHAPE
