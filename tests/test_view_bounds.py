"""Bounds of views whose extents, strides or offsets pass 64 bits when they are
multiplied or added: refused as out of bounds, not taken for the wrapped value.
Nothing here needs a GPU (a view that passed would stop at the missing or
foreign device instead, with another error)."""
import ctypes

import pytest

import momiru_b200 as mb
from momiru_b200 import _abi
from momiru_b200.execution import OutOfBounds

pytestmark = pytest.mark.usefixtures("cuda_lib")
BF16, F32 = mb.DType.BF16, mb.DType.F32
WRAP = (1 << 24) + 1  # rows: (WRAP - 1) * 2^40 is 2^64, which 64 bits hold as 0


def view(address, dims, strides, nbytes, offset=0, dtype=BF16):
    return mb.DeviceView(mb.DeviceBuffer(address, nbytes), dims, strides, offset, dtype)


def operands(m, dtype=BF16):
    es = dtype.itemsize
    return dict(lhs=view(1 << 44, (m, 8), (8, 1), m * 8 * es, dtype=dtype),
                rhs=view(2 << 44, (8, 8), (8, 1), 64 * es, dtype=dtype),
                out=view(3 << 44, (m, 8), (8, 1), m * 8 * es, dtype=dtype))


def strided(name, rows, stride, dtype=BF16):
    ops = operands(rows, dtype)
    ops[name] = view(4 << 44, (rows, 8), (stride, 1), 16 * dtype.itemsize, dtype=dtype)
    return ops


@pytest.mark.parametrize("name", ["lhs", "out"])
@pytest.mark.parametrize("rows,stride", [(WRAP, 1 << 40), (WRAP - 1, 1 << 40), (WRAP + 1, 1 << 40), (1 << 25, 1 << 39),
                                         (WRAP, -(1 << 40)), ((1 << 31) - 1024, 1 << 33)])
def test_operators_refuse_strides_that_wrap(name, rows, stride):
    for dtype in (BF16, F32):
        with pytest.raises(OutOfBounds):
            mb.BoundLinear(mb.LinearNode(), **strided(name, rows, stride, dtype))


@pytest.mark.parametrize("name", ["lhs", "rhs", "out"])
@pytest.mark.parametrize("offset", [-1, -8, -(1 << 30), (1 << 62) - 1])
def test_operators_refuse_offsets_that_wrap(name, offset):
    """A negative offset arrives as a huge unsigned one; the last one wraps with the extent added."""
    ops = operands(8)
    ops[name] = view(4 << 44, (8, 8), (8, 1), 1 << 20, offset)
    with pytest.raises(OutOfBounds):
        mb.BoundLinear(mb.LinearNode(), **ops)


def test_operators_refuse_buffers_past_the_address_space():
    ops = operands(8)
    ops["lhs"] = view((1 << 64) - 64, (8, 8), (8, 1), 128)
    with pytest.raises(OutOfBounds):
        mb.BoundLinear(mb.LinearNode(), **ops)


@pytest.mark.parametrize("name", ["lhs", "out"])
@pytest.mark.parametrize("rows,stride", [(WRAP, 1 << 40), (WRAP + 1, 1 << 40), (WRAP, -(1 << 40)), (1 << 25, 1 << 39)])
def test_node_refuses_strides_that_wrap(name, rows, stride):
    ops = strided(name, rows, stride, F32)
    with pytest.raises(OutOfBounds):
        mb.validate(mb.MatMulNode(), ops["lhs"], ops["rhs"], ops["out"])


@pytest.mark.parametrize("name", ["lhs", "rhs", "out"])
@pytest.mark.parametrize("offset", [-1, -8, -(1 << 30), (1 << 62) - 1])
def test_node_refuses_offsets_that_wrap(name, offset):
    ops = operands(8, F32)
    ops[name] = view(4 << 44, (8, 8), (8, 1), 1 << 20, offset, F32)
    with pytest.raises(OutOfBounds):
        mb.validate(mb.MatMulNode(), ops["lhs"], ops["rhs"], ops["out"])


def test_node_refuses_batches_that_wrap():
    """2^24 + 1 matrices 2^40 elements apart."""
    ops = operands(8, F32)
    lhs = view(4 << 44, (WRAP, 8, 8), (1 << 40, 8, 1), 256, dtype=F32)
    out = view(5 << 44, (WRAP, 8, 8), (64, 8, 1), WRAP * 256, dtype=F32)
    with pytest.raises(OutOfBounds):
        mb.validate(mb.MatMulNode(), lhs, ops["rhs"], out)


def test_host_entry_refuses_pitches_that_wrap():
    """2^31 + 1 rows, 2^31 elements apart."""
    lib = _abi.load()
    ops = operands(8, F32)
    d = _abi.MmrMatmulDesc()
    d.lhs, d.rhs, d.out = (ops[n].to_abi() for n in ("lhs", "rhs", "out"))
    d.lhs.dims[0], d.lhs.strides[0], d.lhs.bytes = (1 << 31) + 1, 1 << 31, 32  # (rows - 1) * pitch * 4 is 2^64
    h = ctypes.c_void_p()
    assert lib.mmr_gemm_bind_host(ctypes.byref(d), 0, ctypes.byref(h)) == _abi.ERR_INVALID_SHAPE
