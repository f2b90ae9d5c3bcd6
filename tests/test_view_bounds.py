"""Bounds of views whose extents, strides or offsets pass 64 bits when they are
multiplied or added: refused as out of bounds, not taken for the wrapped value.
Nothing here needs a GPU (a view that passed would stop at the missing or
foreign device instead, with another error)."""
import pytest

import momiru_b200 as mb
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
