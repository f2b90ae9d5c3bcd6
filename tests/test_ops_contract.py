"""The operators' C boundary on CPU: the ctypes mirror against the header, the
sizes of the sorted buffers, and every refusal that needs no GPU (bind checks
its arguments before it looks for a device)."""
import ctypes
import os
import re

import numpy as np
import pytest

import momiru_b200 as mb
from momiru_b200 import _abi, _ops_abi
from momiru_b200.execution import (InvalidArgument, InvalidAccuracyContract, InvalidShape, OutOfBounds, PlanError,
                                   UnsafeAliasing, UnsupportedDevice, UnsupportedLayout)
from momiru_b200.tensor import ViewError

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
with open(os.path.join(ROOT, "include", "momiru_ops.h")) as f:
    HEADER = f.read()

pytestmark = pytest.mark.usefixtures("cuda_lib")
BF16, F16, F32, I32 = mb.DType.BF16, mb.DType.F16, mb.DType.F32, mb.DType.I32


def at(address, dims, dtype=BF16, strides=None, offset=0, nbytes=None):
    """A view over made-up addresses: bind refuses, or stops at the missing or foreign device."""
    n = int(np.prod(dims)) if len(dims) else 1
    buf = mb.DeviceBuffer(address, nbytes if nbytes is not None else max(n, 1) * dtype.itemsize)
    v = mb.DeviceView.contiguous(buf, dims, offset, dtype)
    return v if strides is None else v.as_strided_view(dims, strides)


def linear(node=None, **kw):
    a = dict(lhs=at(0x100000, (4, 32)), rhs=at(0x200000, (32, 16)), out=at(0x300000, (4, 16)))
    a.update(kw)
    return mb.BoundLinear(node or mb.LinearNode(), **a)


def layout(tokens=6, top_k=2, experts=4, align=16, base=0x1000000):
    rows = mb.ExpertLayout.capacity(tokens, top_k, experts, align)
    return mb.ExpertLayout(tokens, top_k, experts, align, at(base, (tokens, top_k), I32),
                           at(base + 0x10000, (rows,), I32), at(base + 0x20000, (experts + 1,), I32),
                           at(base + 0x30000, (experts,), I32))


def test_exports_and_structs_follow_the_header():
    declared = set(re.findall(r"MMR_API\s+(?:int32_t|const char \*)\s*(mmr_\w+)\s*\(", HEADER))
    assert declared == set(_ops_abi.EXPORTED)
    for name, struct in [("mmr_tensor", _ops_abi.MmrTensor), ("mmr_linear_desc", _ops_abi.MmrLinearDesc),
                         ("mmr_linear_grad_desc", _ops_abi.MmrLinearGradDesc),
                         ("mmr_expert_layout", _ops_abi.MmrExpertLayout),
                         ("mmr_dispatch_desc", _ops_abi.MmrDispatchDesc),
                         ("mmr_combine_desc", _ops_abi.MmrCombineDesc),
                         ("mmr_combine_grad_desc", _ops_abi.MmrCombineGradDesc),
                         ("mmr_expert_linear_desc", _ops_abi.MmrExpertLinearDesc),
                         ("mmr_expert_linear_grad_desc", _ops_abi.MmrExpertLinearGradDesc)]:
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), HEADER, re.S).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        names = [re.findall(r"(\w+)\s*$", part.strip())[0]
                 for decl in body.split(";") if decl.strip() for part in decl.split(",")]
        assert names == [f for f, _ in struct._fields_], name


def test_rust_binding_follows_the_header():
    with open(os.path.join(ROOT, "rust", "src", "gpu_gemm", "ops_ffi.rs")) as f:
        rust = f.read()
    consts = dict(re.findall(r"\b(MMR_(?:DTYPE|ACT)_\w+) = (\d+)", HEADER))
    assert dict(re.findall(r"pub const (MMR_\w+): i32 = (\d+);", rust)) == consts
    assert set(re.findall(r"pub fn (mmr_\w+)\(", rust)) == set(_ops_abi.EXPORTED)
    structs = re.findall(r"pub struct (mmr_\w+) \{(.*?)\n\}", rust, re.S)
    mirror = {"Mmr" + "".join(w.title() for w in n.split("_")[1:]): re.findall(r"pub (\w+):", body) for n, body in structs
              if n != "mmr_op_handle"}
    assert len(mirror) == 9
    for name, fields in mirror.items():
        assert fields == [f for f, _ in getattr(_ops_abi, name)._fields_], name
    with open(os.path.join(ROOT, "rust", "build_gpu.rs")) as f:
        units = re.search(r"UNITS: \[&str; \d+\] = \[(.*?)\];", f.read(), re.S).group(1)
    from momiru_b200 import build
    assert sorted(re.findall(r'"(\w+)"', units)) == sorted(os.path.splitext(u)[0] for u in build.SOURCES)


@pytest.mark.parametrize("tokens,top_k,experts,align", [
    (0, 1, 1, 1), (1, 1, 1, 1), (1, 1, 8, 128), (3, 2, 64, 16), (100, 8, 64, 64), (4099, 4, 24, 64), (7, 1, 1024, 1)])
def test_capacity_holds_the_worst_routing(tokens, top_k, experts, align):
    rows = mb.ExpertLayout.capacity(tokens, top_k, experts, align)
    n = tokens * top_k
    # the padded total is largest with one assignment in as many experts as there can be, the rest in one of them
    used = min(experts, n)
    counts = [1] * used
    if used:
        counts[0] += n - used
    assert rows >= sum(-(-c // align) * align for c in counts)
    assert rows % align == 0 and rows <= n + used * (align - 1)


@pytest.mark.parametrize("args,error", [
    ((-1, 1, 1, 1), InvalidShape), ((1, 0, 1, 1), InvalidShape), ((1, 1, 0, 1), InvalidShape),
    ((1, 1, 1025, 1), InvalidShape), ((1, 1, 1, 3), InvalidArgument), ((1, 1, 1, 256), InvalidArgument),
    ((1 << 30, 4, 8, 1), InvalidShape)])
def test_capacity_refuses(args, error):
    with pytest.raises(error):
        mb.ExpertLayout.capacity(*args)


@pytest.mark.parametrize("kw,error", [
    (dict(lhs=at(0x100000, (4, 31))), InvalidShape),
    (dict(out=at(0x300000, (5, 16))), InvalidShape),
    (dict(bias=at(0x400000, (15,))), InvalidShape),
    (dict(bias=at(0x400000, (1, 16))), InvalidShape),
    (dict(residual=at(0x400000, (4, 17))), InvalidShape),
    (dict(lhs=at(0x100000, (2, 4, 32))), InvalidShape),
    (dict(rhs=at(0x200000, (32, 16), F16)), InvalidArgument),
    (dict(out=at(0x300000, (4, 16), F32)), InvalidArgument),
    (dict(lhs=at(0x100000, (4, 32), I32)), InvalidArgument),
    (dict(lhs=at(0x100000, (4, 32), nbytes=100)), OutOfBounds),
    (dict(lhs=at(0x100000, (4, 32), strides=(-32, 1))), OutOfBounds),
    (dict(lhs=at(0x100001, (4, 32))), UnsupportedLayout),
    (dict(lhs=at(0, (4, 32))), InvalidArgument),
    (dict(out=at(0x300000, (4, 16), strides=(0, 1))), UnsafeAliasing),
    (dict(out=at(0x300000, (4, 16), strides=(8, 1))), UnsafeAliasing),
    (dict(out=at(0x100000, (4, 16))), UnsafeAliasing),
    (dict(residual=at(0x300002, (4, 16))), UnsafeAliasing),
    (dict(pre=at(0x300000, (4, 16))), UnsafeAliasing),
    (dict(residual=at(0x400000, (4, 16)), pre=at(0x400000, (4, 16))), UnsafeAliasing),
])
def test_linear_refuses(kw, error):
    with pytest.raises(error):
        linear(**kw)


def test_linear_math_modes():
    A = mb.AccuracyContract
    tf32 = mb.LinearNode(math_mode=mb.KernelMathMode.Tf32, accuracy=A.AllowTf32)
    with pytest.raises(InvalidAccuracyContract):
        linear(tf32)  # 16-bit operands have one mode
    with pytest.raises(InvalidAccuracyContract):
        mb.LinearNode(math_mode=mb.KernelMathMode.Tf32)


def test_what_passes_the_checks_stops_at_the_device():
    """In place, column blocks of one buffer, reversed rows: admitted (and then there is no such device memory)."""
    wide = at(0x100000, (4, 96))
    blocks = dict(lhs=wide.narrow(1, 0, 32), out=wide.narrow(1, 40, 16), residual=wide.narrow(1, 64, 16))
    reverse = mb.DeviceView(mb.DeviceBuffer(0x100000, 256), (4, 32), (-32, 1), 96, BF16)
    out = at(0x300000, (4, 16))
    for kw in (blocks, dict(lhs=reverse), dict(out=out, residual=out)):
        with pytest.raises((UnsupportedDevice, PlanError)) as e:
            linear(**kw)
        assert e.value.code in (_abi.ERR_UNSUPPORTED_DEVICE, _abi.ERR_CUDA)


def test_matmul_node_refuses_other_types():
    with pytest.raises(ViewError):
        mb.validate(mb.MatMulNode(), at(0x100000, (4, 32)), at(0x200000, (32, 16)), at(0x300000, (4, 16)))


def test_linear_grad_refuses():
    def grad(node=mb.LinearNode(), **kw):
        a = dict(d_out=at(0x100000, (4, 16)), lhs=at(0x200000, (4, 32)), rhs=at(0x300000, (32, 16)),
                 d_lhs=at(0x400000, (4, 32)))
        a.update(kw)
        return mb.BoundLinearGrad(node, **a)

    with pytest.raises(InvalidArgument):
        grad(d_lhs=None)
    with pytest.raises(InvalidArgument):
        grad(mb.LinearNode(activation=mb.Activation.SILU))  # without pre
    with pytest.raises(InvalidShape):
        grad(d_lhs=at(0x400000, (32, 4)))
    with pytest.raises(InvalidShape):
        grad(d_bias=at(0x500000, (4,)))
    with pytest.raises(UnsafeAliasing):
        grad(d_lhs=at(0x200000, (4, 32)))
    with pytest.raises(UnsafeAliasing):
        grad(d_rhs=at(0x400000, (32, 16)))


def test_routing_refuses():
    lay = layout()
    x, rows = at(0x2000000, (6, 40)), at(0x3000000, (lay.rows, 40))
    ids = at(0x4000000, (6, 2), I32)
    for kw, error in [(dict(ids=at(0x4000000, (6, 3), I32)), InvalidShape),
                      (dict(ids=at(0x4000000, (6, 2), F32)), InvalidArgument),
                      (dict(x=at(0x2000000, (6, 41))), InvalidShape),
                      (dict(x=at(0x2000000, (6, 40), F16)), InvalidArgument),
                      (dict(x=at(0x2000000, (6, 40), strides=(1, 6))), UnsupportedLayout),
                      (dict(rows=at(0x3000000, (lay.rows - 1, 40))), InvalidShape),
                      (dict(rows=at(0x2000000, (lay.rows, 40))), UnsafeAliasing)]:
        with pytest.raises(error):
            mb.BoundDispatch(lay, **{**dict(ids=ids, x=x, rows=rows), **kw})
    out, w = at(0x5000000, (6, 40)), at(0x6000000, (6, 2), F32)
    for kw, error in [(dict(weights=at(0x6000000, (6, 2), BF16)), InvalidArgument),
                      (dict(weights=at(0x6000000, (2, 6), F32)), InvalidShape),
                      (dict(out=at(0x5000000, (5, 40))), InvalidShape),
                      (dict(out=rows.narrow(0, 0, 6)), UnsafeAliasing),
                      (dict(residual=out.narrow(0, 0, 5)), InvalidShape)]:
        with pytest.raises(error):
            mb.BoundCombine(lay, **{**dict(rows=rows, out=out, weights=w), **kw})
    d_rows = at(0x7000000, (lay.rows, 40))
    with pytest.raises(InvalidArgument):
        mb.BoundCombineGrad(lay, out, rows, w)
    with pytest.raises(InvalidArgument):  # the rows are needed for the weights' gradient
        mb.BoundCombineGrad(lay, out, None, w, d_weights=at(0x8000000, (6, 2), F32))
    with pytest.raises(UnsafeAliasing):
        mb.BoundCombineGrad(lay, out, rows, w, d_rows=rows, d_weights=at(0x8000000, (6, 2), F32))
    with pytest.raises(InvalidShape):
        mb.BoundCombineGrad(lay, out, rows, w, d_rows=at(0x7000000, (lay.rows, 39)))
    with pytest.raises(InvalidArgument):
        mb.BoundCombineGrad(lay, out, rows, w, d_rows=at(0x7000000, (lay.rows, 40), F16))
    _ = d_rows


def test_layout_arrays_are_checked():
    lay = layout()
    x, rows, ids = at(0x2000000, (6, 40)), at(0x3000000, (lay.rows, 40)), at(0x4000000, (6, 2), I32)
    import dataclasses
    for change, error in [(dict(offsets=at(0x1020000, (4,), I32)), InvalidShape),
                          (dict(counts=at(0x1030000, (4,), F32)), InvalidArgument),
                          (dict(slots=at(0x1000000, (6, 2), I32, strides=(1, 6))), UnsupportedLayout),
                          (dict(row_align=48), InvalidArgument), (dict(experts=0), InvalidShape)]:
        with pytest.raises(error):
            mb.BoundDispatch(dataclasses.replace(lay, **change), ids, x, rows)


def test_expert_products_refuse():
    lay = layout()
    rows, w, out = at(0x2000000, (lay.rows, 32)), at(0x3000000, (4, 32, 24)), at(0x4000000, (lay.rows, 24))
    node = mb.LinearNode()
    for kw, error in [(dict(weights=at(0x3000000, (3, 32, 24))), InvalidShape),
                      (dict(weights=at(0x3000000, (4, 24, 32))), InvalidShape),
                      (dict(weights=at(0x3000000, (32, 24))), InvalidShape),
                      (dict(rows=at(0x2000000, (lay.rows, 32), F32)), InvalidArgument),
                      (dict(bias=at(0x5000000, (24,))), InvalidShape),
                      (dict(out=at(0x2000000, (lay.rows, 24))), UnsafeAliasing)]:
        with pytest.raises(error):
            mb.BoundExpertLinear(node, lay, **{**dict(rows=rows, weights=w, out=out), **kw})
    with pytest.raises(InvalidArgument):
        mb.BoundExpertLinear(mb.LinearNode(transpose_lhs=True), lay, rows, w, out)
    d_w = at(0x6000000, (4, 32, 24))
    with pytest.raises(UnsupportedLayout):  # segments of 16 rows
        mb.BoundExpertLinearGrad(node, lay, out, rows, w, d_weights=d_w)
    with pytest.raises(InvalidArgument):
        mb.BoundExpertLinearGrad(node, lay, out, rows, w)


def test_null_arguments():
    lib = _ops_abi.load()
    h = ctypes.c_void_p()
    for name, desc in _ops_abi._DESCS.items():
        fn = getattr(lib, name)
        assert fn(None, ctypes.byref(h)) == _abi.ERR_INVALID_ARGUMENT
        assert fn(ctypes.byref(desc()), None) == _abi.ERR_INVALID_ARGUMENT
        assert fn(ctypes.byref(desc()), ctypes.byref(h)) != _abi.OK and not h.value
    assert lib.mmr_op_run(None) == _abi.ERR_INVALID_ARGUMENT
    assert lib.mmr_op_quiesce(None, 1) == _abi.ERR_INVALID_ARGUMENT
    assert lib.mmr_op_destroy(None) == _abi.OK
    assert lib.mmr_expert_rows(1, 1, 1, 1, None) == _abi.ERR_INVALID_ARGUMENT
