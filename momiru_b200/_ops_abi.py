"""ctypes bindings of the C ABI declared in include/momiru_ops.h: the linear
layer, tokens sorted by expert, and the experts' products. Same library and
statuses as _abi.py; no fallback."""
from __future__ import annotations

import ctypes

from . import _abi
from ._abi import MmrView

DTYPE_F32, DTYPE_BF16, DTYPE_F16, DTYPE_I32 = 0, 1, 2, 3
ACT_NONE, ACT_RELU, ACT_RELU6, ACT_GELU_ERF, ACT_GELU_TANH, ACT_SILU = 0, 1, 2, 3, 4, 5

EXPORTED = [
    "mmr_expert_rows", "mmr_linear_bind", "mmr_linear_grad_bind", "mmr_dispatch_bind", "mmr_combine_bind",
    "mmr_combine_grad_bind", "mmr_expert_linear_bind", "mmr_expert_linear_grad_bind", "mmr_op_run", "mmr_op_run_on",
    "mmr_op_quiesce", "mmr_op_destroy", "mmr_op_plan",
]


class MmrTensor(ctypes.Structure):
    _fields_ = [("view", MmrView), ("dtype", ctypes.c_int32), ("reserved", ctypes.c_int32)]


def _tensors(*names):
    return [(n, MmrTensor) for n in names]


def _ints(*names):
    return [(n, ctypes.c_int32) for n in names]


_TAIL = _ints("device_ordinal", "reserved") + [("stream", ctypes.c_void_p)]


class MmrLinearDesc(ctypes.Structure):
    _fields_ = (_tensors("lhs", "rhs", "out", "bias", "residual", "pre")
                + _ints("transpose_lhs", "transpose_rhs", "activation", "math_mode") + _TAIL)


class MmrLinearGradDesc(ctypes.Structure):
    _fields_ = (_tensors("d_out", "lhs", "rhs", "pre", "d_lhs", "d_rhs", "d_bias")
                + _ints("transpose_lhs", "transpose_rhs", "activation", "math_mode") + _TAIL)


class MmrExpertLayout(ctypes.Structure):
    _fields_ = ([(n, ctypes.c_int64) for n in ("tokens", "top_k", "experts", "row_align")]
                + _tensors("slots", "sources", "offsets", "counts"))


class MmrDispatchDesc(ctypes.Structure):
    _fields_ = [("layout", MmrExpertLayout)] + _tensors("ids", "x", "rows") + _TAIL


class MmrCombineDesc(ctypes.Structure):
    _fields_ = [("layout", MmrExpertLayout)] + _tensors("rows", "weights", "residual", "out") + _TAIL


class MmrCombineGradDesc(ctypes.Structure):
    _fields_ = ([("layout", MmrExpertLayout)] + _tensors("d_out", "rows", "weights", "d_rows", "d_weights") + _TAIL)


class MmrExpertLinearDesc(ctypes.Structure):
    _fields_ = ([("layout", MmrExpertLayout)] + _tensors("rows", "weights", "bias", "out", "pre")
                + _ints("transpose_rhs", "activation") + _TAIL)


class MmrExpertLinearGradDesc(ctypes.Structure):
    _fields_ = ([("layout", MmrExpertLayout)]
                + _tensors("d_out", "rows", "weights", "pre", "d_rows", "d_weights", "d_bias")
                + _ints("transpose_rhs", "activation") + _TAIL)


_DESCS = {"mmr_linear_bind": MmrLinearDesc, "mmr_linear_grad_bind": MmrLinearGradDesc,
          "mmr_dispatch_bind": MmrDispatchDesc, "mmr_combine_bind": MmrCombineDesc,
          "mmr_combine_grad_bind": MmrCombineGradDesc, "mmr_expert_linear_bind": MmrExpertLinearDesc,
          "mmr_expert_linear_grad_bind": MmrExpertLinearGradDesc}

_ready = False


def load() -> ctypes.CDLL:
    global _ready
    lib = _abi.load()
    if not _ready:
        P, h = ctypes.POINTER, ctypes.c_void_p
        for name, desc in _DESCS.items():
            getattr(lib, name).argtypes = [P(desc), P(h)]
        lib.mmr_expert_rows.argtypes = [ctypes.c_int64] * 4 + [P(ctypes.c_int64)]
        lib.mmr_op_run.argtypes = [h]
        lib.mmr_op_run_on.argtypes = [h, ctypes.c_void_p]
        lib.mmr_op_quiesce.argtypes = [h, ctypes.c_uint64]
        lib.mmr_op_destroy.argtypes = [h]
        lib.mmr_op_plan.argtypes = [h]
        for name in EXPORTED:
            getattr(lib, name).restype = ctypes.c_int32
        lib.mmr_op_plan.restype = ctypes.c_char_p
        _ready = True
    return lib
