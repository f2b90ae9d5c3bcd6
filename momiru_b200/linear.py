"""The linear layer: a matrix product with bias, activation and residual in its
epilogue, and its gradient.

    pre = lhs @ rhs + bias
    out = act(pre) + residual

Beside the f32 MatMul node (execution.py) this takes bf16 and f16 operands
(f32 sums, one rounding), adds the residual, and keeps `pre` for the gradient.
Bound, replayed and quiesced as the MatMul node is; errors are its typed
exceptions. The activations are the node's (the reference CPU provider's
elementwise kernels, src/momiru/tensor_light/execution/cpu.rs:2117-2222): bit
for bit in KernelMathMode.Exact, the same functions in f32 arithmetic of their
own in the other modes.
"""
from __future__ import annotations

import ctypes
import enum
from dataclasses import dataclass

from . import _abi, _ops_abi
from .execution import (AccuracyContract, InvalidArgument, KernelMathMode, _MATH_TO_ABI, _check,
                        validate_node_math_contract)
from .tensor import DeviceView


class Activation(enum.IntEnum):
    NONE = _ops_abi.ACT_NONE
    RELU = _ops_abi.ACT_RELU
    RELU6 = _ops_abi.ACT_RELU6
    GELU_ERF = _ops_abi.ACT_GELU_ERF
    GELU_TANH = _ops_abi.ACT_GELU_TANH
    SILU = _ops_abi.ACT_SILU


@dataclass(frozen=True)
class LinearNode:
    """What a linear layer computes. transpose_rhs takes weights stored as
    [n, k]. 16-bit operands run in StrictFp32 only (exact products, f32 sums);
    f32 operands in the MatMul node's modes."""
    transpose_lhs: bool = False
    transpose_rhs: bool = False
    activation: Activation = Activation.NONE
    math_mode: KernelMathMode = KernelMathMode.StrictFp32
    accuracy: AccuracyContract = AccuracyContract.StrictFp32

    def __post_init__(self):
        validate_node_math_contract(self.math_mode, self.accuracy)


def _fill(desc, device_ordinal: int, stream: int | None, **views: DeviceView | None):
    for name, view in views.items():
        if view is not None:
            setattr(desc, name, view.to_abi_tensor())
    desc.device_ordinal = device_ordinal
    desc.stream = stream or None
    return desc


class BoundOp:
    """A bound operator: replay enqueues it, quiesce_or_abort waits for it and
    reports a kernel's error, close releases it. Runs follow one another
    whatever streams and host threads they come from. The views (and so their
    buffers) are kept alive until close."""

    def __init__(self, bind: str, desc, views):
        self._lib = _ops_abi.load()
        self._views = views
        self._handle = ctypes.c_void_p()
        _check(getattr(self._lib, bind)(ctypes.byref(desc), ctypes.byref(self._handle)))

    def replay(self, stream: int | None = None) -> None:
        """Enqueue one pass on `stream` (a cudaStream_t; None: the bound one)."""
        if not self._handle:
            raise InvalidArgument("handle closed", _abi.ERR_INVALID_ARGUMENT)
        if stream is None:
            rc = self._lib.mmr_op_run(self._handle)
        else:
            rc = self._lib.mmr_op_run_on(self._handle, stream)
        if rc:
            _check(rc)

    def quiesce_or_abort(self, timeout_s: float = 30.0) -> None:
        if not self._handle:
            raise InvalidArgument("handle closed", _abi.ERR_INVALID_ARGUMENT)
        _check(self._lib.mmr_op_quiesce(self._handle, int(timeout_s * 1e9)))

    @property
    def plan(self) -> str:
        """The launches of one pass, one per line."""
        return self._lib.mmr_op_plan(self._handle).decode()

    def close(self) -> None:
        if self._handle:
            rc = self._lib.mmr_op_destroy(self._handle)
            self._handle = ctypes.c_void_p()
            _check(rc)

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def __del__(self):
        try:
            if self._handle:
                self._lib.mmr_op_destroy(self._handle)
        except Exception:
            pass


class BoundLinear(BoundOp):
    """out [m, n] = act(lhs [m, k] @ rhs [k, n] + bias [n]) + residual [m, n].

    All operands have one type: bf16, f16 or f32. `pre`, where given, receives
    the value before the activation. Views may have any strides. `residual` may
    be `out`'s own view (an update in place)."""

    def __init__(self, node: LinearNode, lhs: DeviceView, rhs: DeviceView, out: DeviceView,
                 bias: DeviceView | None = None, residual: DeviceView | None = None, pre: DeviceView | None = None,
                 stream: int | None = None):
        self.node = node
        d = _fill(_ops_abi.MmrLinearDesc(), out.buffer.device_ordinal, stream, lhs=lhs, rhs=rhs, out=out, bias=bias,
                  residual=residual, pre=pre)
        d.transpose_lhs, d.transpose_rhs = int(node.transpose_lhs), int(node.transpose_rhs)
        d.activation, d.math_mode = int(node.activation), _MATH_TO_ABI[node.math_mode]
        super().__init__("mmr_linear_bind", d, (lhs, rhs, out, bias, residual, pre))


class BoundLinearGrad(BoundOp):
    """The linear layer's gradient from d_out [m, n]:

        d_pre = d_out * act'(pre);  d_lhs = d_pre @ rhs^T;  d_rhs = lhs^T @ d_pre;  d_bias = sum of d_pre over m

    d_lhs and d_rhs have the layouts of lhs and rhs (transposed ones as the node
    says); each gradient is optional. The residual's gradient is d_out itself.
    `pre` is what BoundLinear kept, needed where the node has an activation."""

    def __init__(self, node: LinearNode, d_out: DeviceView, lhs: DeviceView, rhs: DeviceView,
                 d_lhs: DeviceView | None = None, d_rhs: DeviceView | None = None, d_bias: DeviceView | None = None,
                 pre: DeviceView | None = None, stream: int | None = None):
        self.node = node
        d = _fill(_ops_abi.MmrLinearGradDesc(), d_out.buffer.device_ordinal, stream, d_out=d_out, lhs=lhs, rhs=rhs,
                  pre=pre, d_lhs=d_lhs, d_rhs=d_rhs, d_bias=d_bias)
        d.transpose_lhs, d.transpose_rhs = int(node.transpose_lhs), int(node.transpose_rhs)
        d.activation, d.math_mode = int(node.activation), _MATH_TO_ABI[node.math_mode]
        super().__init__("mmr_linear_grad_bind", d, (d_out, lhs, rhs, pre, d_lhs, d_rhs, d_bias))
