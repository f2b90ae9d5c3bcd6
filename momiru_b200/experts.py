"""Tokens sorted by expert and back, and the experts' products between.

A mixture-of-experts feed-forward in the framework's operators:

    layout = ExpertLayout.empty(tokens, top_k, experts, row_align)
    BoundDispatch(layout, ids, x, rows)                 rows of each expert, contiguous
    BoundExpertLinear(node, layout, rows, w_up, hidden) each expert's product on its own rows
    BoundExpertLinear(node, layout, hidden, w_down, rows_out)
    BoundCombine(layout, rows_out, out, weights, residual)

and their gradients (the dispatch's is BoundCombine without weights). The
layout's arrays live on the device and no count is read back to the host:
buffers have ExpertLayout.capacity rows, which hold any routing.

A sorted row that holds no token (a segment's padding, or past the last
segment) is zero. Every operator here writes it so, and the gradients rely on
it: a caller who fills a sorted buffer by other means keeps those rows zero.
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

from . import _ops_abi
from .execution import InvalidArgument, KernelMathMode, _check
from .linear import Activation, BoundOp, LinearNode, _fill
from .tensor import DeviceView, DType


@dataclass(frozen=True)
class ExpertLayout:
    """Where each assignment of a token to an expert goes.

    Assignment i = t * top_k + j; an id outside [0, experts) drops it.
    slots [tokens, top_k]: its row or -1. sources [rows]: a row's assignment or
    -1. offsets [experts + 1]: where each expert's segment starts, a multiple
    of row_align (a power of two up to 128). counts [experts]: its assignments.
    All i32. Within a segment assignments keep their order."""
    tokens: int
    top_k: int
    experts: int
    row_align: int
    slots: DeviceView
    sources: DeviceView
    offsets: DeviceView
    counts: DeviceView

    @staticmethod
    def capacity(tokens: int, top_k: int, experts: int, row_align: int = 64) -> int:
        """Rows of the sorted buffers: enough for any ids."""
        rows = ctypes.c_int64()
        _check(_ops_abi.load().mmr_expert_rows(tokens, top_k, experts, row_align, ctypes.byref(rows)))
        return rows.value

    @staticmethod
    def empty(tokens: int, top_k: int, experts: int, row_align: int = 64, device_ordinal: int = 0) -> "ExpertLayout":
        rows = ExpertLayout.capacity(tokens, top_k, experts, row_align)
        new = lambda *dims: DeviceView.empty(dims, device_ordinal, DType.I32)  # noqa: E731
        return ExpertLayout(tokens, top_k, experts, row_align, new(tokens, top_k), new(rows), new(experts + 1),
                            new(experts))

    @property
    def rows(self) -> int:
        return self.sources.dims[0]

    def to_abi(self) -> _ops_abi.MmrExpertLayout:
        return _ops_abi.MmrExpertLayout(self.tokens, self.top_k, self.experts, self.row_align,
                                        self.slots.to_abi_tensor(), self.sources.to_abi_tensor(),
                                        self.offsets.to_abi_tensor(), self.counts.to_abi_tensor())


def _product_node(node: LinearNode) -> LinearNode:
    if node.transpose_lhs:
        raise InvalidArgument("an expert product's rows are not transposed", InvalidArgument.code)
    if node.math_mode != KernelMathMode.StrictFp32:
        raise InvalidArgument("an expert product runs in StrictFp32", InvalidArgument.code)
    return node


class BoundDispatch(BoundOp):
    """Sorts: writes the layout from ids [tokens, top_k] i32 and gathers rows
    [capacity, h] from x [tokens, h] (f32, bf16 or f16, unit column strides)."""

    def __init__(self, layout: ExpertLayout, ids: DeviceView, x: DeviceView, rows: DeviceView,
                 stream: int | None = None):
        self.layout = layout
        d = _fill(_ops_abi.MmrDispatchDesc(layout=layout.to_abi()), rows.buffer.device_ordinal, stream, ids=ids, x=x,
                  rows=rows)
        super().__init__("mmr_dispatch_bind", d, (layout, ids, x, rows))


class BoundCombine(BoundOp):
    """out[t] = sum over j of weights[t, j] * rows[slots[t, j]] (+ residual[t]),
    dropped assignments left out; f32 sums in increasing j. weights [tokens,
    top_k] f32, or None for all ones, which is the dispatch's gradient.
    `residual` may be `out`'s own view."""

    def __init__(self, layout: ExpertLayout, rows: DeviceView, out: DeviceView, weights: DeviceView | None = None,
                 residual: DeviceView | None = None, stream: int | None = None):
        self.layout = layout
        d = _fill(_ops_abi.MmrCombineDesc(layout=layout.to_abi()), out.buffer.device_ordinal, stream, rows=rows,
                  weights=weights, residual=residual, out=out)
        super().__init__("mmr_combine_bind", d, (layout, rows, weights, residual, out))


class BoundCombineGrad(BoundOp):
    """d_rows[slots[t, j]] = weights[t, j] * d_out[t] and d_weights[t, j] =
    <d_out[t], rows[slots[t, j]]> (f32); either may be left out. The residual's
    gradient is d_out itself."""

    def __init__(self, layout: ExpertLayout, d_out: DeviceView, rows: DeviceView | None = None,
                 weights: DeviceView | None = None, d_rows: DeviceView | None = None,
                 d_weights: DeviceView | None = None, stream: int | None = None):
        self.layout = layout
        d = _fill(_ops_abi.MmrCombineGradDesc(layout=layout.to_abi()), d_out.buffer.device_ordinal, stream,
                  d_out=d_out, rows=rows, weights=weights, d_rows=d_rows, d_weights=d_weights)
        super().__init__("mmr_combine_grad_bind", d, (layout, d_out, rows, weights, d_rows, d_weights))


class BoundExpertLinear(BoundOp):
    """out = act(rows @ weights[e] + bias[e]) on each expert's rows; bf16 or f16.
    weights [experts, k, n], or [experts, n, k] with the node's transpose_rhs."""

    def __init__(self, node: LinearNode, layout: ExpertLayout, rows: DeviceView, weights: DeviceView,
                 out: DeviceView, bias: DeviceView | None = None, pre: DeviceView | None = None,
                 stream: int | None = None):
        self.node, self.layout = _product_node(node), layout
        d = _fill(_ops_abi.MmrExpertLinearDesc(layout=layout.to_abi()), out.buffer.device_ordinal, stream, rows=rows,
                  weights=weights, bias=bias, out=out, pre=pre)
        d.transpose_rhs, d.activation = int(node.transpose_rhs), int(node.activation)
        super().__init__("mmr_expert_linear_bind", d, (layout, rows, weights, bias, out, pre))


class BoundExpertLinearGrad(BoundOp):
    """The expert products' gradient: d_rows, d_weights (zero for an expert
    without tokens) and d_bias, each optional. d_weights and d_bias need a
    layout with row_align of 64 or 128."""

    def __init__(self, node: LinearNode, layout: ExpertLayout, d_out: DeviceView, rows: DeviceView,
                 weights: DeviceView, d_rows: DeviceView | None = None, d_weights: DeviceView | None = None,
                 d_bias: DeviceView | None = None, pre: DeviceView | None = None, stream: int | None = None):
        self.node, self.layout = _product_node(node), layout
        d = _fill(_ops_abi.MmrExpertLinearGradDesc(layout=layout.to_abi()), d_out.buffer.device_ordinal, stream,
                  d_out=d_out, rows=rows, weights=weights, pre=pre, d_rows=d_rows, d_weights=d_weights, d_bias=d_bias)
        d.transpose_rhs, d.activation = int(node.transpose_rhs), int(node.activation)
        super().__init__("mmr_expert_linear_grad_bind", d,
                         (layout, d_out, rows, weights, pre, d_rows, d_weights, d_bias))


__all__ = ["Activation", "BoundCombine", "BoundCombineGrad", "BoundDispatch", "BoundExpertLinear",
           "BoundExpertLinearGrad", "ExpertLayout"]
