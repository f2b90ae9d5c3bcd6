"""momiru_b200 -- B200 (sm_100a) f32 matmul hot path for Momiru's frozen-plan GEMM node.

The compute path is the in-tree CUDA library (csrc/, built by build.py) behind
the C ABI in include/momiru_gemm.h (and, for the operators around the node,
include/momiru_ops.h); this package is the host-side mirror of
the reference's node / bind / replay / quiesce interface.
"""
from .execution import (AccuracyContract, BoundGemm, Epilogue, HostGemm, KernelFamily,
                        KernelMathMode, MatMulNode, PlanError, check_launch_record, matmul, output_dims,
                        plan_launch, selftest_bounded_wait, shard_columns, validate)
from .experts import (BoundCombine, BoundCombineGrad, BoundDispatch, BoundExpertLinear, BoundExpertLinearGrad,
                      ExpertLayout)
from .linear import Activation, BoundLinear, BoundLinearGrad, LinearNode
from .tensor import DeviceBuffer, DeviceView, DType

__all__ = [
    "AccuracyContract", "Activation", "BoundCombine", "BoundCombineGrad", "BoundDispatch", "BoundExpertLinear",
    "BoundExpertLinearGrad", "BoundGemm", "BoundLinear", "BoundLinearGrad", "DType", "DeviceBuffer", "DeviceView",
    "Epilogue", "ExpertLayout", "HostGemm",
    "KernelFamily",
    "KernelMathMode", "LinearNode", "MatMulNode", "PlanError", "check_launch_record", "matmul", "output_dims", "plan_launch",
    "selftest_bounded_wait", "shard_columns", "validate",
]
