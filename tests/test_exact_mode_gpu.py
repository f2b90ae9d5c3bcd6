"""KernelMathMode.Exact through the linear layer: the MatMul node's own bits, sum,
bias and activation alike, whatever follows them."""
import pytest
import torch

import momiru_b200 as mb
from test_linear_gpu import ACT, V, gen, rand, replay

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda_lib")]
EXACT = dict(math_mode=mb.KernelMathMode.Exact, accuracy=mb.AccuracyContract.Exact)


def node_result(epilogue, lhs, rhs, bias, tr):
    out = torch.full((lhs.shape[0], rhs.shape[0 if tr else 1]), float("nan"), device="cuda")
    node = mb.MatMulNode(transpose_rhs=tr, epilogue=mb.Epilogue[epilogue], **EXACT)
    replay(mb.BoundGemm(node, V(lhs), V(rhs), V(out), bias=V(bias) if "BIAS" in epilogue else None))
    return out


def same_bits(x, y):
    assert torch.equal(x.isnan(), y.isnan())  # NaN payloads aside
    assert torch.equal(x.nan_to_num(0.0).view(torch.int32), y.nan_to_num(0.0).view(torch.int32))


@pytest.mark.parametrize("act", list(ACT))
@pytest.mark.parametrize("m,n,k,tr", [(1, 300, 40, True), (5, 132, 77, False), (150, 260, 64, False), (33, 7, 0, False)])
def test_bits_of_the_node(act, m, n, k, tr):
    g = gen(int(act) + m)
    lhs, bias, r = rand(g, m, k), rand(g, n, scale=3.0), rand(g, m, n)
    rhs = rand(g, *((n, k) if tr else (k, n)), scale=2 * max(k, 1) ** -0.5)
    if k > 40:
        lhs[0, 1], lhs[1, 2], lhs[2, 3] = float("inf"), float("-inf"), float("nan")
    plain = "NONE" if act == ACT.NONE else act.name
    biased = "BIAS" if act == ACT.NONE else "BIAS_" + act.name
    node = mb.LinearNode(transpose_rhs=tr, activation=act, **EXACT)
    new = lambda: torch.full((m, n), float("nan"), device="cuda")  # noqa: E731
    for b in (None, bias):
        want = node_result(biased if b is not None else plain, lhs, rhs, bias, tr)
        before = node_result("BIAS" if b is not None else "NONE", lhs, rhs, bias, tr)
        args = dict(bias=V(b)) if b is not None else {}
        out = new()
        replay(mb.BoundLinear(node, V(lhs), V(rhs), V(out), **args))
        same_bits(out, want)
        out, pre = new(), new()
        replay(mb.BoundLinear(node, V(lhs), V(rhs), V(out), pre=V(pre), residual=V(r), **args))
        same_bits(out, want + r)
        same_bits(pre, before)
        out = new().t().contiguous().t()  # the other storage order, element by element
        replay(mb.BoundLinear(node, V(lhs), V(rhs), V(out), **args))
        same_bits(out, want)
