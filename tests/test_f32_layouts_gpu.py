"""f32 layers over views that share a buffer or a row pitch: each is computed,
whatever the MatMul node itself would take."""
import pytest
import torch

import momiru_b200 as mb
from test_linear_gpu import V, gen, rand, rel, replay

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda_lib")]
STRICT = mb.LinearNode()
EXACT = mb.LinearNode(math_mode=mb.KernelMathMode.Exact, accuracy=mb.AccuracyContract.Exact)


@pytest.mark.parametrize("m", [4, 12, 200])
@pytest.mark.parametrize("node", [STRICT, EXACT], ids=["strict", "exact"])
def test_column_blocks_of_one_buffer(m, node):
    """lhs and out (and d_lhs) side by side in every row; the bytes between them keep their values."""
    g = gen(41)
    n, k = 260, 136
    wide = rand(g, m, 1024)
    lhs, out, d_lhs = wide[:, :k], wide[:, 256:256 + n], wide[:, 600:600 + k]
    rhs, b, dy = rand(g, k, n, scale=k ** -0.5), rand(g, n), rand(g, m, n)
    before = wide.clone()
    replay(mb.BoundLinear(node, V(lhs), V(rhs), V(out)))
    assert rel(out, lhs.double() @ rhs.double()) <= 1e-5
    replay(mb.BoundLinear(node, V(lhs), V(rhs), V(out), bias=V(b)))
    assert rel(out, lhs.double() @ rhs.double() + b.double()) <= 1e-5
    d_rhs = torch.empty_like(rhs)
    replay(mb.BoundLinearGrad(node, V(dy), V(lhs), V(rhs), d_lhs=V(d_lhs), d_rhs=V(d_rhs)))
    assert rel(d_lhs, dy.double() @ rhs.double().t()) <= 1e-5
    assert rel(d_rhs, lhs.double().t() @ dy.double()) <= 1e-5
    kept = torch.ones(1024, dtype=torch.bool, device="cuda")
    kept[256:256 + n], kept[600:600 + k] = False, False
    assert torch.equal(wide[:, kept], before[:, kept])
