"""Handles of one kernel and different sizes, all bound before the first runs."""
import pytest
import torch

import momiru_b200 as mb
from test_linear_gpu import V, gen, rand, rel, replay

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda_lib")]


@pytest.mark.parametrize("m", [1, 2, 4, 7, 16])
def test_node_gemv_of_long_and_short_contractions(m):
    """lhs transposed, so that the streaming product runs on the CUDA cores for every number of rows."""
    g = gen(m)
    made = []
    for k in (8192, 4096, 512, 16):
        lhs, rhs = rand(g, k, m), rand(g, k, 256, scale=k ** -0.5)
        out = torch.zeros(m, 256, device="cuda")
        node = mb.MatMulNode(transpose_lhs=True, family=mb.KernelFamily.Gemv)
        made.append((mb.BoundGemm(node, V(lhs), V(rhs), V(out)), lhs, rhs, out))
    for order in (made, made[::-1]):
        for op, lhs, rhs, out in order:
            out.zero_()
            torch.cuda.synchronize()
            op.replay()
            op.quiesce_or_abort(20)
            assert rel(out, lhs.double().t() @ rhs.double()) <= 1e-5
    for op, *_ in made:
        op.close()


def test_one_gradient_with_two_streaming_products():
    """d_lhs by columns (16 x 33 over 582) and d_rhs (16 x 582 over 33) in one handle."""
    g = gen(9)
    m, n, k = 33, 582, 16
    lhs, rhs, dy = rand(g, m, k), rand(g, k, n, scale=0.25), rand(g, m, n)
    d_lhs, d_rhs = torch.empty(k, m, device="cuda").t(), torch.empty_like(rhs)
    replay(mb.BoundLinearGrad(mb.LinearNode(), V(dy), V(lhs), V(rhs), d_lhs=V(d_lhs), d_rhs=V(d_rhs)))
    assert rel(d_lhs, dy.double() @ rhs.double().t()) <= 1e-5
    assert rel(d_rhs, lhs.double().t() @ dy.double()) <= 1e-5
