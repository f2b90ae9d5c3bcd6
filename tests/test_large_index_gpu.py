"""The operators where element offsets pass 2^31 on more rows than a strip takes:
the CTA-pair product with residual and kept pre, the packing of an odd pitch, a
gradient through an activation; and the most rows that a view may have. Bounds
as in test_linear_gpu.py."""
import pytest
import torch

import momiru_b200 as mb
from test_linear_gpu import ACT, TINY, TYPES, V, act64, check, check_forward, gen, rand, replay

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda_lib")]
ROWS = 1100  # above 1024 the pair kernel takes every product; (ROWS - 1) * pitch is 2.3e9 elements


def blocks(pitch, *widths):
    """Column blocks of one buffer of ROWS rows, 512 columns apart."""
    buf = torch.empty((ROWS - 1) * pitch + 512 * len(widths), dtype=torch.bfloat16, device="cuda")
    return [buf.as_strided((ROWS, w), (pitch, 1), 512 * i) for i, w in enumerate(widths)]


@pytest.mark.parametrize("pitch,kernel", [(2 << 20, None), ((2 << 20) + 1, "mmr_pack_kernel")])
def test_pair_product_with_residual_and_pre(pitch, kernel):
    t, u = TYPES["bf16"]
    g = gen(21)
    n, k = 264, 136
    lhs, out, res, pre = blocks(pitch, k, n, n, n)
    lhs.copy_(rand(g, ROWS, k))
    res.copy_(rand(g, ROWS, n))
    rhs, b = rand(g, k, n, dtype=t, scale=k ** -0.5), rand(g, n, dtype=t)
    op = mb.BoundLinear(mb.LinearNode(activation=ACT.SILU), V(lhs), V(rhs), V(out), bias=V(b), residual=V(res), pre=V(pre))
    assert "mmr_linear_pair_kernel" in op.plan and (kernel is None or kernel in op.plan)
    replay(op)
    check_forward(t, u, lhs, rhs, b, res, ACT.SILU, out, pre)


@pytest.mark.parametrize("n", [264, 131])
def test_gradient_through_an_activation(n):
    t, u = TYPES["bf16"]
    g = gen(22)
    k, pitch = 136, 2 << 20
    lhs, dy, pre, d_lhs = blocks(pitch, k, n, n, k)
    lhs.copy_(rand(g, ROWS, k))
    dy.copy_(rand(g, ROWS, n))
    pre.copy_(rand(g, ROWS, n, scale=2.0))
    rhs = rand(g, k, n, dtype=t, scale=k ** -0.5)
    d_rhs, d_bias = torch.empty_like(rhs), torch.empty(n, dtype=t, device="cuda")
    node = mb.LinearNode(activation=ACT.GELU_TANH)
    replay(mb.BoundLinearGrad(node, V(dy), V(lhs), V(rhs), d_lhs=V(d_lhs), d_rhs=V(d_rhs), d_bias=V(d_bias), pre=V(pre)))
    a, b = lhs.double(), rhs.double()
    dp = dy.double() * act64(ACT.GELU_TANH, pre.double())[1]
    off = u * dp.abs() + 2.0 ** -18 * dy.double().abs()
    want, tol = dp @ b.t(), off @ b.t().abs() + (n + 1) * 2.0 ** -23 * (dp.abs() @ b.t().abs())
    check(d_lhs, want, u * want.abs() + tol * (1 + u) + TINY, "d_lhs")
    want, tol = a.t() @ dp, a.t().abs() @ off + (ROWS + 1) * 2.0 ** -23 * (a.t().abs() @ dp.abs())
    check(d_rhs, want, u * want.abs() + tol * (1 + u) + TINY, "d_rhs")
    want = dp.sum(0)
    tol = u * want.abs() + (2.0 ** -18 + (ROWS + 1) * 2.0 ** -24) * (dp.abs() + dy.double().abs()).sum(0)
    check(d_bias, want, tol + TINY, "d_bias")


def test_the_most_rows():
    """2^31 - 1024 rows times the identity: every row comes back as it was."""
    m = 2 ** 31 - 1024
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GB of free device memory")
    lhs, out = (torch.empty(m, 8, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    step = 1 << 26
    g = gen(23)
    for i in range(0, m, step):
        lhs[i:i + step].normal_(generator=g)
    out.zero_()
    one = torch.eye(8, dtype=torch.bfloat16, device="cuda")
    replay(mb.BoundLinear(mb.LinearNode(), V(lhs), V(one), V(out)))
    assert all(torch.equal(lhs[i:i + step], out[i:i + step]) for i in range(0, m, step))
    del lhs, out
    torch.cuda.empty_cache()
