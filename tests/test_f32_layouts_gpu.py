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


def planned(op):
    """One run of `op`, which may not fall to the node's scalar kernel."""
    assert "simt" not in op.plan, op.plan
    replay(op)


TF32 = mb.LinearNode(math_mode=mb.KernelMathMode.Tf32, accuracy=mb.AccuracyContract.AllowTf32)


@pytest.mark.parametrize("m,n,k", [
    (1, 1001, 11008), (1, 1000, 11008), (2, 130, 8193), (16, 500, 8193), (16, 77, 12000), (9, 515, 8192), (16, 1, 9000),
    (9, 1, 900), (40, 1, 900), (200, 1, 4001), (1, 1, 9001), (17, 3, 5), (8200, 12, 40), (8195, 3, 9), (300, 1, 1)])
def test_no_product_falls_to_the_scalar_kernel(m, n, k):
    """Few rows with a long contraction, single columns, gradients of many rows: in both layouts of rhs."""
    g = gen(m + n + k)
    lhs, b, r, dy = rand(g, m, k), rand(g, n), rand(g, m, n), rand(g, m, n)
    for tr in (False, True):
        rhs = rand(g, *((n, k) if tr else (k, n)), scale=k ** -0.5)
        b64 = (rhs.t() if tr else rhs).double()
        want = lhs.double() @ b64
        for node, bound in ((STRICT, 1e-5), (TF32, 2e-3)):
            node = mb.LinearNode(transpose_rhs=tr, math_mode=node.math_mode, accuracy=node.accuracy)
            out = torch.full((m, n), float("nan"), device="cuda")
            planned(mb.BoundLinear(node, V(lhs), V(rhs), V(out)))
            assert rel(out, want) <= bound
            planned(mb.BoundLinear(node, V(lhs), V(rhs), V(out), bias=V(b), residual=V(r)))
            assert rel(out, want + b.double() + r.double()) <= bound
            d_lhs, d_rhs = torch.full_like(lhs, float("nan")), torch.full_like(rhs, float("nan"))
            planned(mb.BoundLinearGrad(node, V(dy), V(lhs), V(rhs), d_lhs=V(d_lhs), d_rhs=V(d_rhs)))
            assert rel(d_lhs, dy.double() @ b64.t()) <= bound
            assert rel(d_rhs.t() if tr else d_rhs, lhs.double().t() @ dy.double()) <= bound


@pytest.mark.parametrize("m", [1, 5, 12, 200])
@pytest.mark.parametrize("k", [136, 8195])
def test_strided_outputs_bias_and_reversed_rows(m, k):
    """Every second column of a buffer, every second entry of a bias, an lhs read from its last row or column on."""
    g = gen(m + k)
    n = 260
    lhs, rhs, bias = rand(g, m, k), rand(g, k, n, scale=k ** -0.5), rand(g, 2 * n)[::2]
    want = lhs.double() @ rhs.double() + bias.double()
    buf = torch.full((m, 2 * n), 7.0, device="cuda")
    planned(mb.BoundLinear(STRICT, V(lhs), V(rhs), V(buf[:, ::2]), bias=V(bias)))
    assert rel(buf[:, ::2], want) <= 1e-5 and bool((buf[:, 1::2] == 7).all())
    out = torch.empty(m, n, device="cuda")
    planned(mb.BoundLinear(STRICT, V(lhs), V(rhs), V(out), bias=V(bias)))
    assert rel(out, want) <= 1e-5
    v = V(lhs)
    rows = mb.DeviceView(v.buffer, v.dims, (-k, 1), (m - 1) * k)
    planned(mb.BoundLinear(STRICT, rows, V(rhs), V(out), bias=V(bias)))
    assert rel(out, want.flip(0)) <= 1e-5
    cols = mb.DeviceView(v.buffer, v.dims, (k, -1), k - 1)
    planned(mb.BoundLinear(STRICT, cols, V(rhs), V(out)))
    assert rel(out, lhs.double().flip(1) @ rhs.double()) <= 1e-5


@pytest.mark.parametrize("m", [1, 12, 16, 40])
def test_repeated_rows_and_columns(m):
    """Operands broadcast along one of their axes (a stride of 0)."""
    g = gen(m)
    n, k = 528, 4163
    lhs, row, col = rand(g, m, k, scale=k ** -0.5), rand(g, n), rand(g, k)
    out = torch.empty(m, n, device="cuda")
    repeated = mb.DeviceView(V(row).buffer, (k, n), (0, 1))
    planned(mb.BoundLinear(STRICT, V(lhs), repeated, V(out)))
    # the sums over lhs cancel: the error is that of the absolute sums
    want, size = lhs.double().sum(1, keepdim=True) * row.double(), lhs.double().abs().sum(1, keepdim=True) * row.double().abs()
    assert float((out.double() - want).norm() / size.norm()) <= 1e-5
    repeated = mb.DeviceView(V(col).buffer, (k, n), (1, 0))
    planned(mb.BoundLinear(STRICT, V(lhs), repeated, V(out)))
    want, size = (lhs.double() @ col.double())[:, None].expand(m, n), (lhs.double().abs() @ col.double().abs())[:, None].expand(m, n)
    assert float((out.double() - want).norm() / size.norm()) <= 1e-5
