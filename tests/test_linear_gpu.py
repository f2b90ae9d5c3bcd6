"""The linear layer on the GPU against the same formula in 64 bits.

Bounds, per element. With u the output type's unit roundoff, S = |lhs| |rhs|
and products exact in f32:
  pre   |err| <= u |pre| + K 2^-23 S        (every f32 addition of the tensor
        core may truncate; the partial sums stay below S)
  out   the same carried through the activation (slope at most 1.13), plus
        2^-19 (1 + |pre|) for the 16-bit activations' approximations and
        rounding of the residual's sum
  gradients: d_pre is rounded once more to the operands' type, so its error
        u |d_pre| and the derivative's 2^-18 |d_out| join the sum.
2^-25 covers f16's subnormals. f32 operands: the StrictFp32 node's 1e-5
relative Frobenius bound.
"""
import numpy as np
import pytest
import torch

import momiru_b200 as mb

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda_lib")]

TYPES = {"bf16": (torch.bfloat16, 2.0 ** -8), "f16": (torch.float16, 2.0 ** -11)}
TINY = 2.0 ** -25
V = mb.DeviceView.from_torch
ACT = mb.Activation


def act64(act, x):
    """The activation and its derivative in 64 bits."""
    if act == ACT.NONE:
        return x, torch.ones_like(x)
    if act == ACT.RELU:
        return x.clamp(min=0), (x > 0).double()
    if act == ACT.RELU6:
        return x.clamp(0, 6), ((x > 0) & (x < 6)).double()
    if act == ACT.SILU:
        s = torch.sigmoid(x)
        return x * s, s * (1 + x * (1 - s))
    if act == ACT.GELU_ERF:
        c = 0.5 * torch.special.erfc(-x * 0.5 ** 0.5)
        return x * c, c + x * torch.exp(-0.5 * x * x) * (2 * np.pi) ** -0.5
    c = (2 / np.pi) ** 0.5
    s = torch.sigmoid(2 * c * (x + 0.044715 * x ** 3))
    return x * s, s + 2 * x * s * (1 - s) * c * (1 + 3 * 0.044715 * x * x)


def rand(gen, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def replay(op, stream=None):
    with op:
        op.replay(stream)
        op.quiesce_or_abort(20)


def check(got, want, tol, what):
    err = (got.double() - want).abs()
    assert bool((err <= tol).all()), f"{what}: worst {float((err / tol).max()):.3f} of its bound"


def forward_case(dtype, m, n, k, act=ACT.NONE, bias=False, residual=False, pre=False, tl=False, tr=False, seed=0):
    t, u = TYPES[dtype]
    g = gen(seed)
    lhs = rand(g, k, m, dtype=t).t() if tl else rand(g, m, k, dtype=t)
    rhs = rand(g, n, k, dtype=t, scale=k ** -0.5 if k else 1).t() if tr else rand(g, k, n, dtype=t, scale=k ** -0.5 if k else 1)
    b = rand(g, n, dtype=t) if bias else None
    r = rand(g, m, n, dtype=t) if residual else None
    out = torch.full((m, n), float("nan"), dtype=t, device="cuda")
    p = torch.full((m, n), float("nan"), dtype=t, device="cuda") if pre else None
    node = mb.LinearNode(transpose_lhs=tl, transpose_rhs=tr, activation=act)
    replay(mb.BoundLinear(node, V(lhs.t() if tl else lhs), V(rhs.t() if tr else rhs), V(out), bias=b is not None and V(b) or None,
                          residual=r is not None and V(r) or None, pre=p is not None and V(p) or None))
    check_forward(t, u, lhs, rhs, b, r, act, out, p)


def check_forward(t, u, lhs, rhs, b, r, act, out, p):
    k = lhs.shape[1]
    want_pre = lhs.double() @ rhs.double()
    s = lhs.double().abs() @ rhs.double().abs()
    if b is not None:
        want_pre = want_pre + b.double()
        s = s + b.double().abs()
    acc = (k + 1) * 2.0 ** -23 * s
    if p is not None:
        check(p, want_pre, u * want_pre.abs() + acc + TINY, "pre")
    want = act64(act, want_pre)[0]
    if r is not None:
        want = want + r.double()
    check(out, want, u * want.abs() + 1.13 * acc + 2.0 ** -19 * (1 + want_pre.abs()) + TINY, "out")


SHAPES = [(1, 16, 16), (1, 4096, 1000), (3, 8, 515), (16, 129, 64), (17, 1001, 130), (77, 1001, 515), (129, 264, 200),
          (256, 512, 1024), (257, 256, 64), (300, 520, 72), (513, 1000, 1025), (700, 30, 333), (1030, 2056, 264)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_shapes(dtype, m, n, k):
    forward_case(dtype, m, n, k, bias=True, residual=True, seed=m + n)
    forward_case(dtype, m, n, k, tr=True, pre=True, seed=m + n + 1)


@pytest.mark.parametrize("m", [5, 300])
@pytest.mark.parametrize("act", list(ACT))
def test_activations(m, act):
    forward_case("f16", m, 136, 96, act=act, bias=True, residual=True, pre=True, seed=int(act))
    forward_case("bf16", m, 136, 96, act=act, tr=True, seed=int(act) + 10)


@pytest.mark.parametrize("m", [24, 264])
@pytest.mark.parametrize("tl", [False, True])
@pytest.mark.parametrize("tr", [False, True])
@pytest.mark.parametrize("k", [64, 72, 77])
def test_transposed_operands(m, tl, tr, k):
    forward_case("bf16", m, 200, k, tl=tl, tr=tr, bias=True, seed=k)


@pytest.mark.parametrize("m,n,k", [(0, 64, 64), (64, 0, 64), (7, 24, 0), (300, 24, 0)])
def test_empty_axes(m, n, k):
    """No rows or columns: nothing; no contraction: act(bias) + residual."""
    forward_case("bf16", m, n, k, act=ACT.SILU, bias=True, residual=True)


@pytest.mark.parametrize("m", [9, 270])
def test_views_of_wider_buffers(m):
    """Column blocks of one buffer, a reversed operand, every second row, a
    transposed output; the bytes between them keep their values."""
    t, u = TYPES["bf16"]
    g = gen(3)
    wide = rand(g, m, 400, dtype=t)
    lhs, out, r = wide[:, :136], wide[:, 144:300], wide[:, 300:].contiguous()
    rest = wide[:, 300:].clone()
    r = rand(g, 2 * m, 156, dtype=t)[::2]
    rhs = rand(g, 136, 156, dtype=t, scale=0.1)
    b = rand(g, 312, dtype=t)[::2]
    lhs0 = lhs.clone()
    replay(mb.BoundLinear(mb.LinearNode(), V(lhs), V(rhs), V(out), bias=V(b), residual=V(r)))
    check_forward(t, u, lhs0, rhs, b, r, ACT.NONE, out, None)
    assert torch.equal(wide[:, 300:], rest) and torch.equal(lhs, lhs0)
    # rhs with both axes reversed, by a view of negative strides
    v = V(rhs)
    flipped = mb.DeviceView(v.buffer, v.dims, (-v.strides[0], -1), v.offset + rhs.numel() - 1, v.dtype)
    out_t = torch.zeros(156, m, dtype=t, device="cuda")
    replay(mb.BoundLinear(mb.LinearNode(), V(lhs), flipped, V(out_t).transpose()))
    check_forward(t, u, lhs0, rhs.flip(0, 1), None, None, ACT.NONE, out_t.t(), None)


@pytest.mark.parametrize("m", [6, 300])
def test_residual_in_place_and_repeat(m):
    """out += act(lhs rhs), twice: the second run reads what the first wrote; equal inputs give equal bits."""
    t, u = TYPES["f16"]
    g = gen(4)
    lhs, rhs, x0 = rand(g, m, 264, dtype=t), rand(g, 264, 512, dtype=t, scale=0.06), rand(g, m, 512, dtype=t)
    runs = []
    for _ in range(2):
        x = x0.clone()
        with mb.BoundLinear(mb.LinearNode(activation=ACT.GELU_ERF), V(lhs), V(rhs), V(x), residual=V(x)) as op:
            op.replay()
            op.quiesce_or_abort(20)
            once = x.clone()
            op.replay()
            op.quiesce_or_abort(20)
        check_forward(t, u, lhs, rhs, None, x0, ACT.GELU_ERF, once, None)
        check_forward(t, u, lhs, rhs, None, once, ACT.GELU_ERF, x, None)
        runs.append(x.clone())
    assert torch.equal(runs[0].view(torch.int16), runs[1].view(torch.int16))


@pytest.mark.parametrize("m", [5, 300])
def test_infinities_and_nan_stay_in_their_rows_and_columns(m):
    t = torch.bfloat16
    g = gen(5)
    lhs, rhs = rand(g, m, 128, dtype=t), rand(g, 128, 264, dtype=t)
    lhs[2, 7], rhs[9, 33] = float("nan"), float("inf")
    out = torch.zeros(m, 264, dtype=t, device="cuda")
    replay(mb.BoundLinear(mb.LinearNode(), V(lhs), V(rhs), V(out)))
    want = lhs.double() @ rhs.double()
    assert torch.equal(out.isnan(), want.isnan()) and torch.equal(out.isinf(), want.isinf())
    assert torch.equal(out[want.isinf()].double(), want[want.isinf()])


def test_activations_at_infinity():
    """One column times +-big: the activations' limits, not inf / inf; NaN stays."""
    t = torch.float16
    x = torch.tensor([[float("inf")], [-float("inf")], [float("nan")], [60000.0], [-60000.0], [0.0]], dtype=t, device="cuda")
    one = torch.ones(1, 16, dtype=t, device="cuda")
    for act in list(ACT)[1:]:
        out = torch.zeros(6, 16, dtype=t, device="cuda")
        replay(mb.BoundLinear(mb.LinearNode(activation=act), V(x), V(one), V(out)))
        col = out[:, 0].tolist()
        high = 6.0 if act == ACT.RELU6 else None
        assert col[0] == (high or float("inf")) and col[1] == 0 and col[2] != col[2]
        assert col[3] == (high or 60000.0) and col[4] == 0 and col[5] == 0


def test_handles_of_many_sizes_live_together():
    """Products of different shapes, all bound before the first runs, in both orders."""
    t, u = TYPES["bf16"]
    g = gen(13)
    made = []
    for m, n, k in [(128, 1024, 512), (1, 512, 512), (40, 2048, 256), (300, 512, 64), (16, 128, 4096)]:
        lhs, rhs = rand(g, m, k, dtype=t), rand(g, k, n, dtype=t, scale=k ** -0.5)
        out = torch.zeros(m, n, dtype=t, device="cuda")
        made.append((mb.BoundLinear(mb.LinearNode(), V(lhs), V(rhs), V(out)), lhs, rhs, out))
    for order in (made, made[::-1]):
        for op, lhs, rhs, out in order:
            out.zero_()
            torch.cuda.synchronize()
            op.replay()
        for op, lhs, rhs, out in order:
            op.quiesce_or_abort(20)
            check_forward(t, u, lhs, rhs, None, None, ACT.NONE, out, None)
    for op, *_ in made:
        op.close()


def test_offsets_past_32_bits():
    """Rows whose element offsets pass 2^31: output, residual and lhs by row pitch."""
    t, u = TYPES["bf16"]
    g = gen(6)
    rows, pitch = 5, 3 << 28
    big = torch.empty((rows - 1) * pitch + 4096, dtype=t, device="cuda")
    lhs = big.as_strided((rows, 128), (pitch, 1), 0)
    out = big.as_strided((rows, 264), (pitch, 1), 512)
    lhs.copy_(rand(g, rows, 128))
    rhs = rand(g, 128, 264, dtype=t, scale=0.1)
    out.zero_()
    replay(mb.BoundLinear(mb.LinearNode(), V(lhs), V(rhs), V(out)))
    check_forward(t, u, lhs, rhs, None, None, ACT.NONE, out, None)


def test_streams_and_graph_capture():
    t, u = TYPES["bf16"]
    g = gen(7)
    lhs, rhs = rand(g, 77, 515, dtype=t), rand(g, 515, 1001, dtype=t, scale=0.05)
    out = torch.zeros(77, 1001, dtype=t, device="cuda")
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with mb.BoundLinear(mb.LinearNode(), V(lhs), V(rhs), V(out)) as op:
        for s in (s1, s2, s1):
            op.replay(s.cuda_stream)  # packs into the handle's workspace: runs follow one another
        op.quiesce_or_abort(20)
        check_forward(t, u, lhs, rhs, None, None, ACT.NONE, out, None)
        out.zero_()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            op.replay(torch.cuda.current_stream().cuda_stream)
        graph.replay()
        torch.cuda.synchronize()
        check_forward(t, u, lhs, rhs, None, None, ACT.NONE, out, None)
        del graph
        op.quiesce_or_abort(20)


# ---------------------------------------------------------------- gradient --
def grad_case(dtype, m, n, k, act, tl=False, tr=False, seed=0, only=None):
    t, u = TYPES[dtype]
    g = gen(seed)
    lhs = rand(g, k, m, dtype=t) if tl else rand(g, m, k, dtype=t)
    rhs = rand(g, n, k, dtype=t, scale=k ** -0.5) if tr else rand(g, k, n, dtype=t, scale=k ** -0.5)
    dy, pre = rand(g, m, n, dtype=t), rand(g, m, n, dtype=t, scale=2.0)
    d = {"d_lhs": torch.full_like(lhs, float("nan")), "d_rhs": torch.full_like(rhs, float("nan")),
         "d_bias": torch.full((n,), float("nan"), dtype=t, device="cuda")}
    if only:
        d = {only: d[only]}
    node = mb.LinearNode(transpose_lhs=tl, transpose_rhs=tr, activation=act)
    replay(mb.BoundLinearGrad(node, V(dy), V(lhs), V(rhs), pre=V(pre) if act else None, **{q: V(x) for q, x in d.items()}))
    a, b = (lhs.t() if tl else lhs).double(), (rhs.t() if tr else rhs).double()
    slope = act64(act, pre.double())[1]
    dp = dy.double() * slope
    off = (u * dp.abs() + 2.0 ** -18 * dy.double().abs()) if act else torch.zeros_like(dp)
    if "d_lhs" in d:
        want, tol = dp @ b.t(), off @ b.t().abs() + (n + 1) * 2.0 ** -23 * (dp.abs() @ b.t().abs())
        check(d["d_lhs"].t() if tl else d["d_lhs"], want, u * want.abs() + tol * (1 + u) + TINY, "d_lhs")
    if "d_rhs" in d:
        want, tol = a.t() @ dp, a.t().abs() @ off + (m + 1) * 2.0 ** -23 * (a.t().abs() @ dp.abs())
        check(d["d_rhs"].t() if tr else d["d_rhs"], want, u * want.abs() + tol * (1 + u) + TINY, "d_rhs")
    if "d_bias" in d:
        want = dp.sum(0)
        tol = u * want.abs() + (2.0 ** -18 + (m + 1) * 2.0 ** -24) * (dp.abs() + dy.double().abs()).sum(0)
        check(d["d_bias"], want, tol + TINY, "d_bias")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 16, 24), (5, 264, 515), (130, 200, 264), (300, 520, 1000), (515, 1001, 77)])
@pytest.mark.parametrize("act", [ACT.NONE, ACT.GELU_TANH])
def test_gradient_shapes(dtype, m, n, k, act):
    grad_case(dtype, m, n, k, act, seed=m)
    grad_case(dtype, m, n, k, act, tr=True, seed=m + 1)


@pytest.mark.parametrize("act", list(ACT))
def test_gradient_activations(act):
    grad_case("f16", 70, 136, 72, act, tl=True, seed=int(act))


@pytest.mark.parametrize("only", ["d_lhs", "d_rhs", "d_bias"])
def test_one_gradient_alone(only):
    grad_case("bf16", 66, 136, 72, ACT.SILU, only=only)


def test_gradient_of_no_rows_is_zero():
    t = torch.bfloat16
    e = lambda *s: torch.empty(*s, dtype=t, device="cuda")  # noqa: E731
    d_rhs, d_bias = e(64, 24).fill_(3), e(24).fill_(3)
    replay(mb.BoundLinearGrad(mb.LinearNode(), V(e(0, 24)), V(e(0, 64)), V(e(64, 24)), d_rhs=V(d_rhs), d_bias=V(d_bias)))
    assert not d_rhs.any() and not d_bias.any()


@pytest.mark.parametrize("act", [ACT.GELU_ERF, ACT.GELU_TANH, ACT.SILU])
def test_gradient_against_differences(act):
    """The directional derivative of sum(out * G) by central differences of the
    64-bit formula at step h, whose own error is below 1e-6 relative here; the
    operator's gradient carries one rounding of d_pre and one of the result,
    which the direction's dot product averages: 4 u of the absolute sum."""
    t, u = TYPES["f16"]
    g = gen(8)
    m, n, k = 40, 72, 56
    lhs, rhs, bias, dy = rand(g, m, k, dtype=t), rand(g, k, n, dtype=t, scale=0.13), rand(g, n, dtype=t), rand(g, m, n, dtype=t)
    out, pre = torch.empty(m, n, dtype=t, device="cuda"), torch.empty(m, n, dtype=t, device="cuda")
    node = mb.LinearNode(activation=act)
    replay(mb.BoundLinear(node, V(lhs), V(rhs), V(out), bias=V(bias), pre=V(pre)))
    d = [torch.empty_like(lhs), torch.empty_like(rhs), torch.empty_like(bias)]
    replay(mb.BoundLinearGrad(node, V(dy), V(lhs), V(rhs), d_lhs=V(d[0]), d_rhs=V(d[1]), d_bias=V(d[2]), pre=V(pre)))
    loss = lambda a, b, c: (act64(act, a @ b + c)[0] * dy.double()).sum()  # noqa: E731
    at = [lhs.double(), rhs.double(), bias.double()]
    for i in range(3):
        v = torch.randn(at[i].shape, generator=g, device="cuda", dtype=torch.float64)
        h = 1e-4
        hi, lo = list(at), list(at)
        hi[i], lo[i] = at[i] + h * v, at[i] - h * v
        want = float((loss(*hi) - loss(*lo)) / (2 * h))
        got = float((d[i].double() * v).sum())
        # pre was rounded before the derivative was taken there: u |pre| times a curvature of at most 1.2
        assert abs(got - want) <= 4 * u * float((d[i].double() * v).abs().sum()) + 1e-6 * abs(want), (i, got, want)


# --------------------------------------------------------------------- f32 --
def rel(x, y):
    return float((x.double() - y).norm() / y.norm())


@pytest.mark.parametrize("m,n,k", [(1, 64, 128), (7, 130, 515), (300, 520, 264), (129, 1001, 77)])
@pytest.mark.parametrize("act", [ACT.NONE, ACT.GELU_ERF, ACT.SILU])
def test_f32_operands(m, n, k, act):
    """The MatMul node's StrictFp32 mode under the same layer, its bound 1e-5."""
    g = gen(9)
    lhs, rhs, b, r = rand(g, m, k), rand(g, k, n, scale=k ** -0.5), rand(g, n), rand(g, m, n)
    want_pre = lhs.double() @ rhs.double() + b.double()
    want = act64(act, want_pre)[0]
    for residual, keep in [(False, False), (True, False), (True, True)]:
        out, pre = torch.empty(m, n, device="cuda"), torch.empty(m, n, device="cuda")
        replay(mb.BoundLinear(mb.LinearNode(activation=act), V(lhs), V(rhs), V(out), bias=V(b),
                              residual=V(r) if residual else None, pre=V(pre) if keep else None))
        assert rel(out, want + r.double() if residual else want) <= 1e-5
        assert not keep or rel(pre, want_pre) <= 1e-5
    x = r.clone()
    replay(mb.BoundLinear(mb.LinearNode(activation=act), V(lhs), V(rhs), V(x), bias=V(b), residual=V(x)))
    assert rel(x, want + r.double()) <= 1e-5


def test_f32_capture():
    """A captured f32 run, replayed after others; waiting and closing work as before it."""
    g = gen(14)
    lhs, rhs, r = rand(g, 300, 256), rand(g, 256, 264, scale=0.06), rand(g, 300, 264)
    out = torch.zeros(300, 264, device="cuda")
    op = mb.BoundLinear(mb.LinearNode(activation=ACT.SILU), V(lhs), V(rhs), V(out), residual=V(r))
    want = act64(ACT.SILU, lhs.double() @ rhs.double())[0] + r.double()
    op.replay()
    op.quiesce_or_abort(20)
    assert rel(out, want) <= 1e-5
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.replay(torch.cuda.current_stream().cuda_stream)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert rel(out, want) <= 1e-5
    op.quiesce_or_abort(20)
    del graph
    op.close()


@pytest.mark.parametrize("tr", [False, True])
def test_f32_gradient(tr):
    g = gen(10)
    m, n, k = 130, 264, 136
    lhs, rhs, dy, pre = rand(g, m, k), rand(g, n, k) if tr else rand(g, k, n), rand(g, m, n), rand(g, m, n)
    d = [torch.empty_like(lhs), torch.empty_like(rhs), torch.empty(n, device="cuda")]
    node = mb.LinearNode(transpose_rhs=tr, activation=ACT.GELU_TANH)
    replay(mb.BoundLinearGrad(node, V(dy), V(lhs), V(rhs), d_lhs=V(d[0]), d_rhs=V(d[1]), d_bias=V(d[2]), pre=V(pre)))
    dp = dy.double() * act64(ACT.GELU_TANH, pre.double())[1]
    b = (rhs.t() if tr else rhs).double()
    assert rel(d[0], dp @ b.t()) <= 1e-5
    assert rel(d[1].t() if tr else d[1], lhs.double().t() @ dp) <= 1e-5
    assert rel(d[2], dp.sum(0)) <= 1e-5


def test_tf32_mode():
    g = gen(11)
    lhs, rhs, r = rand(g, 300, 256), rand(g, 256, 264), rand(g, 300, 264)
    out = torch.empty(300, 264, device="cuda")
    node = mb.LinearNode(math_mode=mb.KernelMathMode.Tf32, accuracy=mb.AccuracyContract.AllowTf32)
    replay(mb.BoundLinear(node, V(lhs), V(rhs), V(out), residual=V(r)))
    assert rel(out, lhs.double() @ rhs.double() + r.double()) <= 2e-3


F32_SHAPES = [(1, 64, 64), (1, 1001, 4096), (2, 130, 515), (3, 129, 1), (8, 300, 2048), (9, 515, 77), (16, 500, 4000),
              (17, 512, 512), (100, 1000, 4000), (129, 77, 5000), (300, 515, 77), (260, 264, 4099), (1, 1, 1), (40, 1, 900)]


@pytest.mark.parametrize("m,n,k", F32_SHAPES)
@pytest.mark.parametrize("tl,tr", [(False, False), (False, True), (True, False)])
def test_f32_layouts(m, n, k, tl, tr):
    """Odd pitches, few rows, a long contraction over few tiles: each in both directions."""
    g = gen(m + n + k)
    lhs, rhs = rand(g, *((k, m) if tl else (m, k))), rand(g, *((n, k) if tr else (k, n)), scale=k ** -0.5)
    b, r = rand(g, n), rand(g, m, n)
    a64, b64 = (lhs.t() if tl else lhs).double(), (rhs.t() if tr else rhs).double()
    node = mb.LinearNode(transpose_lhs=tl, transpose_rhs=tr)
    out, pre = torch.full((m, n), float("nan"), device="cuda"), torch.full((m, n), float("nan"), device="cuda")
    replay(mb.BoundLinear(node, V(lhs), V(rhs), V(out), bias=V(b)))
    assert rel(out, a64 @ b64 + b.double()) <= 1e-5
    replay(mb.BoundLinear(node, V(lhs), V(rhs), V(pre)))
    assert rel(pre, a64 @ b64) <= 1e-5
    replay(mb.BoundLinear(node, V(lhs), V(rhs), V(out), bias=V(b), residual=V(r), pre=V(pre)))
    assert rel(out, a64 @ b64 + b.double() + r.double()) <= 1e-5
    assert rel(pre, a64 @ b64 + b.double()) <= 1e-5
    dy, d_lhs, d_rhs = rand(g, m, n), torch.full_like(lhs, float("nan")), torch.full_like(rhs, float("nan"))
    replay(mb.BoundLinearGrad(node, V(dy), V(lhs), V(rhs), d_lhs=V(d_lhs), d_rhs=V(d_rhs)))
    dy64 = dy.double()
    assert rel(d_lhs.t() if tl else d_lhs, dy64 @ b64.t()) <= 1e-5
    assert rel(d_rhs.t() if tr else d_rhs, a64.t() @ dy64) <= 1e-5


@pytest.mark.parametrize("m", [4, 12, 200])
def test_f32_views(m):
    """Column blocks at odd offsets, reversed rows, a transposed output; what lies between them stays."""
    g = gen(m)
    n, k = 140, 2050
    wide, weights = rand(g, 2 * m, k + 7), rand(g, n + 3, k + 5, scale=k ** -0.5)
    lhs, rhs = wide[::2, 3:3 + k], weights[1:n + 1, 2:2 + k]
    buf = torch.full((n, m + 3), 7.0, device="cuda")
    out = buf[:, 1:m + 1].t()
    replay(mb.BoundLinear(mb.LinearNode(transpose_rhs=True), V(lhs), V(rhs), V(out)))
    assert rel(out, lhs.double() @ rhs.double().t()) <= 1e-5
    assert bool((buf[:, 0] == 7).all()) and bool((buf[:, m + 1:] == 7).all())


def test_f32_empty_contraction():
    g = gen(15)
    b, r = rand(g, 24), rand(g, 7, 24)
    out = torch.empty(7, 24, device="cuda")
    lhs, rhs = torch.empty(7, 0, device="cuda"), torch.empty(0, 24, device="cuda")
    replay(mb.BoundLinear(mb.LinearNode(activation=ACT.RELU), V(lhs), V(rhs), V(out), bias=V(b), residual=V(r)))
    assert torch.equal(out, b.relu() + r)


@pytest.mark.parametrize("m,n,k", [(5, 64, 512), (100, 264, 4002)])
def test_f32_infinities_stay_in_their_rows_and_columns(m, n, k):
    g = gen(16)
    lhs, rhs = rand(g, m, k), rand(g, n, k)
    lhs[2, k - 1], rhs[7, 0] = float("inf"), float("nan")
    out = torch.empty(m, n, device="cuda")
    replay(mb.BoundLinear(mb.LinearNode(transpose_rhs=True), V(lhs), V(rhs), V(out)))
    assert not bool(torch.isfinite(out[2]).any()) and bool(torch.isnan(out[:, 7]).all())
    keep = torch.ones(m, n, dtype=torch.bool, device="cuda")
    keep[2], keep[:, 7] = False, False
    assert bool(torch.isfinite(out[keep]).all())
