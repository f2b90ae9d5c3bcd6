"""Tokens sorted by expert, back, and the experts' products, on the GPU.

The sort is integers and copies: equal to a plain loop over the assignments.
The sums are bounded as in the linear layer's tests: u the type's unit
roundoff, f32 sums of n terms off by at most n 2^-24 (n 2^-23 on the tensor
core, which may truncate) of the sum of magnitudes.
"""
import numpy as np
import pytest
import torch

import momiru_b200 as mb
from test_linear_gpu import ACT, TINY, TYPES, V, act64, check, gen, rand, replay

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda_lib")]
ALL = dict(TYPES, f32=(torch.float32, 2.0 ** -24))
NAN = float("nan")


def sort_plain(ids, experts, align, rows):
    slots = np.full(ids.size, -1, np.int32)
    sources = np.full(rows, -1, np.int32)
    counts = np.array([(ids == e).sum() for e in range(experts)], np.int32)
    offsets = np.zeros(experts + 1, np.int32)
    offsets[1:] = np.cumsum((counts + align - 1) // align * align)
    at = offsets[:-1].copy()
    for i, e in enumerate(ids.ravel()):
        if 0 <= e < experts:
            slots[i] = at[e]
            sources[at[e]] = i
            at[e] += 1
    return slots.reshape(ids.shape), sources, offsets, counts


def routing(kind, tokens, top_k, experts, seed):
    g = np.random.default_rng(seed)
    if kind == "even":
        ids = np.stack([g.permutation(max(experts, top_k))[:top_k] % experts for _ in range(tokens)]) if tokens else np.zeros((0, top_k))
    elif kind == "one":
        ids = np.full((tokens, top_k), experts - 1)
    elif kind == "dropped":
        ids = g.integers(-3, experts + 3, (tokens, top_k))
        ids[g.random((tokens, top_k)) < 0.1] = 2 ** 31 - 1
    elif kind == "none":
        ids = np.full((tokens, top_k), -1)
    else:  # a few popular experts
        ids = np.minimum(g.geometric(0.4, (tokens, top_k)) - 1, experts - 1)
    return ids.astype(np.int32)


def dispatch(ids, experts, align, x, top_k=None):
    tokens, top_k = ids.shape
    lay = mb.ExpertLayout.empty(tokens, top_k, experts, align)
    rows = torch.full((lay.rows, x.shape[1]), NAN, dtype=x.dtype, device="cuda")
    for v in (lay.slots, lay.sources, lay.offsets, lay.counts):
        v.torch_view().fill_(-7)
    ids_t = torch.from_numpy(ids).cuda()
    replay(mb.BoundDispatch(lay, V(ids_t), V(x), V(rows)))
    return lay, rows


def check_dispatch(ids, experts, align, x, lay, rows):
    slots, sources, offsets, counts = sort_plain(ids, experts, align, lay.rows)
    for got, want in ((lay.slots, slots), (lay.sources, sources), (lay.offsets, offsets), (lay.counts, counts)):
        assert np.array_equal(got.to_host(), want)
    src = torch.from_numpy(sources).cuda().long()
    want = torch.where((src >= 0)[:, None], x[src.clamp(min=0) // ids.shape[1]] if x.shape[0] else rows * 0, torch.zeros((), dtype=x.dtype, device="cuda"))
    assert torch.equal(rows, want)


@pytest.mark.parametrize("kind", ["even", "one", "dropped", "none", "few"])
@pytest.mark.parametrize("tokens,top_k,experts,align", [
    (1, 1, 1, 1), (1, 8, 64, 16), (5, 3, 7, 1), (33, 2, 5, 64), (257, 4, 40, 128), (700, 6, 300, 16), (3000, 2, 64, 128),
    (2500, 8, 1024, 1)])
def test_dispatch(kind, tokens, top_k, experts, align):
    ids = routing(kind, tokens, top_k, experts, tokens)
    x = rand(gen(1), tokens, 72, dtype=torch.bfloat16)
    check_dispatch(ids, experts, align, x, *dispatch(ids, experts, align, x))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("h", [1, 6, 64, 515, 1002, 4104])
def test_dispatch_row_widths(dtype, h):
    ids = routing("dropped", 41, 3, 9, h)
    x = rand(gen(2), 41, h, dtype=ALL[dtype][0])
    check_dispatch(ids, 9, 16, x, *dispatch(ids, 9, 16, x))


def test_dispatch_of_views():
    """x as a column block at an odd offset, ids transposed, rows inside a wider buffer that keeps its other columns."""
    ids = routing("few", 40, 2, 6, 0)
    wide = rand(gen(3), 40, 200, dtype=torch.float16)
    x = wide[:, 3:103]
    lay = mb.ExpertLayout.empty(40, 2, 6, 16)
    buf = torch.full((lay.rows, 111), 5.0, dtype=torch.float16, device="cuda")
    ids_t = torch.from_numpy(np.ascontiguousarray(ids.T)).cuda().t()
    replay(mb.BoundDispatch(lay, V(ids_t), V(x), V(buf[:, 5:105])))
    check_dispatch(ids, 6, 16, x, lay, buf[:, 5:105])
    assert bool((buf[:, :5] == 5).all()) and bool((buf[:, 105:] == 5).all())


def test_no_tokens():
    lay, rows = dispatch(np.zeros((0, 2), np.int32), 5, 64, torch.zeros(0, 16, device="cuda"))
    assert lay.rows == 0 and not lay.offsets.to_host().any() and not lay.counts.to_host().any()
    w = rand(gen(0), 5, 16, 8, dtype=torch.bfloat16)
    e = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device="cuda")  # noqa: E731
    replay(mb.BoundExpertLinear(mb.LinearNode(), lay, V(e(0, 16)), V(w), V(e(0, 8))))
    d_w, d_b = torch.ones_like(w), torch.ones(5, 8, dtype=torch.bfloat16, device="cuda")
    replay(mb.BoundExpertLinearGrad(mb.LinearNode(), lay, V(e(0, 8)), V(e(0, 16)), V(w), d_weights=V(d_w), d_bias=V(d_b)))
    assert not d_w.any() and not d_b.any()
    replay(mb.BoundCombine(lay, V(e(0, 16)), V(e(0, 16))))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("tokens,top_k,h", [(1, 1, 8), (1, 8, 2048), (37, 3, 515), (300, 6, 264), (65, 9, 1002)])
@pytest.mark.parametrize("weighted,residual", [(True, True), (False, False)])
def test_combine(dtype, tokens, top_k, h, weighted, residual):
    t, u = ALL[dtype]
    ids = routing("dropped", tokens, top_k, 12, h)
    lay, _ = dispatch(ids, 12, 16, torch.zeros(tokens, 8, device="cuda"))
    g = gen(4)
    rows = rand(g, lay.rows, h, dtype=t)
    rows[torch.from_numpy(lay.sources.to_host() < 0).cuda()] = NAN  # never read
    w = rand(g, tokens, top_k) if weighted else None
    if weighted:
        w[torch.from_numpy(lay.slots.to_host() < 0).cuda()] = NAN
    r = rand(g, tokens, h, dtype=t) if residual else None
    out = torch.full((tokens, h), NAN, dtype=t, device="cuda")
    replay(mb.BoundCombine(lay, V(rows), V(out), weights=V(w) if weighted else None, residual=V(r) if residual else None))
    slots = torch.from_numpy(lay.slots.to_host()).cuda().long()
    terms = rows.double()[slots.clamp(min=0)] * (w.double()[..., None] if weighted else 1)
    terms = torch.where((slots >= 0)[..., None], terms, 0.0)
    want, size = terms.sum(1), terms.abs().sum(1)
    if residual:
        want, size = want + r.double(), size + r.double().abs()
    check(out, want, u * want.abs() + (top_k + 1) * 2.0 ** -24 * size + TINY, "out")
    if residual:
        replay(mb.BoundCombine(lay, V(rows), V(r), weights=V(w) if weighted else None, residual=V(r)))
        assert torch.equal(r, out)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("tokens,top_k,h", [(1, 1, 8), (3, 8, 2048), (37, 3, 515), (300, 6, 264), (65, 9, 1002)])
def test_combine_gradient(dtype, tokens, top_k, h):
    t, u = ALL[dtype]
    ids = routing("dropped", tokens, top_k, 12, h)
    lay, _ = dispatch(ids, 12, 64, torch.zeros(tokens, 8, device="cuda"))
    g = gen(5)
    rows, dy, w = rand(g, lay.rows, h, dtype=t), rand(g, tokens, h, dtype=t), rand(g, tokens, top_k)
    d_rows, d_w = torch.full_like(rows, NAN), torch.full_like(w, NAN)
    replay(mb.BoundCombineGrad(lay, V(dy), V(rows), V(w), d_rows=V(d_rows), d_weights=V(d_w)))
    slots, src = (torch.from_numpy(v.to_host()).cuda().long() for v in (lay.slots, lay.sources))
    want = dy.double()[src.clamp(min=0) // top_k] * w.double().reshape(-1)[src.clamp(min=0)][:, None]
    want = torch.where((src >= 0)[:, None], want, 0.0)
    check(d_rows, want, u * want.abs() + 2.0 ** -24 * want.abs() + TINY, "d_rows")
    terms = torch.where((slots >= 0)[..., None], rows.double()[slots.clamp(min=0)] * dy.double()[:, None], 0.0)
    check(d_w, terms.sum(2), (h + 1) * 2.0 ** -24 * terms.abs().sum(2) + 1e-30, "d_weights")
    # each alone gives the same
    only_rows, only_w = torch.empty_like(rows), torch.empty_like(w)
    replay(mb.BoundCombineGrad(lay, V(dy), None, V(w), d_rows=V(only_rows)))
    replay(mb.BoundCombineGrad(lay, V(dy), V(rows), None, d_weights=V(only_w)))
    assert torch.equal(only_rows, d_rows) and torch.equal(only_w, d_w)


def test_combine_gradient_against_differences():
    """sum(out * G) differs linearly in rows and in weights, so a difference of
    any step is the derivative: rounding alone, 2^-24 of the absolute sums per
    term, remains."""
    ids = routing("dropped", 30, 4, 6, 0)
    lay, _ = dispatch(ids, 6, 16, torch.zeros(30, 8, device="cuda"))
    g = gen(6)
    rows, dy, w = rand(g, lay.rows, 48), rand(g, 30, 48), rand(g, 30, 4)
    d_rows, d_w = torch.empty_like(rows), torch.empty_like(w)
    replay(mb.BoundCombineGrad(lay, V(dy), V(rows), V(w), d_rows=V(d_rows), d_weights=V(d_w)))
    slots = torch.from_numpy(lay.slots.to_host()).cuda().long()

    def loss(r, a):
        terms = torch.where((slots >= 0)[..., None], r[slots.clamp(min=0)] * a[..., None], 0.0)
        return (terms.sum(1) * dy.double()).sum()

    vr, vw = torch.randn(rows.shape, generator=g, device="cuda").double(), torch.randn(w.shape, generator=g, device="cuda").double()
    for got, hi, lo, size in [
            ((d_rows.double() * vr).sum(), loss(rows.double() + vr, w.double()), loss(rows.double() - vr, w.double()), (d_rows.double() * vr).abs().sum()),
            ((d_w.double() * vw).sum(), loss(rows.double(), w.double() + vw), loss(rows.double(), w.double() - vw), (rows.double().abs().sum() * 8))]:
        assert abs(float(got - (hi - lo) / 2)) <= 50 * 2.0 ** -24 * float(size)


def expert_setup(dtype, kind, tokens, top_k, experts, align, k, n, tr, seed=0):
    t, u = TYPES[dtype]
    ids = routing(kind, tokens, top_k, experts, seed)
    g = gen(seed)
    lay, rows = dispatch(ids, experts, align, rand(g, tokens, k, dtype=t))
    w = rand(g, experts, n, k, dtype=t, scale=k ** -0.5) if tr else rand(g, experts, k, n, dtype=t, scale=k ** -0.5)
    return t, u, g, lay, rows, w


EXPERT_SHAPES = [  # tokens, top_k, experts, align, k, n: few rows an expert, many, uneven, odd widths
    (1, 1, 1, 1, 64, 64), (3, 2, 8, 16, 136, 72), (16, 4, 32, 1, 264, 520), (40, 2, 6, 128, 77, 131), (200, 2, 3, 64, 200, 264),
    (700, 2, 4, 128, 320, 512), (900, 1, 2, 1, 131, 77), (1500, 2, 5, 16, 64, 1000)]


@pytest.mark.parametrize("kind", ["even", "dropped", "few"])
@pytest.mark.parametrize("tokens,top_k,experts,align,k,n", EXPERT_SHAPES)
def test_expert_products(kind, tokens, top_k, experts, align, k, n):
    for dtype, tr, act, bias in (("bf16", False, ACT.GELU_TANH, True), ("f16", True, ACT.SILU, False)):
        t, u, g, lay, rows, w = expert_setup(dtype, kind, tokens, top_k, experts, align, k, n, tr, tokens)
        counts = lay.counts.to_host()
        w[torch.from_numpy(counts == 0).cuda()] = NAN  # unused experts are not multiplied
        b = rand(g, experts, n, dtype=t) if bias else None
        out, pre = (torch.full((lay.rows, n), NAN, dtype=t, device="cuda") for _ in range(2))
        node = mb.LinearNode(transpose_rhs=tr, activation=act)
        replay(mb.BoundExpertLinear(node, lay, V(rows), V(w), V(out), bias=V(b) if bias else None, pre=V(pre)))
        wf = w.double().transpose(1, 2) if tr else w.double()
        held = torch.from_numpy(lay.sources.to_host() >= 0).cuda()
        assert not out[~held].any() and not pre[~held].any()
        for e, (o, c) in enumerate(zip(lay.offsets.to_host(), counts)):
            x = rows[o:o + c].double()
            want_pre = x @ wf[e] if c else x.new_zeros(0, n)
            acc = (k + 1) * 2.0 ** -23 * (x.abs() @ wf[e].abs() + (b[e].double().abs() if bias else 0)) if c else want_pre
            want_pre = want_pre + (b[e].double() if bias else 0)
            want = act64(act, want_pre)[0]
            if c:
                check(pre[o:o + c], want_pre, u * want_pre.abs() + acc + TINY, "pre")
                check(out[o:o + c], want, u * want.abs() + 1.13 * acc + 2.0 ** -19 * (1 + want_pre.abs()) + TINY, "out")


@pytest.mark.parametrize("kind", ["even", "dropped", "few", "one", "none"])
@pytest.mark.parametrize("tokens,top_k,experts,align,k,n", [
    (1, 1, 3, 64, 64, 64), (40, 2, 6, 128, 77, 131), (200, 2, 3, 64, 200, 264), (700, 2, 4, 128, 320, 512)])
def test_expert_gradient(kind, tokens, top_k, experts, align, k, n):
    for dtype, tr, act in (("bf16", False, ACT.GELU_ERF), ("f16", True, ACT.NONE)):
        t, u, g, lay, rows, w = expert_setup(dtype, kind, tokens, top_k, experts, align, k, n, tr, tokens)
        held = torch.from_numpy(lay.sources.to_host() >= 0).cuda()
        dy, pre = rand(g, lay.rows, n, dtype=t) * held[:, None], rand(g, lay.rows, n, dtype=t)
        d_rows, d_w = torch.full_like(rows, NAN), torch.full_like(w, NAN)
        d_b = torch.full((experts, n), NAN, dtype=t, device="cuda")
        node = mb.LinearNode(transpose_rhs=tr, activation=act)
        replay(mb.BoundExpertLinearGrad(node, lay, V(dy), V(rows), V(w), d_rows=V(d_rows), d_weights=V(d_w),
                                        d_bias=V(d_b), pre=V(pre) if act else None))
        wf = (w.transpose(1, 2) if tr else w).double()
        assert not d_rows[~held].any()
        for e, (o, c) in enumerate(zip(lay.offsets.to_host(), lay.counts.to_host())):
            x, y = rows[o:o + c].double(), dy[o:o + c].double()
            dp = y * act64(act, pre[o:o + c].double())[1]
            off = u * dp.abs() + 2.0 ** -18 * y.abs() if act else torch.zeros_like(dp)
            if c:
                want, tol = dp @ wf[e].t(), (off + (n + 1) * 2.0 ** -23 * dp.abs()) @ wf[e].t().abs()
                check(d_rows[o:o + c], want, u * want.abs() + tol * (1 + u) + TINY, "d_rows")
            want, tol = x.t() @ dp, x.t().abs() @ (off + (c + 1) * 2.0 ** -23 * dp.abs())
            check((d_w[e].t() if tr else d_w[e]), want, u * want.abs() + tol * (1 + u) + TINY, "d_weights")
            want = dp.sum(0)
            check(d_b[e], want, u * want.abs() + (2.0 ** -18 + (c + 1) * 2.0 ** -24) * (dp.abs() + y.abs()).sum(0) + TINY, "d_bias")


def test_offsets_past_32_bits():
    """Sorted rows a long pitch apart: the last ones lie beyond 2^31 elements."""
    pitch, h, tokens = 3 << 28, 64, 3
    ids = np.array([[0, 1], [1, 0], [1, -1]], np.int32)
    x = rand(gen(16), tokens, h, dtype=torch.bfloat16)
    lay = mb.ExpertLayout.empty(tokens, 2, 2, 1)
    big = torch.empty((lay.rows - 1) * pitch + h, dtype=torch.bfloat16, device="cuda")
    rows = big.as_strided((lay.rows, h), (pitch, 1))
    replay(mb.BoundDispatch(lay, V(torch.from_numpy(ids).cuda()), V(x), V(rows)))
    check_dispatch(ids, 2, 1, x, lay, rows)
    y, w = torch.empty_like(x), torch.ones(tokens, 2, device="cuda")
    replay(mb.BoundCombine(lay, V(rows), V(y), weights=V(w)))
    assert torch.equal(y, x * torch.tensor([[2.0], [2.0], [1.0]], device="cuda", dtype=torch.bfloat16))
    d_w = torch.empty_like(w)
    replay(mb.BoundCombineGrad(lay, V(x), V(rows), V(w), d_rows=V(rows.clone()), d_weights=V(d_w)))
    square = (x.double() ** 2).sum(1)
    want = torch.stack((square, square * torch.tensor([1, 1, 0], device="cuda")), 1)
    check(d_w, want, (h + 1) * 2.0 ** -24 * want + 1e-30, "d_weights")
    k = rand(gen(17), 2, h, 24, dtype=torch.bfloat16)
    out = torch.empty(lay.rows, 24, dtype=torch.bfloat16, device="cuda")
    replay(mb.BoundExpertLinear(mb.LinearNode(), lay, V(rows), V(k), V(out)))
    same = torch.empty_like(out)
    replay(mb.BoundExpertLinear(mb.LinearNode(), lay, V(rows.contiguous()), V(k), V(same)))
    assert torch.equal(out, same)


def test_equal_runs_give_equal_bits():
    t, u, g, lay, rows, w = expert_setup("bf16", "few", 600, 2, 5, 64, 136, 264, False)
    outs = []
    for _ in range(3):
        out = torch.empty(lay.rows, 264, dtype=t, device="cuda")
        replay(mb.BoundExpertLinear(mb.LinearNode(), lay, V(rows), V(w), V(out)))
        d_w, d_b = torch.empty_like(w), torch.empty(5, 264, dtype=t, device="cuda")
        replay(mb.BoundExpertLinearGrad(mb.LinearNode(), lay, V(out), V(rows), V(w), d_weights=V(d_w), d_bias=V(d_b)))
        outs.append((out, d_w, d_b))
    for o in outs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(o, outs[0]))


def test_a_layout_of_nonsense_touches_nothing_outside():
    """Counts, offsets and slots that no sort made (out of range either way):
    every access is bounded by the buffers, whose guard rows keep their values."""
    tokens, k, n, experts = 64, 64, 136, 4
    t = torch.bfloat16
    g = gen(15)
    rows_n = mb.ExpertLayout.capacity(tokens, 2, experts, 64)
    bad = torch.tensor([2 ** 30, -5, rows_n + 7, 10 ** 9], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([rows_n - 3, -64, 10 ** 9, 64, 2 ** 30], dtype=torch.int32, device="cuda")
    slots = torch.full((tokens, 2), 10 ** 9, dtype=torch.int32, device="cuda")
    slots[::2] = rows_n
    sources = torch.full((rows_n,), -1, dtype=torch.int32, device="cuda")
    lay = mb.ExpertLayout(tokens, 2, experts, 64, V(slots), V(sources), V(offsets), V(bad))
    rows = rand(g, rows_n, k, dtype=t)
    for experts_rows in (1, 2):  # twice: nothing is left behind either
        w = rand(g, experts, k, n, dtype=t)
        buf = torch.full((rows_n + 512, n), 7.0, dtype=t, device="cuda")
        replay(mb.BoundExpertLinear(mb.LinearNode(), lay, V(rows), V(w), V(buf[256:256 + rows_n])))
        assert bool((buf[:256] == 7).all()) and bool((buf[256 + rows_n:] == 7).all())
        d_w, d_b = torch.empty_like(w), torch.empty(experts, n, dtype=t, device="cuda")
        replay(mb.BoundExpertLinearGrad(mb.LinearNode(), lay, V(buf[256:256 + rows_n]), V(rows), V(w), d_weights=V(d_w), d_bias=V(d_b)))
    y = torch.ones(tokens, k, dtype=t, device="cuda")
    replay(mb.BoundCombine(lay, V(rows), V(y)))
    assert not y.any()
    d_rows, d_wt = torch.ones_like(rows), torch.ones(tokens, 2, device="cuda")
    replay(mb.BoundCombineGrad(lay, V(rand(g, tokens, k, dtype=t)), V(rows), None, d_rows=V(d_rows), d_weights=V(d_wt)))
    assert not d_rows.any() and not d_wt.any()


def test_layout_changes_between_replays():
    """One bound chain, other ids on every replay: nothing of the previous routing stays."""
    tokens, k, n, experts = 50, 72, 136, 6
    t = torch.bfloat16
    g = gen(12)
    lay = mb.ExpertLayout.empty(tokens, 2, experts, 16)
    ids, x = torch.zeros(tokens, 2, dtype=torch.int32, device="cuda"), torch.zeros(tokens, k, dtype=t, device="cuda")
    rows, hid = torch.empty(lay.rows, k, dtype=t, device="cuda"), torch.empty(lay.rows, n, dtype=t, device="cuda")
    w, y = rand(g, experts, k, n, dtype=t, scale=0.1), torch.empty(tokens, n, dtype=t, device="cuda")
    ops = [mb.BoundDispatch(lay, V(ids), V(x), V(rows)),
           mb.BoundExpertLinear(mb.LinearNode(), lay, V(rows), V(w), V(hid)), mb.BoundCombine(lay, V(hid), V(y))]
    for seed, kind in enumerate(("even", "one", "dropped", "none", "few")):
        r = routing(kind, tokens, 2, experts, seed)
        ids.copy_(torch.from_numpy(r))
        x.copy_(rand(g, tokens, k))
        for op in ops:
            op.replay()
        for op in ops:
            op.quiesce_or_abort(20)
        check_dispatch(r, experts, 16, x, lay, rows)
        want = torch.zeros(tokens, n, dtype=torch.float64, device="cuda")
        size = torch.zeros_like(want)
        for j in range(2):
            e = torch.from_numpy(r[:, j]).cuda().long()
            ok = (e >= 0) & (e < experts)
            term = torch.einsum("tk,tkn->tn", x.double(), w.double()[e.clamp(0, experts - 1)])
            want += torch.where(ok[:, None], term, 0.0)
            size += torch.where(ok[:, None], torch.einsum("tk,tkn->tn", x.double().abs(), w.double().abs()[e.clamp(0, experts - 1)]), 0.0)
        # each product is rounded to bf16 once, then their sum
        check(y, want, 2.0 ** -8 * (want.abs() + 1.01 * size) + (k + 3) * 2.0 ** -23 * size + TINY, kind)
    for op in ops:
        op.close()
