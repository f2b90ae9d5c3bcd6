"""The cases by which the linear, expert-routing and expert-product operators are measured.

A case names one operator and its sizes. `prepare` makes its inputs, `run` is
one pass over them: in the plain form (elementary torch operations in 32 bits,
rounded once) or through momiru_b200, and `exact` is the same result from the
definition in 64 bits.

  linear        out = act(lhs @ rhs + bias) + residual, `pre` (the value before
                the activation) kept for training where asked
  linear_grad   its gradient: d_lhs, d_rhs, d_bias from d_out and pre
  dispatch      tokens sorted by expert: the layout and the gathered rows
  combine       the rows back to their tokens, weighted, plus a residual
  combine_grad  its gradient: d_rows and d_weights
  expert        each expert's product over its segment of the sorted rows
  expert_grad   its gradient: d_rows, d_weights, d_bias

Segments start at multiples of `align` rows; a row that holds no token is zero.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
ACTS = ("none", "relu", "gelu_erf", "gelu_tanh", "silu")

LINEAR_WORK = 4096 * 4096 * 11008  # the largest product drawn, in multiply-adds


def listed():
    return [
        # one token through a down projection, its residual added: serving, bound by the weights' bytes
        dict(name="linear_token_bf16", op="linear", m=1, n=4096, k=11008, dtype="bf16", act="none", bias=False,
             residual=True, pre=False, wt=True),
        # a short ragged batch with sizes that no tile or 16-byte pitch divides
        dict(name="linear_odd_f16", op="linear", m=77, n=1001, k=515, dtype="f16", act="gelu_erf", bias=True,
             residual=True, pre=False, wt=False),
        # an up projection over a training batch, the value before the activation kept
        dict(name="linear_train_bf16", op="linear", m=4096, n=11008, k=4096, dtype="bf16", act="gelu_tanh", bias=True,
             residual=False, pre=True, wt=True),
        # the framework's own type, in its fp32-accurate mode
        dict(name="linear_f32", op="linear", m=1024, n=4096, k=1024, dtype="f32", act="silu", bias=True,
             residual=True, pre=False, wt=False),
        # the gradient of a square projection over a training batch
        dict(name="linear_grad_bf16", op="linear_grad", m=4096, n=4096, k=4096, dtype="bf16", act="gelu_tanh",
             bias=True, wt=True),
        # eight decoding sequences sorted over many experts: latency
        dict(name="dispatch_decode_bf16", op="dispatch", tokens=8, top_k=8, experts=64, h=2048, dtype="bf16", align=16,
             drop=0.0),
        # a long prompt sorted for training: bandwidth
        dict(name="dispatch_prompt_bf16", op="dispatch", tokens=16384, top_k=2, experts=64, h=4096, dtype="bf16",
             align=128, drop=0.0),
        # the experts' rows back to their tokens, onto the residual stream
        dict(name="combine_prompt_f16", op="combine", tokens=8192, top_k=8, experts=64, h=2048, dtype="f16", align=64,
             drop=0.0, weighted=True, residual=True),
        # the combine's gradient in f32, odd sizes, some assignments dropped (over capacity or padding tokens)
        dict(name="combine_grad_odd_f32", op="combine_grad", tokens=4099, top_k=4, experts=24, h=1002, dtype="f32",
             align=64, drop=0.1),
        # decoding sequences through few-token experts: bound by the used experts' weights
        dict(name="expert_decode_bf16", op="expert", tokens=16, top_k=4, experts=32, k=2048, n=1024, dtype="bf16",
             align=16, act="silu", bias=False, pre=False, wt=True, drop=0.0),
        # a prompt's tokens through the experts' up projection
        dict(name="expert_prompt_bf16", op="expert", tokens=8192, top_k=2, experts=16, k=2048, n=4096, dtype="bf16",
             align=128, act="gelu_tanh", bias=True, pre=False, wt=False, drop=0.0),
        # its gradient in a training step
        dict(name="expert_grad_bf16", op="expert_grad", tokens=4096, top_k=2, experts=8, k=2048, n=2048, dtype="bf16",
             align=128, act="silu", bias=True, wt=True, drop=0.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("linear", "linear", "linear_grad", "dispatch", "combine", "combine_grad", "expert", "expert_grad"))
    dtype = rng.choice(("bf16", "f16"))
    if op in ("linear", "linear_grad"):
        if op == "linear" and rng.random() < 0.2:
            dtype = "f32"
        most = LINEAR_WORK // (2 if op == "linear_grad" else 1) // (4 if dtype == "f32" else 1)
        while True:
            m, n, k = _log(rng, 1, 8192), _log(rng, 16, 11008), _log(rng, 16, 11008)
            if rng.random() < 0.5:
                n, k = (n + 7) // 8 * 8, (k + 7) // 8 * 8
            if m * n * k <= most:
                break
        case = dict(op=op, m=m, n=n, k=k, dtype=dtype, act=rng.choice(ACTS), bias=rng.random() < 0.7,
                    wt=rng.random() < 0.5)
        if op == "linear":
            case.update(residual=rng.random() < 0.5, pre=rng.random() < 0.3 and dtype != "f32")
        return case
    experts = _log(rng, 2, 128)
    top_k = min(experts, rng.choice((1, 2, 4, 6, 8)))
    drop = rng.choice((0.0, 0.0, 0.05, 0.5))
    if op in ("dispatch", "combine", "combine_grad"):
        if rng.random() < 0.3:
            dtype = "f32"
        while True:
            tokens, h = _log(rng, 1, 32768), _log(rng, 64, 8192)
            if rng.random() < 0.7:
                h = (h + 7) // 8 * 8
            if tokens * top_k * h <= 16384 * 8 * 1024:
                break
        case = dict(op=op, tokens=tokens, top_k=top_k, experts=experts, h=h, dtype=dtype,
                    align=rng.choice((1, 16, 64, 128)), drop=drop)
        if op == "combine":
            case.update(weighted=rng.random() < 0.8, residual=rng.random() < 0.5)
        return case
    while True:
        tokens, k, n = _log(rng, 1, 16384), _log(rng, 64, 4096), _log(rng, 64, 4096)
        if rng.random() < 0.7:
            n, k = (n + 7) // 8 * 8, (k + 7) // 8 * 8
        if tokens * top_k * n * k <= LINEAR_WORK // 4 and experts * n * k <= 1 << 28:
            break
    case = dict(op=op, tokens=tokens, top_k=top_k, experts=experts, k=k, n=n, dtype=dtype, act=rng.choice(ACTS),
                bias=rng.random() < 0.5, wt=rng.random() < 0.5, drop=drop)
    if op == "expert":
        case.update(align=rng.choice((1, 16, 64, 128)), pre=rng.random() < 0.3)
    else:
        case.update(align=rng.choice((64, 128)))
    return case


def _capacity(tokens, top_k, experts, align):
    """Rows that hold every assignment of any routing: each used expert pads its segment by at most align - 1."""
    n = tokens * top_k
    return (n + min(experts, n) * (align - 1)) // align * align


# ------------------------------------------------------------------ inputs --
def _inputs(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, dt=dtype):
        t = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
        return t.mul_(scale).to(dt)

    op = case["op"]
    if op in ("linear", "linear_grad"):
        m, n, k = case["m"], case["n"], case["k"]
        s = {"lhs": normal(m, k), "rhs": normal(n, k, scale=k ** -0.5) if case["wt"] else normal(k, n, scale=k ** -0.5)}
        if op == "linear":
            s["bias"] = normal(n, scale=0.5) if case["bias"] else None
            s["residual"] = normal(m, n) if case["residual"] else None
        else:
            s["d_out"] = normal(m, n, scale=0.1)
            s["pre"] = normal(m, n) if case["act"] != "none" else None
        return s
    tokens, top_k, experts = case["tokens"], case["top_k"], case["experts"]
    # a router's choices: the best of noisy scores with some experts preferred, so loads are uneven
    scores = torch.randn(tokens, experts, generator=g, device="cuda")
    scores += torch.randn(experts, generator=g, device="cuda")
    best, ids = scores.topk(top_k, dim=1)
    weights = torch.softmax(best, dim=1)
    ids = ids.to(torch.int32)
    if case["drop"]:
        ids[torch.rand(tokens, top_k, generator=g, device="cuda") < case["drop"]] = -1
    rows = _capacity(tokens, top_k, experts, case["align"])
    if op == "dispatch":
        return {"ids": ids, "x": normal(tokens, case["h"])}
    layout = dict(zip(("slots", "sources", "offsets", "counts"), _plain_layout(ids, experts, case["align"], rows)))
    held = (layout["sources"] >= 0).unsqueeze(1)

    def sorted_rows(width, scale=1.0):
        return normal(rows, width, scale=scale).mul_(held)

    if op == "combine":
        return dict(layout, rows=sorted_rows(case["h"]), weights=weights if case["weighted"] else None,
                    residual=normal(tokens, case["h"]) if case["residual"] else None)
    if op == "combine_grad":
        return dict(layout, rows=sorted_rows(case["h"]), weights=weights, d_out=normal(tokens, case["h"], scale=0.1))
    k, n = case["k"], case["n"]
    s = dict(layout, rows=sorted_rows(k),
             weights=normal(experts, n, k, scale=k ** -0.5) if case["wt"] else normal(experts, k, n, scale=k ** -0.5))
    if op == "expert":
        s["bias"] = normal(experts, n, scale=0.5) if case["bias"] else None
    else:
        s["d_out"] = sorted_rows(n, 0.1)
        s["pre"] = sorted_rows(n) if case["act"] != "none" else None
    return s


def prepare(case, seed):
    state = {"case": case, "inputs": _inputs(case, seed)}
    if own:
        state["op"], state["outputs"] = _bind(case, state["inputs"])
    return state


def run(state):
    if own:
        state["op"].replay(torch.cuda.current_stream().cuda_stream)
        return state["outputs"]
    return _PLAIN[state["case"]["op"]](state["case"], state["inputs"])


# ------------------------------------------------- through the framework --
def _bind(case, s):
    """The bound operator and its output tensors, as a user's program sets them up once."""
    import momiru_b200 as mb

    op, dtype = case["op"], DTYPES[case["dtype"]]
    view = lambda t: None if t is None else mb.DeviceView.from_torch(t)  # noqa: E731
    new = lambda *shape, dt=dtype: torch.empty(*shape, dtype=dt, device="cuda")  # noqa: E731
    act = lambda: mb.Activation[case["act"].upper()]  # noqa: E731
    if op == "linear":
        node = mb.LinearNode(transpose_rhs=case["wt"], activation=act())
        out = {"out": new(case["m"], case["n"])}
        if case["pre"]:
            out["pre"] = new(case["m"], case["n"])
        return mb.BoundLinear(node, view(s["lhs"]), view(s["rhs"]), view(out["out"]), bias=view(s["bias"]),
                              residual=view(s["residual"]), pre=view(out.get("pre"))), out
    if op == "linear_grad":
        node = mb.LinearNode(transpose_rhs=case["wt"], activation=act())
        out = {"d_lhs": torch.empty_like(s["lhs"]), "d_rhs": torch.empty_like(s["rhs"])}
        if case["bias"]:
            out["d_bias"] = new(case["n"])
        return mb.BoundLinearGrad(node, view(s["d_out"]), view(s["lhs"]), view(s["rhs"]), d_lhs=view(out["d_lhs"]),
                                  d_rhs=view(out["d_rhs"]), d_bias=view(out.get("d_bias")), pre=view(s["pre"])), out
    sizes = (case["tokens"], case["top_k"], case["experts"], case["align"])
    if op == "dispatch":
        layout = mb.ExpertLayout.empty(*sizes)
        out = {"rows": new(layout.rows, case["h"])}
        for name in ("slots", "sources", "offsets", "counts"):
            out[name] = getattr(layout, name).torch_view()
        return mb.BoundDispatch(layout, view(s["ids"]), view(s["x"]), view(out["rows"])), out
    layout = mb.ExpertLayout(*sizes, *(view(s[name]) for name in ("slots", "sources", "offsets", "counts")))
    if op == "combine":
        out = {"out": new(case["tokens"], case["h"])}
        return mb.BoundCombine(layout, view(s["rows"]), view(out["out"]), weights=view(s["weights"]),
                               residual=view(s["residual"])), out
    if op == "combine_grad":
        out = {"d_rows": torch.empty_like(s["rows"]), "d_weights": torch.empty_like(s["weights"])}
        return mb.BoundCombineGrad(layout, view(s["d_out"]), view(s["rows"]), view(s["weights"]),
                                   d_rows=view(out["d_rows"]), d_weights=view(out["d_weights"])), out
    node = mb.LinearNode(transpose_rhs=case["wt"], activation=act())
    if op == "expert":
        out = {"out": new(layout.rows, case["n"])}
        if case["pre"]:
            out["pre"] = new(layout.rows, case["n"])
        return mb.BoundExpertLinear(node, layout, view(s["rows"]), view(s["weights"]), view(out["out"]),
                                    bias=view(s["bias"]), pre=view(out.get("pre"))), out
    out = {"d_rows": torch.empty_like(s["rows"]), "d_weights": torch.empty_like(s["weights"])}
    if case["bias"]:
        out["d_bias"] = new(case["experts"], case["n"])
    return mb.BoundExpertLinearGrad(node, layout, view(s["d_out"]), view(s["rows"]), view(s["weights"]),
                                    d_rows=view(out["d_rows"]), d_weights=view(out["d_weights"]),
                                    d_bias=view(out.get("d_bias")), pre=view(s["pre"])), out


# -------------------------------------------------------------- plain form --
def _act(name, x):
    if name == "relu":
        return x.clamp(min=0)
    if name == "gelu_erf":
        return 0.5 * x * (1 + torch.erf(x * 0.5 ** 0.5))
    if name == "gelu_tanh":
        return 0.5 * x * (1 + torch.tanh((2 / math.pi) ** 0.5 * (x + 0.044715 * x * x * x)))
    if name == "silu":
        return x * torch.sigmoid(x)
    return x


def _act_grad(name, x):
    if name == "relu":
        return (x > 0).float()
    if name == "gelu_erf":
        return 0.5 * (1 + torch.erf(x * 0.5 ** 0.5)) + x * torch.exp(-0.5 * x * x) * (2 * math.pi) ** -0.5
    if name == "gelu_tanh":
        c = (2 / math.pi) ** 0.5
        t = torch.tanh(c * (x + 0.044715 * x * x * x))
        return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * c * (1 + 0.134145 * x * x)
    s = torch.sigmoid(x)
    return s * (1 + x * (1 - s))


def _plain_linear(case, s):
    dtype = DTYPES[case["dtype"]]
    rhs = s["rhs"].float()
    pre = s["lhs"].float() @ (rhs.t() if case["wt"] else rhs)
    if s["bias"] is not None:
        pre = pre + s["bias"].float()
    y = _act(case["act"], pre)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"out": y.to(dtype)}
    if case["pre"]:
        out["pre"] = pre.to(dtype)
    return out


def _plain_linear_grad(case, s):
    dtype = DTYPES[case["dtype"]]
    dp = s["d_out"].float()
    if s["pre"] is not None:
        dp = dp * _act_grad(case["act"], s["pre"].float())
    lhs, rhs = s["lhs"].float(), s["rhs"].float()
    out = {"d_lhs": (dp @ (rhs if case["wt"] else rhs.t())).to(dtype),
           "d_rhs": (dp.t() @ lhs if case["wt"] else lhs.t() @ dp).to(dtype)}
    if case["bias"]:
        out["d_bias"] = dp.sum(0).to(dtype)
    return out


def _plain_layout(ids, experts, align, rows):
    flat = ids.reshape(-1).long()
    n = flat.numel()
    index = torch.arange(n, device=flat.device)
    key = torch.where((flat >= 0) & (flat < experts), flat, experts)  # dropped assignments sort last
    order = torch.argsort(key, stable=True)
    counts = torch.zeros(experts + 1, dtype=torch.long, device=flat.device).scatter_add_(0, key, torch.ones_like(key))
    firsts = counts.cumsum(0) - counts  # of each expert's assignments in the sorted order
    padded = (counts[:experts] + align - 1) // align * align
    offsets = torch.cat((padded.new_zeros(1), padded.cumsum(0)))
    ranked = key[order]
    slot = torch.where(ranked < experts, offsets[ranked] + index - firsts[ranked], -1)
    slots = torch.empty_like(slot).scatter_(0, order, slot)
    sources = torch.full((rows + 1,), -1, dtype=torch.long, device=flat.device)
    sources.scatter_(0, torch.where(slots < 0, rows, slots), index)
    sources[rows] = -1
    to = torch.int32
    return slots.view(ids.shape).to(to), sources[:rows].to(to), offsets.to(to), counts[:experts].to(to)


def _plain_dispatch(case, s):
    rows = _capacity(case["tokens"], case["top_k"], case["experts"], case["align"])
    slots, sources, offsets, counts = _plain_layout(s["ids"], case["experts"], case["align"], rows)
    taken = s["x"][sources.clamp(min=0).long() // case["top_k"]]
    return {"rows": torch.where((sources >= 0).unsqueeze(1), taken, torch.zeros_like(taken)), "slots": slots,
            "sources": sources, "offsets": offsets, "counts": counts}


def _plain_combine(case, s):
    held = s["slots"] >= 0
    taken = s["rows"].float()[s["slots"].clamp(min=0).long()]
    if s["weights"] is not None:
        taken = taken * s["weights"].unsqueeze(2)
    y = torch.where(held.unsqueeze(2), taken, 0.0).sum(1)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"out": y.to(DTYPES[case["dtype"]])}


def _plain_combine_grad(case, s):
    d_out, k = s["d_out"].float(), case["top_k"]
    source = s["sources"].clamp(min=0).long()
    d_rows = d_out[source // k] * s["weights"].reshape(-1)[source].unsqueeze(1)
    d_rows = torch.where((s["sources"] >= 0).unsqueeze(1), d_rows, 0.0)
    taken = s["rows"].float()[s["slots"].clamp(min=0).long()]
    d_weights = torch.where(s["slots"] >= 0, (taken * d_out.unsqueeze(1)).sum(2), 0.0)
    return {"d_rows": d_rows.to(DTYPES[case["dtype"]]), "d_weights": d_weights}


def _segments(s):
    """(expert, first row, end of its tokens) of the experts that have any: read back, as an eager program does."""
    return [(e, o, o + c) for e, (o, c) in enumerate(zip(s["offsets"].tolist(), s["counts"].tolist())) if c]


def _plain_expert(case, s):
    dtype = DTYPES[case["dtype"]]
    rows, n = s["rows"].shape[0], case["n"]
    out = {"out": torch.zeros(rows, n, dtype=dtype, device="cuda")}
    if case["pre"]:
        out["pre"] = torch.zeros(rows, n, dtype=dtype, device="cuda")
    for e, r0, r1 in _segments(s):  # the experts' products have no single elementary form: one per used expert
        w = s["weights"][e].float()
        pre = s["rows"][r0:r1].float() @ (w.t() if case["wt"] else w)
        if s["bias"] is not None:
            pre = pre + s["bias"][e].float()
        out["out"][r0:r1] = _act(case["act"], pre).to(dtype)
        if case["pre"]:
            out["pre"][r0:r1] = pre.to(dtype)
    return out


def _plain_expert_grad(case, s):
    dtype = DTYPES[case["dtype"]]
    out = {"d_rows": torch.zeros_like(s["rows"]), "d_weights": torch.zeros_like(s["weights"])}
    if case["bias"]:
        out["d_bias"] = torch.zeros(case["experts"], case["n"], dtype=dtype, device="cuda")
    for e, r0, r1 in _segments(s):
        dp = s["d_out"][r0:r1].float()
        if s["pre"] is not None:
            dp = dp * _act_grad(case["act"], s["pre"][r0:r1].float())
        w, x = s["weights"][e].float(), s["rows"][r0:r1].float()
        out["d_rows"][r0:r1] = (dp @ (w if case["wt"] else w.t())).to(dtype)
        out["d_weights"][e] = (dp.t() @ x if case["wt"] else x.t() @ dp).to(dtype)
        if case["bias"]:
            out["d_bias"][e] = dp.sum(0).to(dtype)
    return out


_PLAIN = {"linear": _plain_linear, "linear_grad": _plain_linear_grad, "dispatch": _plain_dispatch,
          "combine": _plain_combine, "combine_grad": _plain_combine_grad, "expert": _plain_expert,
          "expert_grad": _plain_expert_grad}


# -------------------------------------------------------------------- exact --
def _act64(name, x):
    """The activation and its derivative at x, in 64 bits."""
    if name == "none":
        return x, torch.ones_like(x)
    if name == "relu":
        on = (x > 0).double()
        return torch.where(on > 0, x, torch.zeros_like(x)), on
    if name == "silu":
        p = 1 / (1 + torch.exp(-x))
        return x * p, p + x * p * (1 - p)
    if name == "gelu_erf":
        cdf = 0.5 * torch.special.erfc(-x / math.sqrt(2.0))
        return x * cdf, cdf + x * torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    u = math.sqrt(2 / math.pi) * (x + 0.044715 * x ** 3)
    p = 1 / (1 + torch.exp(-2 * u))  # (1 + tanh u) / 2
    return x * p, p + x * 2 * p * (1 - p) * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * x ** 2)


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    wide = lambda t: None if t is None else t.double()  # noqa: E731
    if op == "linear":
        w = wide(s["rhs"])
        pre = torch.einsum("mk,nk->mn" if case["wt"] else "mk,kn->mn", wide(s["lhs"]), w)
        if case["bias"]:
            pre += wide(s["bias"])[None, :]
        y = _act64(case["act"], pre)[0]
        if case["residual"]:
            y = y + wide(s["residual"])
        return {"out": y, "pre": pre} if case["pre"] else {"out": y}
    if op == "linear_grad":
        dp = wide(s["d_out"])
        if s["pre"] is not None:
            dp = dp * _act64(case["act"], wide(s["pre"]))[1]
        w, x = wide(s["rhs"]), wide(s["lhs"])
        out = {"d_lhs": torch.einsum("mn,nk->mk" if case["wt"] else "mn,kn->mk", dp, w),
               "d_rhs": torch.einsum("mn,mk->nk" if case["wt"] else "mn,mk->kn", dp, x)}
        if case["bias"]:
            out["d_bias"] = torch.einsum("mn->n", dp)
        return out
    tokens, k = case["tokens"], case["top_k"]
    if op == "dispatch":
        ids = s["ids"].flatten().tolist()
        lists = [[] for _ in range(case["experts"])]
        for i, e in enumerate(ids):
            if 0 <= e < case["experts"]:
                lists[e].append(i)
        rows = torch.zeros(_capacity(tokens, k, case["experts"], case["align"]), case["h"], dtype=torch.float64,
                           device="cuda")
        at = 0
        for members in lists:
            if members:
                rows[at:at + len(members)] = s["x"][torch.tensor(members, device="cuda") // k].double()
            at += -(-len(members) // case["align"]) * case["align"]
        return {"rows": rows, "slots": None, "sources": None, "offsets": None, "counts": None}
    if op == "combine":
        y = torch.zeros(tokens, case["h"], dtype=torch.float64, device="cuda")
        if case["residual"]:
            y += s["residual"]
        for j in range(k):
            here = (s["slots"][:, j] >= 0).nonzero().flatten()
            w = s["weights"][here, j].double()[:, None] if case["weighted"] else 1.0
            y[here] += w * s["rows"][s["slots"][here, j].long()].double()
        return {"out": y}
    if op == "combine_grad":
        d_rows = torch.zeros(s["rows"].shape, dtype=torch.float64, device="cuda")
        d_weights = torch.zeros(tokens, k, dtype=torch.float64, device="cuda")
        for j in range(k):
            here = (s["slots"][:, j] >= 0).nonzero().flatten()
            at = s["slots"][here, j].long()
            d = s["d_out"][here].double()
            d_rows[at] = d * s["weights"][here, j].double()[:, None]
            d_weights[here, j] = torch.einsum("th,th->t", d, s["rows"][at].double())
        return {"d_rows": d_rows, "d_weights": d_weights}
    starts, counts = s["offsets"].tolist(), s["counts"].tolist()
    rows, n = s["rows"].shape[0], case["n"]
    if op == "expert":
        y = torch.zeros(rows, n, dtype=torch.float64, device="cuda")
        p = torch.zeros_like(y)
        for e in range(case["experts"]):
            part = slice(starts[e], starts[e] + counts[e])
            pre = torch.einsum("mk,nk->mn" if case["wt"] else "mk,kn->mn", s["rows"][part].double(),
                               s["weights"][e].double())
            if case["bias"]:
                pre += s["bias"][e].double()[None, :]
            p[part], y[part] = pre, _act64(case["act"], pre)[0]
        return {"out": y, "pre": p} if case["pre"] else {"out": y}
    out = {"d_rows": torch.zeros(s["rows"].shape, dtype=torch.float64, device="cuda"),
           "d_weights": torch.zeros(s["weights"].shape, dtype=torch.float64, device="cuda")}
    if case["bias"]:
        out["d_bias"] = torch.zeros(case["experts"], n, dtype=torch.float64, device="cuda")
    for e in range(case["experts"]):
        part = slice(starts[e], starts[e] + counts[e])
        dp = s["d_out"][part].double()
        if s["pre"] is not None:
            dp = dp * _act64(case["act"], s["pre"][part].double())[1]
        w, x = s["weights"][e].double(), s["rows"][part].double()
        out["d_rows"][part] = torch.einsum("mn,nk->mk" if case["wt"] else "mn,kn->mk", dp, w)
        out["d_weights"][e] = torch.einsum("mn,mk->nk" if case["wt"] else "mn,mk->kn", dp, x)
        if case["bias"]:
            out["d_bias"][e] = torch.einsum("mn->n", dp)
    return out


# --------------------------------------------------------------------- work --
def _used(n, experts):
    """Experts that n assignments reach, expected under an even choice."""
    return experts * (1 - (1 - 1 / experts) ** n)


def work(case):
    op, es = case["op"], BYTES[case["dtype"]]
    if op == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        outs = 1 + case["pre"] + case["residual"]
        return {"bytes": es * (m * k + k * n + n * case["bias"] + m * n * outs), "flops": 2 * m * n * k}
    if op == "linear_grad":
        m, n, k = case["m"], case["n"], case["k"]
        seen = 1 + (case["act"] != "none")
        return {"bytes": es * (m * n * seen + 2 * m * k + 2 * k * n + n * case["bias"]), "flops": 4 * m * n * k}
    t, k = case["tokens"], case["top_k"]
    held = t * k * (1 - case["drop"])
    rows = _capacity(t, k, case["experts"], case["align"])
    if op == "dispatch":
        return {"bytes": es * case["h"] * (t + rows) + 4 * (2 * t * k + rows + 2 * case["experts"] + 1), "flops": 0}
    if op == "combine":
        return {"bytes": es * case["h"] * (held + t * (1 + case["residual"])) + 4 * t * k * (1 + case["weighted"]),
                "flops": 2 * held * case["h"]}
    if op == "combine_grad":
        return {"bytes": es * case["h"] * (t + held + rows) + 12 * t * k, "flops": 3 * held * case["h"]}
    kk, n, used = case["k"], case["n"], _used(held, case["experts"])
    if op == "expert":
        return {"bytes": es * (held * kk + used * kk * n + rows * n * (1 + case["pre"])), "flops": 2 * held * n * kk}
    seen = 1 + (case["act"] != "none")
    return {"bytes": es * (held * (n * seen + kk) + rows * kk + (used + case["experts"]) * kk * n),
            "flops": 4 * held * n * kk}
