"""A mixture-of-experts feed-forward block, trained for a few steps.

Every product, sort and sum runs through the framework's bound operators:

    h   = x + x @ w_in                                     BoundLinear with a residual
    r   = h sorted by expert                               BoundDispatch
    a   = silu(r @ up[e] + b[e])                           BoundExpertLinear, pre kept
    o   = a @ down[e]                                      BoundExpertLinear
    y   = h + sum_j weights[t, j] o[slots[t, j]]           BoundCombine with a residual

and back. Everything is bound once; a step only replays. torch holds the memory,
makes the data and applies the gradients. The router (here: fixed scores of each
token) is outside the block: its choices are inputs, as ids and weights.

    python examples/expert_ffn.py [--steps 20]
"""
from __future__ import annotations

import argparse
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import torch  # noqa: E402

import momiru_b200 as mb  # noqa: E402

V = mb.DeviceView.from_torch


class ExpertFfn:
    """The block's parameters, buffers and bound operators for one batch shape."""

    def __init__(self, tokens: int, hidden: int, inner: int, experts: int, top_k: int, dtype=torch.bfloat16,
                 row_align: int = 64, seed: int = 0):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        new = lambda *s: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731

        def weight(*s):
            return (torch.randn(*s, generator=g, device="cuda") * s[-2] ** -0.5).to(dtype)

        self.p = {"w_in": weight(hidden, hidden), "up": weight(experts, hidden, inner),
                  "b": torch.zeros(experts, inner, dtype=dtype, device="cuda"), "down": weight(experts, inner, hidden)}
        self.g = {k: torch.empty_like(v) for k, v in self.p.items()}
        lay = self.layout = mb.ExpertLayout.empty(tokens, top_k, experts, row_align)
        self.x, self.h, self.y = new(tokens, hidden), new(tokens, hidden), new(tokens, hidden)
        self.ids = torch.zeros(tokens, top_k, dtype=torch.int32, device="cuda")
        self.weights = torch.zeros(tokens, top_k, device="cuda")
        rows, pre, act, out = new(lay.rows, hidden), new(lay.rows, inner), new(lay.rows, inner), new(lay.rows, hidden)
        self.d_y, self.d_h, self.d_weights = new(tokens, hidden), new(tokens, hidden), torch.empty_like(self.weights)
        d_out, d_act, d_rows = new(lay.rows, hidden), new(lay.rows, inner), new(lay.rows, hidden)
        plain, silu = mb.LinearNode(), mb.LinearNode(activation=mb.Activation.SILU)
        p, d = {k: V(v) for k, v in self.p.items()}, {k: V(v) for k, v in self.g.items()}
        self.forward_ops = [
            mb.BoundLinear(plain, V(self.x), p["w_in"], V(self.h), residual=V(self.x)),
            mb.BoundDispatch(lay, V(self.ids), V(self.h), V(rows)),
            mb.BoundExpertLinear(silu, lay, V(rows), p["up"], V(act), bias=p["b"], pre=V(pre)),
            mb.BoundExpertLinear(plain, lay, V(act), p["down"], V(out)),
            mb.BoundCombine(lay, V(out), V(self.y), weights=V(self.weights), residual=V(self.h)),
        ]
        self.backward_ops = [
            mb.BoundCombineGrad(lay, V(self.d_y), V(out), V(self.weights), d_rows=V(d_out), d_weights=V(self.d_weights)),
            mb.BoundExpertLinearGrad(plain, lay, V(d_out), V(act), p["down"], d_rows=V(d_act), d_weights=d["down"]),
            mb.BoundExpertLinearGrad(silu, lay, V(d_act), V(rows), p["up"], d_rows=V(d_rows), d_weights=d["up"],
                                     d_bias=d["b"], pre=V(pre)),
            # the dispatch's gradient, and the residual's: d_h = d_y + sum of the rows' gradients
            mb.BoundCombine(lay, V(d_rows), V(self.d_h), residual=V(self.d_y)),
            mb.BoundLinearGrad(plain, V(self.d_h), V(self.x), p["w_in"], d_rhs=d["w_in"]),
        ]

    def forward(self) -> torch.Tensor:
        for op in self.forward_ops:
            op.replay(torch.cuda.current_stream().cuda_stream)
        return self.y

    def backward(self) -> dict:
        for op in self.backward_ops:
            op.replay(torch.cuda.current_stream().cuda_stream)
        return self.g

    def check(self) -> None:
        """Waits for every operator and raises what a kernel reported."""
        for op in self.forward_ops + self.backward_ops:
            op.quiesce_or_abort(30)

    def close(self) -> None:
        for op in self.forward_ops + self.backward_ops:
            op.close()


def route(ffn: ExpertFfn, seed: int) -> None:
    """Choices of a router with uneven preferences; one token in fifty is dropped."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    tokens, top_k = ffn.ids.shape
    scores = torch.randn(tokens, ffn.layout.experts, generator=g, device="cuda")
    scores += torch.randn(ffn.layout.experts, generator=g, device="cuda")
    best, ids = scores.topk(top_k, dim=1)
    ffn.weights.copy_(torch.softmax(best, dim=1))
    ids[torch.rand(tokens, generator=g, device="cuda") < 0.02] = -1
    ffn.ids.copy_(ids.int())


def train(steps: int = 20, tokens: int = 512, hidden: int = 256, inner: int = 512, experts: int = 8, top_k: int = 2,
          rate: float = 4.0, dtype=torch.bfloat16) -> list:
    """Plain gradient descent towards the block's own output under other weights; returns the losses."""
    teacher = ExpertFfn(tokens, hidden, inner, experts, top_k, dtype, seed=1)
    ffn = ExpertFfn(tokens, hidden, inner, experts, top_k, dtype, seed=2)
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    x = torch.randn(tokens, hidden, generator=g, device="cuda").to(dtype)
    losses = []
    for f in (teacher, ffn):
        f.x.copy_(x)
        route(f, 4)
    want = teacher.forward().float()
    for _ in range(steps):
        error = ffn.forward().float() - want
        losses.append(float(error.square().mean()))
        ffn.d_y.copy_(error * (2 / error.numel()))  # of the mean square
        for name, grad in ffn.backward().items():
            ffn.p[name].sub_(rate * grad)
    for f in (teacher, ffn):
        f.check()
        f.close()
    return losses


if __name__ == "__main__":
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=20)
    for i, loss in enumerate(train(ap.parse_args().steps)):
        print(f"step {i:3d}  loss {loss:.5f}")
