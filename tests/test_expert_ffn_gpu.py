"""The expert feed-forward example: its gradients against autograd of the same
block in 64 bits, and its loss going down."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda_lib")]


def block64(ffn):
    """The block from its definition, differentiable in 64 bits."""
    p = {k: v.double().requires_grad_() for k, v in ffn.p.items()}
    w = ffn.weights.double().requires_grad_()
    x = ffn.x.double()
    h = x + x @ p["w_in"]
    y = h
    for j in range(ffn.ids.shape[1]):
        e = ffn.ids[:, j].long()
        kept = (e >= 0)[:, None]
        e = e.clamp(min=0)
        a = torch.einsum("th,thi->ti", h, p["up"][e]) + p["b"][e]
        o = torch.einsum("ti,tih->th", a * torch.sigmoid(a), p["down"][e])
        y = y + torch.where(kept, w[:, j:j + 1] * o, 0.0)
    return p, w, y


@pytest.mark.parametrize("dtype,u", [(torch.bfloat16, 2.0 ** -8), (torch.float16, 2.0 ** -11)])
def test_gradients_of_the_whole_block(dtype, u):
    """Each of the block's ten operators rounds its results once (h, rows are
    exact copies, a, o, y; d_out, d_act, d_pre, d_rows, d_h, the gradients):
    along any path at most eight roundings of relative size u, in norm."""
    import expert_ffn

    ffn = expert_ffn.ExpertFfn(96, 72, 136, 5, 2, dtype, seed=5)
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    ffn.x.copy_(torch.randn(96, 72, generator=g, device="cuda"))
    ffn.p["b"].copy_(torch.randn(5, 136, generator=g, device="cuda") * 0.3)
    ffn.d_y.copy_(torch.randn(96, 72, generator=g, device="cuda"))
    expert_ffn.route(ffn, 7)
    y, grads = ffn.forward(), ffn.backward()
    ffn.check()
    p, w, want = block64(ffn)
    want.backward(ffn.d_y.double())
    far = lambda a, b: float((a.double() - b).norm() / b.norm())  # noqa: E731
    assert far(y, want.detach()) <= 8 * u
    for name in grads:
        assert far(grads[name], p[name].grad) <= 8 * u, name
    assert far(ffn.d_weights, w.grad) <= 8 * u
    ffn.close()


def test_training_lowers_the_loss():
    import expert_ffn

    losses = expert_ffn.train(steps=12)
    assert all(b < a for a, b in zip(losses, losses[1:])), losses
