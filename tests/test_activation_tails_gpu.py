"""The smooth activations of 16-bit layers where they run out towards zero: their
relative error, not only the absolute one, is that of one rounding.

Values: a contraction of one term makes `pre` the given 16-bit number exactly.
Bound: the type's unit roundoff u, and of the evaluation 2^-17 (approximations
of the exponential, the reciprocal and erfc) and 2^-22 for every unit of the
exponent A of the e^-A in the formula (its argument is rounded up to four times
in f32); half of f16's subnormal step."""
import math

import pytest
import torch

import momiru_b200 as mb
from test_linear_gpu import ACT, TYPES, V, check, replay

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda_lib")]
STEP = {"bf16": 2.0 ** -134, "f16": 2.0 ** -25}


def parts(act, x):
    """The activation, its derivative, the derivative's terms by magnitude, and the exponent, in 64 bits."""
    if act == ACT.GELU_ERF:
        cdf = 0.5 * torch.special.erfc(-x * 0.5 ** 0.5)
        slope = x * torch.exp(-0.5 * x * x) * (2 * math.pi) ** -0.5
        return x * cdf, cdf + slope, cdf + slope.abs(), 0.5 * x * x
    if act == ACT.SILU:
        u, du = x, torch.ones_like(x)
    else:
        c = 2 * (2 / math.pi) ** 0.5
        u, du = c * (x + 0.044715 * x ** 3), c * (1 + 3 * 0.044715 * x * x)
    s, t = torch.sigmoid(u), torch.sigmoid(-u)
    slope = x * s * t * du
    return x * s, s + slope, s + slope.abs(), u.abs()


def inputs(t):
    return torch.linspace(-10, 10, 4096, device="cuda").to(t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", [ACT.GELU_ERF, ACT.GELU_TANH, ACT.SILU])
@pytest.mark.parametrize("rows", [1, 1100])  # the strip kernel and the pair kernel
def test_values(dtype, act, rows):
    t, u = TYPES[dtype]
    x = inputs(t)
    one = torch.ones(rows, 1, dtype=t, device="cuda")
    out = torch.full((rows, x.numel()), float("nan"), dtype=t, device="cuda")
    replay(mb.BoundLinear(mb.LinearNode(activation=act), V(one), V(x[None]), V(out)))
    want, _, _, a = parts(act, x.double())
    check(out, want, (u + 2.0 ** -17 + 2.0 ** -22 * a) * want.abs() + STEP[dtype], "out")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", [ACT.GELU_ERF, ACT.GELU_TANH, ACT.SILU])
def test_derivatives(dtype, act):
    """One row and d_out of ones: the bias gradient is the derivative, rounded once."""
    t, u = TYPES[dtype]
    x = inputs(t)[None]
    n = x.shape[1]
    d_bias = torch.full((n,), float("nan"), dtype=t, device="cuda")
    e = lambda *s: torch.ones(*s, dtype=t, device="cuda")  # noqa: E731
    replay(mb.BoundLinearGrad(mb.LinearNode(activation=act), V(torch.ones_like(x)), V(e(1, 8)), V(e(8, n)), d_bias=V(d_bias),
                              pre=V(x)))
    _, want, size, a = parts(act, x[0].double())
    check(d_bias, want, u * want.abs() + (2.0 ** -17 + 2.0 ** -22 * a) * size + STEP[dtype], "d_bias")
