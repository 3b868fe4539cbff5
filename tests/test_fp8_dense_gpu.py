"""A dense feed-forward with matrices in 8-bit floating point: what lies between its products is rounded once, from floats."""
import types

import pytest
import torch

from brolm_b200 import kernels
from brolm_b200.parts.feedforward import DenseFeedForward
from tests.plain import fp8_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def sum_bound(x, w):
    """For every result how far a float sum on the tensor core may be off: nine errors of 2^-23 of the terms' magnitudes a block of 128
    (eight of the additions, one for a piece), and one more."""
    return (9 * ((x.shape[1] + 127) // 128) + 2) * 2.0 ** -23 * (x.abs() @ w.abs().T)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [1, 8, 100, 300])
@pytest.mark.parametrize("activation, bias", [("relu2", False), ("none", False), ("gelu_tanh", False), ("relu2", True), ("silu", True)])
def test_the_middle_is_rounded_once(activation, bias, m, dtype):
    """The same bits as the first product's floats, bias and activation in float, their rounding to 8 bits, the second product; and
    within what float sums allow of 64 bits: a sum of the first product is off by `zb` (and a rounding with the bias), the activation's
    slope is 1.13 at most (2 |z| for the square of relu) and it is off by 4e-6 of itself (and, of numbers far below its argument, of
    that); a number whose rounding moves within that is a step away, 2^-3 of it or 2^-8 of its block's largest over 224."""
    hidden, inter = 256, 640
    g = torch.Generator(device=DEV).manual_seed(m)
    part = DenseFeedForward(hidden, inter, activation, bias)
    params = {n: torch.randn(tuple(s.shape), generator=g, device=DEV).to(dtype) * 0.06 for n, s in part.param_specs().items()}
    part.bind(params)
    part.to_fp8()
    x = torch.randn(m, hidden, generator=g, device=DEV).to(dtype)
    got = part.forward(x, types.SimpleNamespace(dtype=dtype))
    up, act, want = torch.empty(m, inter, device=DEV), torch.empty(m, inter, device=DEV), torch.empty(m, hidden, device=DEV)
    kernels.linear_fp8(x, part.w_up, up)
    kernels.bias_act(up, part.b_up, activation, act)
    kernels.linear_fp8(act, part.w_down, want)
    if bias:
        whole = torch.empty_like(want)
        kernels.bias_act(want, part.b_down, "none", whole)
        want = whole
    assert got.dtype == torch.float32 and torch.equal(got, want)
    xe, ue, de = plain.values(x), part.w_up.float().double(), part.w_down.float().double()
    z, zb = xe @ ue.T, sum_bound(xe, ue)
    if bias:
        z = z + part.b_up.double()
        zb = zb + 2.0 ** -24 * (z.abs() + zb)
    h = plain.act(z, activation)
    off = 2 * z.abs() * zb + zb ** 2 + 2.0 ** -23 * z ** 2 if activation == "relu2" else 1.13 * zb + 4e-6 * (h.abs() + z.abs())
    h8 = plain.values(h)
    tight = (plain.values(h + off) != h8) | (plain.values(h - off) != h8)
    step = 2.0 ** -3 * h.abs() + 2.0 ** -8 * h.abs().amax(dim=1, keepdim=True) / 224.0
    exact, bound = h8 @ de.T, sum_bound(h8, de) + (tight * step) @ de.abs().T
    if bias:
        exact = exact + part.b_down.double()
        bound = bound + 2.0 ** -24 * (exact.abs() + bound)
    assert bool(((got.double() - exact).abs() <= bound).all())
