"""Products in 8-bit floating point against 64 bits, at the sizes and values where they can go wrong.

Tolerances.  Rounding to 8 bits is exact: the same numbers as the oracle's.  A float sum on the tensor core adds 32 products at a
time and cuts off: an addition of the accumulator and one among the products, each at most 2^-23 of the terms' magnitudes, eight
such errors a block of 128, and one rounding for each piece that is added.  A result in bfloat16 is off by 2^-8 of itself at most.
"""
import pytest
import torch

from brolm_b200 import kernels
from brolm_b200.kernels import fp8
from tests.plain import fp8_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def rows_of(g, m, k, dtype, spread=1.0):
    x = torch.randn(m, k, generator=g, device=DEV) * torch.exp(spread * torch.randn(k, generator=g, device=DEV))
    return x.to(dtype)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def read(m):
    y = torch.empty(m.shape, dtype=torch.float32, device=DEV)
    kernels.fp8_read(m, y)
    return y


def sum_bound(x, w):
    """For every result how far a float sum of it may be off."""
    blocks = (x.shape[1] + 127) // 128
    return (8 * blocks + 8 + 2) * 2.0 ** -23 * (x.abs() @ w.abs().T)


def near(y, exact, bound):
    y = y.double()
    if y.numel() == 0:
        return
    if y.dtype != torch.float64:
        raise AssertionError
    off = (y - exact).abs()
    assert bool((off <= bound).all()), f"off by {float((off - bound).max())} beyond the bound, at {torch.nonzero(off > bound)[:4].tolist()}"


def rounded(bound, exact, dtype):
    return bound + (2.0 ** -8 * (exact.abs() + bound) if dtype == torch.bfloat16 else 0.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m, k, pad", [(1, 1, 0), (1, 128, 0), (3, 127, 0), (7, 129, 0), (130, 511, 1), (257, 513, 7), (64, 1000, 600), (5, 2304, 0), (2, 4608, 8)])
def test_rows_to_8_bits_and_back(m, k, pad, dtype):
    g = gen(m * 1000 + k)
    wide = torch.randn(m, k + pad, generator=g, device=DEV) * torch.exp2(torch.randint(-30, 30, (m, k + pad), generator=g, device=DEV).float())
    x = wide.to(dtype)[:, :k]
    x[0, 0] = 448.0
    if k > 128:
        x[m - 1, 128:min(k, 256)] = 0.0
    m8 = kernels.fp8_quantize(x)
    want = plain.values(x)
    assert torch.equal(read(m8).double(), want)
    into = torch.full((m, k + 3), 7.0, dtype=dtype, device=DEV)
    kernels.fp8_read(m8, into[:, :k])
    assert torch.equal(into[:, :k], want.to(torch.float32).to(dtype)) and bool((into[:, k:] == 7.0).all())


def test_rows_at_the_ends_of_a_floats_range():
    x = torch.zeros(8, 256, device=DEV)
    x[0, :3] = torch.tensor([3.4e38, -3.4e38, 1e30])
    x[1, :3] = torch.tensor([1e-45, -1e-40, 2.0 ** -126])
    x[2, 0] = 448.0 * 2.0 ** -127
    x[3, 0] = 449.0 * 2.0 ** -127
    x[4, :2] = torch.tensor([448.0, 2.0 ** -10])              # half of the smallest number: to even, zero
    x[5, :2] = torch.tensor([448.0, 3 * 2.0 ** -10])
    x[6, 128:130] = torch.tensor([-0.0, 5.0])
    want = plain.values(x)
    # 3.4e38 lies nearest to 256 * 2^120 = 2^128, the first power of two that a float does not have: it is read as infinity
    assert float(want[0, 0]) == 2.0 ** 128
    assert torch.equal(read(kernels.fp8_quantize(x)), want.float())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_number_that_is_not_finite_makes_its_block_nan(bad):
    g = gen(4)
    x = rows_of(g, 5, 640, torch.bfloat16)
    w = rows_of(g, 200, 640, torch.bfloat16)
    x[3, 300] = bad
    back = read(kernels.fp8_quantize(x))
    assert torch.isnan(back[3, 256:384]).all() and torch.isfinite(back[3, :256]).all() and torch.isfinite(back[3, 384:]).all()
    for m in (5, 300):
        xs = x if m == 5 else torch.cat([x, rows_of(g, 295, 640, torch.bfloat16)])
        y = torch.empty(m, 200, dtype=torch.float32, device=DEV)
        kernels.linear_fp8(xs, kernels.fp8_quantize(w), y)
        bad_rows = torch.isnan(y).any(dim=1)
        assert bool(torch.isnan(y[3]).all()) and int(bad_rows.sum()) == 1
    w[7, 5] = bad
    kernels.linear_fp8(xs, kernels.fp8_quantize(w), y)
    assert bool(torch.isnan(y[:, 7]).all()) and not bool(torch.isnan(y[:3, :7]).any())


SIZES = [(1, 1, 1), (1, 300, 128), (2, 128, 130), (15, 129, 512), (16, 64, 513), (17, 777, 1000), (33, 2304, 2304), (64, 100, 640), (65, 4096, 384), (128, 640, 9216),
         (129, 256, 128), (129, 1, 7), (200, 300, 1000), (256, 257, 2048), (300, 4095, 513), (1000, 777, 1000), (2049, 512, 2176)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m, n, k", SIZES)
def test_linear(m, n, k, dtype):
    g = gen(m + n + k)
    x, w = rows_of(g, m, k, dtype), rows_of(g, n, k, dtype, 0.3)
    w *= torch.exp2(torch.randint(-20, 20, (n, 1), generator=g, device=DEV).float()).to(dtype)
    xe, we = plain.values(x), plain.values(w)
    exact = xe @ we.T
    out = torch.full((m, n + 5), 7.0, dtype=dtype, device=DEV)
    w8 = kernels.fp8_quantize(w)
    y = out[:, :n] if n % 8 else out[:, :n].contiguous()
    kernels.linear_fp8(x, w8, y)
    near(y, exact, rounded(sum_bound(xe, we), exact, dtype))
    assert bool((out[:, n:] == 7.0).all())
    again = torch.empty_like(y)
    kernels.linear_fp8(kernels.fp8_quantize(x), w8, again)
    assert torch.equal(again, y)
    kernels.linear_fp8(x, w8, y, "relu2")
    near(y, plain.act(exact, "relu2"), rounded(2 * exact.abs() * sum_bound(xe, we) + sum_bound(xe, we) ** 2 + 2.0 ** -23 * exact ** 2, exact ** 2, dtype))


def gated_bound(ge, ue, bg, bu, name, limit=0.0):
    """How far the gated pair may be off: the gate's slope is 1.13 at most, the approximations cost 4e-6 of the result."""
    out = plain.gated(ge, ue, name, limit)
    if name == "clamped_gate":
        g, u = ge.clamp(max=limit), ue.clamp(-limit, limit)
        return out, 1.2 * bg * (u + 1).abs() + (g.abs() + bg) * bu + 8e-6 * (out.abs() + bg) + 4e-6
    return out, 1.13 * bg * (ue.abs() + bu) + (plain.act(ge, name).abs() + 1.13 * bg) * bu + 4e-6 * out.abs()


@pytest.mark.parametrize("name", ["gelu_tanh", "silu", "clamped_gate"])
@pytest.mark.parametrize("m, n, k", [(1, 1, 100), (5, 100, 640), (16, 1024, 2304), (31, 333, 1000), (128, 65, 256), (130, 129, 640), (257, 1000, 1100)])
def test_gated(m, n, k, name):
    g = gen(m * 7 + n)
    x, gate, up = rows_of(g, m, k, torch.bfloat16, 0.2), rows_of(g, n, k, torch.bfloat16, 0.2) * k ** -0.5, rows_of(g, n, k, torch.bfloat16, 0.2) * k ** -0.5
    xe, ge, ue = plain.values(x), plain.values(gate), plain.values(up)
    exact, bound = gated_bound(xe @ ge.T, xe @ ue.T, sum_bound(xe, ge), sum_bound(xe, ue), name, 2.0)
    w8 = kernels.fp8_gate_up(gate, up)
    for dtype in (torch.float32, torch.bfloat16):
        y = torch.empty(m, n, dtype=dtype, device=DEV)
        kernels.linear_fp8(x, w8, y, name, 2.0)
        near(y, exact, rounded(bound, exact, dtype))


@pytest.mark.parametrize("name", ["gelu_tanh", "silu"])
@pytest.mark.parametrize("m, width, inter", [(1, 256, 640), (9, 300, 100), (100, 384, 513), (128, 128, 128), (129, 256, 1000), (300, 500, 2050)])
def test_feedforward(m, width, inter, name):
    g = gen(m + width)
    x = rows_of(g, m, width, torch.bfloat16, 0.5)
    gate, up, down = (rows_of(g, a, b, torch.bfloat16, 0.3) * b ** -0.5 for a, b in ((inter, width), (inter, width), (width, inter)))
    xe, ge, ue, de = (plain.values(t) for t in (x, gate, up, down))
    h, off = gated_bound(xe @ ge.T, xe @ ue.T, sum_bound(xe, ge), sum_bound(xe, ue), name)
    h8 = plain.values(h)
    exact = h8 @ de.T
    # where a float sum lands on the other side of a border the number is a step away: 2^-3 of it, or the smallest step of
    # its block, whose scale may be twice as large, too; such numbers are those within `off` of a border
    tight = (plain.values(h + off) != h8) | (plain.values(h - off) != h8)
    step = 2.0 ** -3 * h.abs() + 2.0 ** -8 * plain.scale_of(1.0) * h.abs().amax(dim=1, keepdim=True) / 224.0
    bound = sum_bound(h8, de) + (tight * step) @ de.abs().T
    for dtype in (torch.bfloat16, torch.float32):
        y = torch.empty(m, width, dtype=dtype, device=DEV)
        kernels.feedforward_fp8(x, kernels.fp8_gate_up(gate, up), kernels.fp8_quantize(down), y, name)
        near(y, exact, rounded(bound, exact, dtype))
        assert float((y.double() - exact).norm() / exact.norm()) < (4e-3 if dtype == torch.bfloat16 else 2e-3)


def test_no_rows_and_no_waits_that_ran_out():
    w = kernels.fp8_quantize(torch.randn(64, 256, device=DEV))
    y = torch.empty(0, 64, device=DEV)
    kernels.linear_fp8(torch.empty(0, 256, device=DEV), w, y)
    assert kernels.fp8_stream_status() == 0 and kernels.fp8_gemm_status() == 0


def routed(g, t, top, e, style):
    z = torch.randn(t, e, generator=g, device=DEV)
    if style == "skewed":
        z += 4.0 * torch.randn(e, generator=g, device=DEV)
    if style == "one":                                       # the same expert for all, several times a token
        return torch.full((t, top), e - 1, dtype=torch.int32, device=DEV)
    ids = torch.topk(z, top, dim=1).indices.to(torch.int32).contiguous()
    if style == "outside":
        ids[torch.rand(t, top, generator=g, device=DEV) < 0.4] = e + 2
        ids[t // 2] = -1
    return ids


@pytest.mark.parametrize("t, top, e, width, inter, act, style, scale_input", [
    (1, 1, 1, 128, 64, "silu", "even", False),
    (1, 2, 4, 100, 30, "gelu_tanh", "even", False),
    (8, 4, 32, 256, 128, "silu", "even", False),
    (9, 3, 8, 300, 130, "relu2", "skewed", True),
    (40, 2, 3, 640, 200, "clamped_gate", "skewed", False),
    (33, 4, 5, 256, 256, "none", "one", False),
    (70, 2, 2, 130, 513, "silu", "even", True),
    (150, 2, 2, 256, 384, "silu", "outside", False),
    (300, 2, 3, 500, 130, "relu2", "skewed", True),
    (333, 3, 2, 384, 640, "gelu_tanh", "one", False),
    (200, 6, 64, 128, 48, "silu", "skewed", False),
    (5, 2, 4, 128, 64, "silu", "outside", False)])
def test_experts(t, top, e, width, inter, act, style, scale_input):
    g = gen(t + e + width)
    ids = routed(g, t, top, e, style)
    weights = torch.rand(t, top, generator=g, device=DEV) + 0.1
    x = rows_of(g, t, width, torch.bfloat16, 0.5)
    plain_up = act in ("relu2", "none")
    up, down = (rows_of(g, e * a, b, torch.bfloat16, 0.3).view(e, a, b) * b ** -0.5 for a, b in ((inter, width), (width, inter)))
    gate = None if plain_up else rows_of(g, e * inter, width, torch.bfloat16, 0.3).view(e, inter, width) * width ** -0.5
    xe, ue, de = plain.values(x), plain.values(up), plain.values(down)
    ge = None if plain_up else plain.values(gate)
    # per pair: what it is, and how far it may be off (as for the feed-forward)
    exact, bound = torch.zeros(t, width, dtype=torch.float64, device=DEV), torch.zeros(t, width, dtype=torch.float64, device=DEV)
    for k in range(e):
        chose = ids == k
        tok, ch = chose.nonzero(as_tuple=True)
        if not len(tok):
            continue
        s = weights[tok, ch].double()[:, None]
        si = s if scale_input else 1.0
        z, zb = (xe[tok] @ ue[k].T) * si, sum_bound(xe[tok], ue[k]) * si
        if plain_up:
            h = plain.act(z, act)
            off = zb if act == "none" else 2 * z.abs() * zb + zb ** 2 + 2.0 ** -23 * z ** 2
        else:
            h, off = gated_bound((xe[tok] @ ge[k].T) * si, z, sum_bound(xe[tok], ge[k]) * si, zb, act, 2.0)
        h8 = plain.values(h)
        tight = (plain.values(h + off) != h8) | (plain.values(h - off) != h8)
        step = 2.0 ** -3 * h.abs() + 2.0 ** -8 * h.abs().amax(dim=1, keepdim=True) / 224.0
        so = 1.0 if scale_input else s
        y = (h8 @ de[k].T) * so
        exact.index_add_(0, tok, y)
        bound.index_add_(0, tok, (sum_bound(h8, de[k]) + (tight * step) @ de[k].abs().T) * so + 2.0 ** -22 * y.abs())
    up8 = kernels.fp8_quantize(up) if plain_up else kernels.fp8_gate_up(gate, up)
    d8 = kernels.fp8_quantize(down)
    for dtype in (torch.float32, torch.bfloat16):
        out = torch.full((t, width + 3), 7.0, dtype=dtype, device=DEV)
        kernels.experts_fp8(x, ids, weights, up8, d8, out[:, :width], act, 2.0, scale_input)
        near(out[:, :width], exact, rounded(bound, exact, dtype))
        assert bool((out[:, width:] == 7.0).all())
    pairs = torch.full((top, t, width), 7.0, dtype=torch.float32, device=DEV)
    kernels.experts_fp8_pairs(x, ids, up8, d8, pairs, act, 2.0, weights if scale_input else None)
    none = ((ids < 0) | (ids >= e)).T
    assert bool((pairs[none] == 7.0).all())
    assert kernels.fp8_stream_status() == 0 and kernels.fp8_gemm_status() == 0
