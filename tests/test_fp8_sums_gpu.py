"""Float results of long sums with matrices in 8-bit floating point: summed in pieces of 32 blocks of 128 along K, in tiles and in
streams.

Bounds.  An addition on the tensor core cuts off: 2^-23 at most, one of the accumulator and one among the products for every 32 along
K, eight a block, so 8 * 32 of the magnitudes of a piece's terms; then a rounding (2^-24) of the running sum for each piece, each
slice, and the result."""
import pytest
import torch

from brolm_b200 import kernels
from brolm_b200.kernels import fp8
from tests.plain import fp8_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
PIECE = 32


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rows_of(g, m, k, dtype, spread=1.0):
    return (torch.randn(m, k, generator=g, device=DEV) * torch.exp(spread * torch.randn(k, generator=g, device=DEV))).to(dtype)


def sum_bound(x, w):
    blocks = (x.shape[1] + 127) // 128
    pieces = (blocks + PIECE - 1) // PIECE + 8              # (eight slices at most, each of which may end inside a piece)
    return (8 * min(blocks, PIECE) + 0.5 * (2 * pieces + 2)) * 2.0 ** -23 * (x.abs() @ w.abs().T)


def near(y, exact, bound):
    off = (y.double() - exact).abs()
    assert bool((off <= bound).all()), f"off by {float((off - bound).max())} beyond the bound, at {torch.nonzero(off > bound)[:4].tolist()}"


# slices of 33 blocks and more (few tiles), one slice (149 tiles), every width of an accumulator; more than 128 rows are tiles
SIZES = [(1, 40, 33_000), (16, 300, 65_536), (17, 100, 40_000), (33, 130, 66_000), (64, 1, 50_000), (65, 257, 70_000), (100, 300, 36_000), (128, 129, 65_536),
         (3, 19_000, 4_300), (40, 19_000, 4_300), (100, 19_000, 4_300), (130, 300, 33_000)]


@pytest.mark.parametrize("m, n, k", SIZES)
def test_long_sums(m, n, k):
    g = gen(m + n + k)
    x, w = rows_of(g, m, k, torch.float32), rows_of(g, n, k, torch.bfloat16, 0.3)
    w8 = kernels.fp8_quantize(w)
    sms = kernels.device_sms(torch.device(DEV))
    blocks = (k + 127) // 128
    if fp8.fp8_streamed(m, n, blocks, sms):
        slices = fp8.fp8_slices((n + 127) // 128, blocks, sms)
        assert (blocks + slices - 1) // slices > PIECE      # what these sizes are for
    some = torch.unique(torch.cat([torch.arange(min(n, 200), device=DEV), torch.arange(max(0, n - 200), n, device=DEV)]))
    xe, we = plain.values(x), plain.values(w[some])
    exact, bound = xe @ we.T, sum_bound(xe, we)
    out = torch.full((m, n + 5), 7.0, device=DEV)
    y = out[:, :n]
    kernels.linear_fp8(x, w8, y)
    near(y[:, some], exact, bound)
    assert bool((out[:, n:] == 7.0).all())
    again = torch.empty(m, n, device=DEV)
    kernels.linear_fp8(kernels.fp8_quantize(x), w8, again)
    assert torch.equal(again, y)
    kernels.linear_fp8(x, w8, again, "relu2")
    near(again[:, some], plain.act(exact, "relu2"), 2 * exact.abs() * bound + bound ** 2 + 2.0 ** -23 * exact ** 2)
    x[m // 2, k // 2] = float("nan")                        # a row that is NaN is no other row's
    kernels.linear_fp8(x, w8, again)
    rest = torch.arange(m, device=DEV) != m // 2
    assert bool(again[m // 2].isnan().all()) and torch.equal(again[rest], y[rest])
    assert kernels.fp8_stream_status() == 0 and kernels.fp8_gemm_status() == 0


@pytest.mark.parametrize("m, n, k", [(2, 65, 40_000), (20, 9_600, 4_200), (64, 130, 66_000), (90, 70, 36_000), (128, 9_600, 4_200), (300, 100, 33_000)])
def test_long_sums_of_gates(m, n, k):
    g = gen(m + n)
    x, gate, up = rows_of(g, m, k, torch.bfloat16, 0.2), *(rows_of(g, n, k, torch.bfloat16, 0.2) * k ** -0.5 for _ in range(2))
    y = torch.empty(m, n, device=DEV)
    kernels.linear_fp8(x, kernels.fp8_gate_up(gate, up), y, "silu")
    some = torch.unique(torch.cat([torch.arange(min(n, 100), device=DEV), torch.arange(max(0, n - 100), n, device=DEV)]))
    xe, ge, ue = plain.values(x), plain.values(gate[some]), plain.values(up[some])
    z, u, bg, bu = xe @ ge.T, xe @ ue.T, sum_bound(xe, ge), sum_bound(xe, ue)
    exact = plain.gated(z, u, "silu")
    # the gate's slope is 1.13 at most, the approximations cost 4e-6 of the result
    near(y[:, some], exact, 1.13 * bg * (u.abs() + bu) + (plain.act(z, "silu").abs() + 1.13 * bg) * bu + 4e-6 * exact.abs())


@pytest.mark.parametrize("t", [3, 40, 300])
def test_long_sums_of_experts(t):
    """A second product of 4,500 along K, streamed (tiles of 16 and 32 rows) and in tiles.  A number between the products whose rounding
    moves within what the first sum may be off is a step away, 2^-3 of it or 2^-8 of its row's largest over 224."""
    g, e, top, width, inter = gen(t), 3, 2, 200, 4_500
    x = rows_of(g, t, width, torch.bfloat16, 0.5)
    ids = torch.topk(torch.randn(t, e, generator=g, device=DEV), top, dim=1).indices.to(torch.int32).contiguous()
    weights = torch.rand(t, top, generator=g, device=DEV) + 0.1
    up, down = (rows_of(g, e * a, b, torch.bfloat16, 0.3).view(e, a, b) * b ** -0.5 for a, b in ((inter, width), (width, inter)))
    up8, down8 = kernels.fp8_quantize(up), kernels.fp8_quantize(down)
    pairs = torch.empty(top, t, width, device=DEV)
    kernels.experts_fp8_pairs(x, ids, up8, down8, pairs, "none")
    exact, bound = torch.zeros(t, width, dtype=torch.float64, device=DEV), torch.zeros(t, width, dtype=torch.float64, device=DEV)
    for k in range(e):
        tok, ch = (ids == k).nonzero(as_tuple=True)
        if not len(tok):
            continue
        xe, ue, de = plain.values(x[tok]), plain.values(up[k]), plain.values(down[k])
        h, off = xe @ ue.T, sum_bound(xe, ue)
        h8 = plain.values(h)
        tight = (plain.values(h + off) != h8) | (plain.values(h - off) != h8)
        step = 2.0 ** -3 * h.abs() + 2.0 ** -8 * h.abs().amax(dim=1, keepdim=True) / 224.0
        y, yb = h8 @ de.T, sum_bound(h8, de) + (tight * step) @ de.abs().T
        near(pairs[ch, tok], y, yb)
        s = weights[tok, ch].double()[:, None]
        exact.index_add_(0, tok, s * y)
        bound.index_add_(0, tok, s * yb + 2.0 ** -22 * (s * y).abs())
    out = torch.empty(t, width, device=DEV)
    kernels.experts_fp8(x, ids, weights, up8, down8, out, "none")
    near(out, exact, bound)


@pytest.mark.parametrize("m", [8, 40, 100, 129])
def test_sums_of_positive_terms_do_not_drift(m):
    """With all terms positive the running sum of a piece is half of its end on average, and what is cut off has one sign: at most
    4 * 32 * 2^-23 / 2 = 7.6e-6 of the result, and 17 roundings of running sums, half of 17 * 2^-24: 5e-7.  Without pieces it is
    sixteen times the first (512 blocks), of which a third was seen."""
    g, n, k = gen(m), 19_000, 65_536
    w = torch.randn(n, k, generator=g, device=DEV, dtype=torch.bfloat16).abs_()
    x = torch.randn(m, k, generator=g, device=DEV).abs_()
    w8 = kernels.fp8_quantize(w)
    y = torch.empty(m, n, device=DEV)
    kernels.linear_fp8(x, w8, y)
    for some in (slice(0, 100), slice(9_000, 9_100), slice(n - 100, n)):
        exact = plain.values(x) @ plain.values(w[some]).T
        assert float((y[:, some].double() - exact).norm() / exact.norm()) <= 8.1e-6


def test_a_matrix_beyond_two_gigabytes_to_the_bound_of_its_sums():
    g, n, k = gen(17), 70_000, 32_768
    w = torch.empty(n, k, dtype=torch.bfloat16, device=DEV)
    for a in range(0, n, 7000):
        w[a:a + 7000] = torch.randn(7000, k, generator=g, device=DEV)
    w8 = kernels.fp8_quantize(w)
    x = rows_of(g, 3, k, torch.bfloat16)
    y = torch.empty(3, n, device=DEV)
    kernels.linear_fp8(x, w8, y)
    xe = plain.values(x)
    for some in (slice(0, 40), slice(65_500, 65_580), slice(n - 40, n)):
        we = plain.values(w[some])
        exact = xe @ we.T
        near(y[:, some], exact, sum_bound(xe, we))
        # a block of 128 that is lost, or a scale that is another's, is a sixteenth of a result
        assert float((y[:, some].double() - exact).norm() / exact.norm()) <= 1e-4


LIMIT = 8_000_000            # clock cycles: about four milliseconds


@pytest.mark.parametrize("code", [2, 3, 5])
@pytest.mark.parametrize("m, n, k", [(8, 300, 40_000), (100, 300, 40_000), (100, 19_000, 4_300)])
def test_a_wait_in_a_long_sum_that_runs_out(m, n, k, code):
    g = gen(m)
    x, w = rows_of(g, m, k, torch.bfloat16), kernels.fp8_quantize(rows_of(g, n, k, torch.bfloat16, 0.3))

    def run():
        out = torch.empty(m, n, device=DEV)
        kernels.linear_fp8(x, w, out)
        torch.cuda.synchronize()
        return out
    good = run()
    assert kernels.fp8_stream_status(reset=True) == 0
    kernels.wait_control("fp8_stream", cycles=LIMIT, stall_code=code)
    try:
        run()
        assert kernels.fp8_stream_status(reset=True) == code and kernels.fp8_stream_status() == 0
    finally:
        kernels.wait_control("fp8_stream", 0, 0)
    assert torch.equal(run(), good) and kernels.fp8_stream_status() == 0
