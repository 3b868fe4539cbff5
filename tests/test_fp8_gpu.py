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


def case(m, n, k, seed=11, gated=False):
    g = gen(seed)
    x, w = rows_of(g, m, k, torch.bfloat16), rows_of(g, n * (2 if gated else 1), k, torch.bfloat16, 0.3) * k ** -0.5
    return x, (kernels.fp8_gate_up(w[:n].contiguous(), w[n:].contiguous()) if gated else kernels.fp8_quantize(w))


LIMIT = 8_000_000            # clock cycles: about four milliseconds


@pytest.mark.parametrize("library, code, m, n, k, gated", [
    ("fp8_stream", 1, 20, 200, 9216, False), ("fp8_stream", 2, 8, 2304, 2304, False), ("fp8_stream", 3, 100, 700, 1000, False),
    ("fp8_stream", 5, 8, 700, 640, True), ("fp8_stream", 6, 8, 2304, 2304, False), ("fp8_gemm", 1, 300, 700, 2304, False), ("fp8_gemm", 2, 300, 700, 2304, False),
    ("fp8_gemm", 3, 300, 700, 640, True), ("fp8_gemm", 5, 300, 700, 640, False), ("fp8_gemm", 6, 300, 700, 640, False), ("fp8_gemm", 7, 300, 700, 640, True)])
def test_a_wait_that_runs_out_is_reported_and_the_next_call_is_right(library, code, m, n, k, gated):
    status = {"fp8_stream": kernels.fp8_stream_status, "fp8_gemm": kernels.fp8_gemm_status}[library]
    x, w = case(m, n, k, gated=gated)
    down = case(1, 40, n)[1]

    def run():
        out = torch.empty(m, 40 if code == 7 else n, dtype=torch.float32, device=DEV)
        if code == 7:                                            # the two warps that share a block of 128 results
            kernels.feedforward_fp8(x, w, down, out, "silu")
        else:
            kernels.linear_fp8(x, w, out, "silu" if gated else "none")
        torch.cuda.synchronize()
        return out
    good = run()
    assert status(reset=True) == 0
    kernels.wait_control(library, cycles=LIMIT, stall_code=code)
    try:
        run()
        assert status(reset=True) == code and status() == 0
    finally:
        kernels.wait_control(library, 0, 0)
    assert torch.equal(run(), good) and status() == 0


@pytest.mark.parametrize("rows", [8, 600])
def test_experts_whose_wait_runs_out(rows):
    g = gen(12)
    x, ids, w = rows_of(g, rows, 256, torch.bfloat16), routed(g, rows, 2, 2, "even"), torch.rand(rows, 2, generator=g, device=DEV)
    up, down = (kernels.fp8_quantize(rows_of(g, 2 * a, b, torch.bfloat16).view(2, a, b) * 0.1) for a, b in ((128, 256), (256, 128)))
    library, status = ("fp8_stream", kernels.fp8_stream_status) if rows == 8 else ("fp8_gemm", kernels.fp8_gemm_status)

    def run():
        out = torch.empty(rows, 256, dtype=torch.float32, device=DEV)
        kernels.experts_fp8(x, ids, w, up, down, out, "relu2")
        torch.cuda.synchronize()
        return out
    good = run()
    kernels.wait_control(library, cycles=LIMIT, stall_code=2)
    try:
        run()
        assert status(reset=True) == 2 and status() == 0
    finally:
        kernels.wait_control(library, 0, 0)
    assert torch.equal(run(), good) and status() == 0


def test_a_matrix_made_right_before_it_is_used():
    """The products read their matrix before they wait for the kernel before them; the one that makes it ends before."""
    g = gen(13)
    x = rows_of(g, 8, 2304, torch.bfloat16)
    xs = rows_of(g, 200, 2304, torch.bfloat16)
    ws = [rows_of(g, 4096, 2304, torch.bfloat16) for _ in range(3)]
    want = []
    for w in ws:
        m = kernels.fp8_quantize(w)
        torch.cuda.synchronize()
        want.append([torch.empty(len(t), 4096, device=DEV) for t in (x, xs)])
        for t, o in zip((x, xs), want[-1]):
            kernels.linear_fp8(t, m, o)
    torch.cuda.synchronize()
    for turn in range(12):
        w = ws[turn % 3]
        outs = [torch.full((len(t), 4096), 7.0, device=DEV) for t in (x, xs)]
        kernels.linear_fp8(x, kernels.fp8_quantize(w), outs[0])
        kernels.linear_fp8(xs, kernels.fp8_quantize(w), outs[1])
        for o, good in zip(outs, want[turn % 3]):
            assert torch.equal(o, good)


def passes():
    """A few calls of every kind: (inputs that change, a function that fills `out`)."""
    g = gen(14)
    made = []
    for m, n, k in ((3, 500, 640), (40, 700, 1100), (300, 600, 640)):
        x, w = case(m, n, k, seed=m)
        made.append((x, torch.empty(m, n, device=DEV), lambda x, o, w=w: kernels.linear_fp8(x, w, o)))
    for m in (5, 200):
        x, gu = case(m, 320, 256, seed=m, gated=True)
        d = case(1, 256, 320, seed=m + 1)[1]
        made.append((x, torch.empty(m, 256, device=DEV), lambda x, o, gu=gu, d=d: kernels.feedforward_fp8(x, gu, d, o, "silu")))
    for t in (6, 300):
        ids, w = routed(g, t, 2, 4, "even"), torch.rand(t, 2, generator=g, device=DEV)
        up, down = (kernels.fp8_quantize(rows_of(g, 4 * a, b, torch.bfloat16).view(4, a, b) * 0.1) for a, b in ((96, 256), (256, 96)))
        made.append((rows_of(g, t, 256, torch.bfloat16), torch.empty(t, 256, device=DEV),
                     lambda x, o, ids=ids, w=w, up=up, down=down: kernels.experts_fp8(x, ids, w, up, down, o, "relu2")))
    return made


def test_captured_calls_of_new_inputs_and_two_graphs_at_once():
    made = passes()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, statics, outs = [], [], []
    for i, s in enumerate(streams):
        xs, os = [x.clone() for x, _, _ in made], [torch.empty_like(o) for _, o, _ in made]
        with torch.cuda.stream(s):
            for x, o, (_, _, f) in zip(xs, os, made):
                f(x, o)                                          # libraries are there before a capture
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            for x, o, (_, _, f) in zip(xs, os, made):
                f(x, o)
        graphs.append(graph), statics.append(xs), outs.append(os)
    for turn in range(4):
        want = []
        for i in range(2):
            for x, (x0, _, _) in zip(statics[i], made):
                x.copy_(x0 * (1.0 + 0.25 * turn + i))
            row = []
            for x, (_, o, f) in zip(statics[i], made):
                f(x, o)
                row.append(o.clone())
            want.append(row)
        for os in outs:
            for o in os:
                o.fill_(7.0)
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(3):
                    graph.replay()
        torch.cuda.synchronize()
        for i in range(2):
            for o, w in zip(outs[i], want[i]):
                assert torch.equal(o, w)


def test_a_stream_that_is_not_the_default_one():
    made = passes()
    want = []
    for x, o, f in made:
        f(x, o)
        want.append(o.clone())
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    slow = torch.randn(4096, 4096, device=DEV)
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(10):
            slow = slow @ slow * 1e-3                            # what follows is behind this
        got = []
        for x, o, f in made:
            fresh = x * 1.0
            out = torch.full_like(o, 7.0)
            f(fresh, out)
            got.append(out)
    s.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("act", ["relu2", "none", "silu", "gelu_tanh", "clamped_gate"])
def test_a_token_that_is_not_finite_is_nobody_elses(act):
    g = gen(15)
    for t in (6, 300):
        ids, w = routed(g, t, 2, 3, "even"), torch.rand(t, 2, generator=g, device=DEV)
        up, gate = (rows_of(g, 3 * 128, 256, torch.bfloat16).view(3, 128, 256) * 0.1 for _ in range(2))
        down = kernels.fp8_quantize(rows_of(g, 3 * 256, 128, torch.bfloat16).view(3, 256, 128) * 0.1)
        up = kernels.fp8_quantize(up) if act in ("relu2", "none") else kernels.fp8_gate_up(gate, up)
        x = rows_of(g, t, 256, torch.bfloat16)
        out, bad = torch.empty(t, 256, device=DEV), torch.empty(t, 256, device=DEV)
        kernels.experts_fp8(x, ids, w, up, down, out, act, 2.0)
        x[2, 5] = float("nan")
        kernels.experts_fp8(x, ids, w, up, down, bad, act, 2.0)
        others = torch.arange(t, device=DEV) != 2
        assert bool(torch.isnan(bad[2]).all()) and torch.equal(bad[others], out[others])


def test_many_experts_and_many_pairs():
    """More experts than a block has threads, and more pairs than the cluster that sorts them looks at in one go."""
    g = gen(16)
    e, t, top = 1500, 17000, 3
    ids = torch.randint(0, e, (t, top), generator=g, device=DEV, dtype=torch.int32)
    x, w = rows_of(g, t, 32, torch.bfloat16), torch.rand(t, top, generator=g, device=DEV)
    up, down = (rows_of(g, e * a, b, torch.bfloat16).view(e, a, b) * 0.3 for a, b in ((16, 32), (32, 16)))
    out = torch.empty(t, 32, device=DEV)
    kernels.experts_fp8(x, ids, w, kernels.fp8_quantize(up), kernels.fp8_quantize(down), out, "none")
    some = torch.randint(0, t, (200,), generator=g, device=DEV)
    xe, ue, de = plain.values(x[some]), read(kernels.fp8_quantize(up)).double(), read(kernels.fp8_quantize(down)).double()
    for i, tok in enumerate(some.tolist()):
        want = torch.zeros(32, dtype=torch.float64, device=DEV)
        for c in range(top):
            k = int(ids[tok, c])
            # (sums of 32 and 16 numbers: a border is missed by too little to matter to a number's step)
            want += float(w[tok, c]) * (plain.values((xe[i] @ ue[k].T)[None])[0] @ de[k].T)
        assert float((out[tok].double() - want).norm()) <= 0.05 * float(want.norm())
    assert float((out[some].double()).norm()) > 0


def test_matrices_beyond_two_gigabytes():
    g = gen(17)
    n, k = 70_000, 32_768
    w = torch.empty(n, k, dtype=torch.bfloat16, device=DEV)
    for a in range(0, n, 7000):
        w[a:a + 7000] = torch.randn(7000, k, generator=g, device=DEV)
    w8 = kernels.fp8_quantize(w)
    assert w8.nbytes > 2 ** 31
    last = plain.values(w[-3:, -2048:])
    back = torch.empty(n, k, dtype=torch.bfloat16, device=DEV)
    kernels.fp8_read(w8, back)
    assert torch.equal(back[-3:, -2048:].double(), last)
    del back
    x = rows_of(g, 3, k, torch.bfloat16)
    y = torch.empty(3, n, device=DEV)
    kernels.linear_fp8(x, w8, y)
    xe = plain.values(x)
    for some in (slice(0, 40), slice(65_500, 65_580), slice(n - 40, n)):
        we = plain.values(w[some])
        near(y[:, some], xe @ we.T, sum_bound(xe, we) * 20)     # (256 blocks of K in slices of a part of them)
    # rows beyond two gigabytes, a result beyond two billion numbers
    few = kernels.fp8_quantize(w[:33_000])
    del w, w8
    wide = kernels.fp8_quantize(torch.randn(66_000, 128, generator=g, device=DEV))
    x = rows_of(g, 33_000, 128, torch.bfloat16)
    y = torch.empty(33_000, 66_000, dtype=torch.bfloat16, device=DEV)
    kernels.linear_fp8(x, wide, y)
    xe, we = plain.values(x[-200:]), read(wide).double()[-300:]
    exact = xe @ we.T
    near(y[-200:, -300:], exact, rounded(sum_bound(xe, we), exact, torch.bfloat16))
    del y, few


def test_refusals_on_the_device():
    x, w = case(5, 64, 256)
    out = torch.empty(5, 64, device=DEV)
    for bad, what in ((dict(x=x.half()), "float16"), (dict(x=x[:, :128]), "256 numbers"), (dict(out=out[:4]), "shape"), (dict(out=out.half()), "float16"),
                      (dict(x=x.cpu()), "CUDA"), (dict(out=out.cpu()), "CUDA"), (dict(out=torch.empty(64, 5, device=DEV).T), "packed"),
                      (dict(x=x.t().contiguous().t()), "packed"), (dict(out=torch.empty(64, device=DEV).expand(5, 64)), "over one another"), (dict(x=x[0]), "dimensions")):
        args = dict(x=x, w=w, out=out) | bad
        with pytest.raises(kernels.KernelError, match=what):
            kernels.linear_fp8(**args)
    g = gen(18)
    up, down = (kernels.fp8_quantize(rows_of(g, 3 * a, b, torch.bfloat16).view(3, a, b)) for a, b in ((64, 256), (256, 64)))
    ids, weights, y = routed(g, 5, 2, 3, "even"), torch.rand(5, 2, device=DEV), torch.empty(5, 256, device=DEV)
    for bad, what in ((dict(ids=ids.long()), "int32"), (dict(ids=ids[:4]), "ids"), (dict(weights=weights.double()), "float32"), (dict(weights=weights[:, :1]), "float32"),
                      (dict(up=w), "follow"), (dict(down=up), "follow"), (dict(activation="silu"), "relu2"), (dict(out=y[:3]), "shape"), (dict(x=x[:, :8]), "256 numbers")):
        args = dict(x=x, ids=ids, weights=weights, up=up, down=down, out=y, activation="relu2") | bad
        with pytest.raises(kernels.KernelError, match=what):
            kernels.experts_fp8(**args)
    with pytest.raises(kernels.KernelError, match="contiguous"):
        kernels.fp8_quantize(torch.zeros(2, 4, 8, device=DEV).transpose(0, 1))
    none = torch.empty(5, 256, device=DEV)
    kernels.experts_fp8(x, ids[:, :0].contiguous(), weights[:, :0].contiguous(), up, down, none, "relu2")
    assert bool((none == 0).all())


@pytest.mark.parametrize("m", [3, 40, 200])
def test_products_of_very_small_and_very_large_numbers(m):
    """Scales at both ends of their range meet in a product: 2^-127 (where nothing is smaller) with 2^100, their sums moderate."""
    g = gen(19)
    x, w = torch.randn(m, 512, generator=g, device=DEV), torch.randn(300, 512, generator=g, device=DEV)
    x[:, :128] *= 2.0 ** -134                          # below the smallest scale's normal numbers
    w[:, :128] *= 2.0 ** 115
    x[:, 128:256] *= 2.0 ** -110
    w[:, 128:256] *= 2.0 ** 108
    x[:, 256:384] *= 2.0 ** 90
    w[:, 256:384] *= 2.0 ** -100
    x[1, 384:] = 0.0
    y = torch.empty(m, 300, device=DEV)
    kernels.linear_fp8(x, kernels.fp8_quantize(w), y)
    xe, we = plain.values(x), plain.values(w)
    near(y, xe @ we.T, sum_bound(xe, we))
    for a, b in ((0, 128), (128, 256), (256, 384)):    # every block by itself
        only = torch.zeros_like(x)
        only[:, a:b] = x[:, a:b]
        kernels.linear_fp8(only, kernels.fp8_quantize(w), y)
        oe = plain.values(only)
        assert float((oe @ we.T).abs().max()) > 0
        near(y, oe @ we.T, sum_bound(oe, we))


def test_rows_that_lie_over_one_another_are_not_read_into():
    m = kernels.fp8_quantize(rows_of(gen(41), 4, 64, torch.bfloat16))
    room = torch.full((256,), 7.0, device=DEV)
    with pytest.raises(kernels.KernelError, match="over one another"):
        kernels.fp8_read(m, room.as_strided((4, 64), (32, 1)))
    with pytest.raises(kernels.KernelError, match="over one another"):
        kernels.fp8_read(m, room[:64].expand(4, 64))
    assert (room == 7.0).all()
    kernels.fp8_read(m, room.view(4, 64))
    assert torch.equal(room.view(4, 64), read(m))


@pytest.mark.parametrize("top", [1, 3])
def test_passes_of_experts_one_right_after_the_other(top):
    """A pass's kernels begin before those ahead of them have ended: many passes without a wait give what one at a time gives."""
    g, e, width, inter = gen(42), 6, 512, 256
    up = kernels.fp8_gate_up(*(rows_of(g, e * inter, width, torch.bfloat16).view(e, inter, width) * 0.1 for _ in range(2)))
    down = kernels.fp8_quantize(rows_of(g, e * width, inter, torch.bfloat16).view(e, width, inter) * 0.1)
    calls = []
    for t in (1, 8, 90, 300, 700):
        calls.append((rows_of(g, t, width, torch.bfloat16), routed(g, t, top, e, "even"), torch.rand(t, top, generator=g, device=DEV)))

    def run(i):
        x, ids, w = calls[i]
        out = torch.full((len(x), width), 7.0, dtype=torch.bfloat16, device=DEV)
        kernels.experts_fp8(x, ids, w, up, down, out)
        return out
    good = []
    for i in range(len(calls)):
        good.append(run(i))
        torch.cuda.synchronize()
    order = torch.randint(len(calls), (60,), generator=torch.Generator().manual_seed(1)).tolist()
    outs = [run(i) for i in order]
    # each pass also reads what the one before left.  (Results are some hundred times the square of what goes in: the first four
    # are finite, then blocks are NaN; so the bits are compared.)
    def chain(wait):
        left = [calls[1][0]]
        for _ in range(6):
            left.append(torch.empty_like(left[0]))
            kernels.experts_fp8(left[-2], calls[1][1], calls[1][2], up, down, left[-1])
            if wait:
                torch.cuda.synchronize()
        torch.cuda.synchronize()
        return left
    chained, again = chain(False), chain(True)
    for i, out in zip(order, outs):
        assert torch.equal(out, good[i])
    for a, b in zip(chained, again):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))
    assert chained[2].isfinite().all()
    assert kernels.fp8_stream_status() == 0 and kernels.fp8_gemm_status() == 0


@pytest.mark.parametrize("m, width, inter, name", [
    (1, 100, 30, "silu"), (8, 256, 64, "gelu_tanh"), (8, 128, 65, "silu"), (16, 200, 129, "clamped_gate"), (17, 256, 384, "silu"), (33, 130, 200, "gelu_tanh"),
    (64, 256, 1000, "silu"), (128, 1024, 8500, "silu"), (3, 256, 20000, "gelu_tanh"), (8, 2304, 9216, "gelu_tanh"), (5, 256, 130, "relu2"), (64, 128, 1111, "relu2"),
    (40, 256, 300, "none"), (2, 64, 40000, "relu2")])
def test_a_feedforward_is_its_two_products(m, width, inter, name):
    """What a product leaves in 8 bits is what it leaves as floats, rounded: the same bits come out."""
    g = gen(m + inter)
    x = rows_of(g, m, width, torch.bfloat16, 0.5)
    mats = [rows_of(g, inter, width, torch.bfloat16, 0.3) * width ** -0.5 for _ in range(1 if name in ("relu2", "none") else 2)]
    up = kernels.fp8_quantize(mats[0]) if len(mats) == 1 else kernels.fp8_gate_up(*mats)
    down = kernels.fp8_quantize(rows_of(g, width, inter, torch.bfloat16, 0.3) * inter ** -0.5)
    x[m // 2, width // 3] = float("inf") if m > 2 else 1.0          # a row that is NaN is no other row's
    for t in (x, kernels.fp8_quantize(x), x.float()):
        h = torch.empty(m, inter, dtype=torch.float32, device=DEV)
        kernels.linear_fp8(t, up, h, name, 1.5)
        good, y = (torch.full((m, width), 7.0, device=DEV) for _ in range(2))
        kernels.linear_fp8(kernels.fp8_quantize(h), down, good)
        kernels.feedforward_fp8(t, up, down, y, name, 1.5)
        assert torch.equal(y.view(torch.int32), good.view(torch.int32))
        assert y.isnan().any(dim=1).sum() == (1 if m > 2 else 0) and y[0].isfinite().all()
    assert kernels.fp8_stream_status() == 0 and kernels.fp8_gemm_status() == 0


@pytest.mark.parametrize("name", ["silu", "relu2"])
def test_a_block_of_results_that_waits_in_vain(name):
    """The warps that share a block of results in 8 bits, of one block and of two, give up in the end."""
    g = gen(51)
    x, up, down = rows_of(g, 8, 256, torch.bfloat16), *(rows_of(g, a, b, torch.bfloat16) * 0.1 for a, b in ((600, 256), (256, 300 if name == "silu" else 600)))
    w = kernels.fp8_quantize(up) if name == "relu2" else kernels.fp8_gate_up(up[:300].contiguous(), up[300:].contiguous())
    d = kernels.fp8_quantize(down)

    def run():
        out = torch.empty(8, 256, dtype=torch.float32, device=DEV)
        kernels.feedforward_fp8(x, w, d, out, name)
        torch.cuda.synchronize()
        return out
    good = run()
    assert kernels.fp8_stream_status(reset=True) == 0
    kernels.wait_control("fp8_stream", cycles=LIMIT, stall_code=7)
    try:
        run()
        assert kernels.fp8_stream_status(reset=True) == 7 and kernels.fp8_stream_status() == 0
    finally:
        kernels.wait_control("fp8_stream", 0, 0)
    assert torch.equal(run(), good) and kernels.fp8_stream_status() == 0


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("post", [True, False])
@pytest.mark.parametrize("m, n", [(1, 4), (3, 100), (2, 128), (1, 1024), (9, 1028), (130, 2304), (8, 2308), (5, 4608), (3, 5124), (2, 8192), (300, 640)])
def test_a_norm_that_leaves_8_bits(m, n, post, dtype):
    """Against 64 bits.  Float sums of n squares, 32 additions one after the other at most, a root and three products: 2^-18 of
    the result, for each of the two norms; the sum of h one rounding.  Then 8 bits: half a step, 2^-4 of the number, or of the
    smallest one, 2^-10 of a scale that is a 224th of the block's largest number at most."""
    g = gen(m + n)
    h, y = (rows_of(g, m, n, torch.float32, 0.5) for _ in range(2))
    wp, wn = ((0.2 * torch.randn(n, generator=g, device=DEV)).to(dtype) for _ in range(2))
    v = y.double()
    if post:
        v = v * (v.square().mean(dim=1, keepdim=True) + 1e-6).rsqrt() * (1.0 + wp.double())
    total = h.double() + v
    off_h = 2.0 ** -18 * v.abs() + 2.0 ** -24 * total.abs()
    gain = (total.square().mean(dim=1, keepdim=True) + 1e-5).rsqrt() * (0.5 + wn.double())
    exact = total * gain
    off = 2.0 ** -17 * exact.abs() + off_h * gain.abs()
    # the root moves with h: by its largest relative change at most
    off = off + exact.abs() * (off_h.norm(dim=1, keepdim=True) / total.norm(dim=1, keepdim=True))
    blocks = torch.nn.functional.pad(exact.abs() + off, (0, -n % 128)).unflatten(1, (-1, 128)).amax(dim=2).repeat_interleave(128, dim=1)[:, :n]
    bound = off + 2.0 ** -4 * (exact.abs() + off) + 2.0 ** -10 * blocks / 224.0
    m8 = kernels.residual_rmsnorm_fp8(h, y, wp if post else None, 1e-6, 1.0, wn, 1e-5, 0.5)
    assert m8.shape == (m, n) and bool(((h.double() - total).abs() <= off_h).all())
    got = read(m8)
    near(got, exact, bound)
    assert torch.equal(read(kernels.fp8_quantize(got)), got) and torch.equal(m8.float(), got)
    w = kernels.fp8_quantize(rows_of(g, 40, n, torch.bfloat16))
    a, b = torch.empty(m, 40, device=DEV), torch.empty(m, 40, device=DEV)
    kernels.linear_fp8(m8, w, a)
    kernels.linear_fp8(kernels.fp8_quantize(got), w, b)
    assert torch.equal(a, b)


def test_a_norm_in_8_bits_of_rows_that_are_not_finite_and_of_none():
    g = gen(61)
    h, y, w = rows_of(g, 4, 300, torch.float32), rows_of(g, 4, 300, torch.float32), torch.ones(300, device=DEV)
    y[1, 17], y[2, 5] = float("inf"), float("nan")
    good = [read(kernels.residual_rmsnorm_fp8(h[i:i + 1].clone(), y[i:i + 1].clone(), w, 1e-6, 0.0, w, 1e-6, 0.0)) for i in (0, 3)]
    got = read(kernels.residual_rmsnorm_fp8(h, y, w, 1e-6, 0.0, w, 1e-6, 0.0))
    assert torch.equal(got[0:1], good[0]) and torch.equal(got[3:4], good[1]) and bool(got[1:3].isnan().all())
    assert kernels.residual_rmsnorm_fp8(h[:0], y[:0], None, 0.0, 0.0, w, 1e-6, 0.0).shape == (0, 300)
    zero = torch.zeros(2, 300, device=DEV)
    assert not read(kernels.residual_rmsnorm_fp8(zero, zero.clone(), None, 0.0, 0.0, w, 1e-6, 0.0)).any()


def test_refusals_of_the_norm_in_8_bits():
    h, y, w = torch.zeros(2, 64, device=DEV), torch.zeros(2, 64, device=DEV), torch.ones(64, device=DEV)
    call = lambda h, y, post, nxt: kernels.residual_rmsnorm_fp8(h, y, post, 1e-6, 0.0, nxt, 1e-6, 0.0)
    for args, what in (((h.bfloat16(), y, None, w), "float32"), ((h, y[:1], None, w), "rows, hidden"), ((h, torch.zeros(2, 128, device=DEV)[:, ::2], None, w), "packed"),
                       ((h[:, :6].contiguous(), y[:, :6].contiguous(), None, w[:6]), "multiple of 4"), ((h, y, None, w[:60]), "gains"),
                       ((torch.zeros(1, 8196, device=DEV), torch.zeros(1, 8196, device=DEV), None, torch.ones(8196, device=DEV)), "8,192"),
                       ((h, y, w.bfloat16(), w), "gains"), ((h, y, None, w.cpu()), "gains"), ((h.cpu(), y, None, w), "CUDA"), ((h, y.half(), None, w), "float32")):
        with pytest.raises(kernels.KernelError, match=what):
            call(*args)
    odd = torch.zeros(2 * 64 + 1, device=DEV)[1:].view(2, 64)           # a base that is no border of 16 bytes
    with pytest.raises(kernels.KernelError):
        call(odd, y, None, w)
    assert not h.any() and not y.any()


@pytest.mark.parametrize("m", [3, 60, 300])
def test_a_new_matrix_is_not_read_ahead_of_what_makes_it(m):
    """One that is made in the stream right before its first product, by this package's kernel or by another's, through a norm whose
    next kernel may begin before it has ended, too."""
    g = gen(71)
    h, y, gain = rows_of(g, m, 1024, torch.float32), torch.zeros(m, 1024, device=DEV), torch.ones(1024, device=DEV)
    x = kernels.residual_rmsnorm_fp8(h.clone(), y, None, 0.0, 0.0, gain, 1e-6, 0.0)
    ws = [rows_of(g, 5000, 1024, torch.bfloat16) for _ in range(3)]
    want = []
    for w in ws:
        m8 = kernels.fp8_quantize(w)
        assert m8.fresh
        torch.cuda.synchronize()
        want.append(torch.empty(m, 5000, device=DEV))
        kernels.linear_fp8(x, m8, want[-1])
        assert not m8.fresh
    old = kernels.fp8_quantize(ws[0])
    data = [kernels.fp8_quantize(w).data for w in ws]
    torch.cuda.synchronize()
    for turn in range(12):
        out, again, other = (torch.full((m, 5000), 7.0, device=DEV) for _ in range(3))
        m8 = kernels.fp8_quantize(ws[turn % 3])
        x2 = kernels.residual_rmsnorm_fp8(h.clone(), y, None, 0.0, 0.0, gain, 1e-6, 0.0) if turn % 2 else x
        kernels.linear_fp8(x2, m8, out)
        kernels.linear_fp8(x2, m8, again)
        copied = kernels.Fp8Matrix(old.data.clone(), old.shape)
        copied.data.copy_(data[turn % 3])
        kernels.linear_fp8(x2, copied, other)
        for o in (out, again, other):
            assert torch.equal(o, want[turn % 3])
    up, down = kernels.fp8_gate_up(ws[0], ws[1]), kernels.fp8_quantize(rows_of(g, 64, 5000, torch.bfloat16))
    assert up.fresh and down.fresh
    kernels.feedforward_fp8(x, up, down, torch.empty(m, 64, device=DEV), "silu")
    assert not up.fresh and not down.fresh
