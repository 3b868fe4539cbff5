"""Matrices in 8-bit floating point right after they are made, on several streams, captured, and copied."""
import copy

import pytest
import torch

from brolm_b200 import kernels
from tests.plain import fp8_plain as plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rows_of(g, m, k, spread=0.3):
    return (torch.randn(m, k, generator=g, device=DEV) * torch.exp(spread * torch.randn(k, generator=g, device=DEV))).to(torch.bfloat16)


@pytest.mark.parametrize("m", [1, 8, 60, 300])
def test_a_matrix_whose_first_product_is_another_streams(m):
    """The other stream waits for the matrix by an event; the making stream multiplies right behind what makes it, never having waited."""
    g = gen(m)
    x, ws = rows_of(g, m, 2304), [rows_of(g, 4096, 2304) for _ in range(3)]
    want = []
    for w in ws:
        w8 = kernels.fp8_quantize(w)
        torch.cuda.synchronize()
        want.append(torch.empty(m, 4096, device=DEV))
        kernels.linear_fp8(x, w8, want[-1])
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    made, outs = [], []
    for turn in range(12):
        a, b = torch.full((m, 4096), 7.0, device=DEV), torch.full((m, 4096), 7.0, device=DEV)
        w8 = kernels.fp8_quantize(ws[turn % 3])
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            kernels.linear_fp8(x, w8, b)
        assert w8.fresh
        kernels.linear_fp8(x, w8, a)
        assert not w8.fresh
        made.append(w8), outs.append((a, b))              # (nothing is freed while the other stream reads it)
    torch.cuda.synchronize()
    for turn, (a, b) in enumerate(outs):
        assert torch.equal(a, want[turn % 3]) and torch.equal(b, want[turn % 3])


def test_a_matrix_whose_first_product_is_captured():
    g = gen(5)
    x, w = rows_of(g, 8, 2304), rows_of(g, 4096, 2304)
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    kernels.linear_fp8(x, kernels.fp8_quantize(w), torch.empty(8, 4096, device=DEV))       # the libraries are there
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        w8 = kernels.fp8_quantize(w)
    torch.cuda.synchronize()
    static, eager, want = (torch.full((8, 4096), 7.0, device=DEV) for _ in range(3))
    with torch.cuda.graph(graph, stream=side):
        kernels.linear_fp8(x, w8, static)
    assert w8.fresh                                        # nothing has run yet
    with torch.cuda.stream(side):
        kernels.linear_fp8(x, w8, eager)
        assert not w8.fresh
        for _ in range(3):
            graph.replay()
    torch.cuda.synchronize()
    kernels.linear_fp8(x, kernels.fp8_quantize(w), want)
    assert torch.equal(static, want) and torch.equal(eager, want)


def test_what_a_capture_makes_and_multiplies():
    """The matrix is made anew by every replay, and its product is captured behind it."""
    g = gen(6)
    x, w = rows_of(g, 8, 1024), rows_of(g, 5000, 1024)
    y, want = torch.empty(8, 5000, device=DEV), torch.empty(8, 5000, device=DEV)
    kernels.linear_fp8(x, kernels.fp8_quantize(w), y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w8 = kernels.fp8_quantize(w)
        kernels.linear_fp8(x, w8, y)
        kernels.linear_fp8(x, w8, y)
    for turn in range(4):
        w.copy_(rows_of(g, 5000, 1024))
        y.fill_(7.0)
        graph.replay()
        kernels.linear_fp8(x, kernels.fp8_quantize(w), want)
        assert torch.equal(y, want)


@pytest.mark.parametrize("m", [8, 200])
def test_a_copied_matrix_after_the_first_is_gone(m):
    g = gen(7)
    x, w = rows_of(g, m, 640), rows_of(g, 700, 640)
    first = kernels.fp8_quantize(w)
    want, y = torch.empty(m, 700, device=DEV), torch.empty(m, 700, device=DEV)
    kernels.linear_fp8(x, first, want)
    second = copy.deepcopy(first)
    first.data.fill_(0)
    kernels.linear_fp8(x, second, y)
    assert torch.equal(y, want) and not torch.equal(first.float(), second.float())


def test_thousands_of_experts_to_the_bound_of_their_sums():
    """More experts than a block has threads and more pairs than the cluster that sorts them looks at in one go, number by number.  Sums
    of 32 and of 16 numbers: one addition of 32 products and one of the accumulator, 2^-23 each, a rounding for each of the three
    choices; a number between whose rounding moves within that is a step away."""
    g = gen(16)
    e, t, top = 1500, 17_000, 3
    ids = torch.randint(-1, e + 1, (t, top), generator=g, device=DEV, dtype=torch.int32)
    x, weights = rows_of(g, t, 32), torch.rand(t, top, generator=g, device=DEV)
    up, down = (rows_of(g, e * a, b).view(e, a, b) * 0.3 for a, b in ((16, 32), (32, 16)))
    out = torch.empty(t, 32, device=DEV)
    kernels.experts_fp8(x, ids, weights, kernels.fp8_quantize(up), kernels.fp8_quantize(down), out, "none")
    some = torch.cat([torch.randint(0, t, (200,), generator=g, device=DEV), torch.tensor([0, t - 1], device=DEV)])
    used = torch.unique(ids[some].clamp(0, e - 1)).long()
    place = torch.zeros(e, dtype=torch.long, device=DEV)
    place[used] = torch.arange(len(used), device=DEV)
    xe, ue, de = plain.values(x[some]), plain.values(up[used]), plain.values(down[used])
    exact, bound = (torch.zeros(len(some), 32, dtype=torch.float64, device=DEV) for _ in range(2))
    for c in range(top):
        k = ids[some, c].long()
        there = ((k >= 0) & (k < e)).double()[:, None]
        at = place[k.clamp(0, e - 1)]
        h = torch.einsum("tk,tnk->tn", xe, ue[at])
        off = 4 * 2.0 ** -23 * torch.einsum("tk,tnk->tn", xe.abs(), ue[at].abs())
        h8 = plain.values(h)
        tight = (plain.values(h + off) != h8) | (plain.values(h - off) != h8)
        step = 2.0 ** -3 * h.abs() + 2.0 ** -8 * h.abs().amax(dim=1, keepdim=True) / 224.0
        s = weights[some, c].double()[:, None] * there
        y = torch.einsum("tn,tkn->tk", h8, de[at])
        yb = 4 * 2.0 ** -23 * torch.einsum("tn,tkn->tk", h8.abs(), de[at].abs()) + torch.einsum("tn,tkn->tk", tight * step, de[at].abs())
        exact += s * y
        bound += s * yb + 2.0 ** -22 * (s * y).abs()
    assert bool(((out[some].double() - exact).abs() <= bound).all())
    few = some[:20]
    weight = torch.where((ids[few] >= 0) & (ids[few] < e), weights[few], 0.0)
    by_pairs = plain.experts(xe[:20], torch.where(weight > 0, place[ids[few].clamp(0, e - 1).long()], 0), weight.double(), ue, de, "none")
    assert bool(((by_pairs - exact[:20]).abs() <= 1e-12 * bound[:20].max()).all())       # the oracle's own loop
