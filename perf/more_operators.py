"""Weights in 8-bit floating point and the products with them, as timed cases.

A case is one pass through one of four operators (``kind``):

* ``rows``: ``kernels.fp8_quantize`` rounds rows of numbers to 8 bits with a scale for every 128 numbers of a row, and
  ``kernels.fp8_read`` gives back the values that these stand for.
* ``linear``: ``kernels.linear_fp8``: rows are rounded so and multiplied with a matrix that is kept so.
* ``feedforward``: ``kernels.feedforward_fp8``: a gated feed-forward whose two products are of that kind; what lies between
  them is rounded to 8 bits, too.
* ``experts``: ``kernels.experts_fp8``: the same by routed experts: the (token, choice) pairs are sorted by expert, each goes
  through its expert's matrices, and a token's results come back, multiplied by their weights and added.

8 bits: e4m3 (a sign, four bits of exponent, three of mantissa, largest number 448) times 2^e, e being the least integer from
-127 on under which none of a block's 128 numbers is beyond 448 * 2^e; ties are rounded to even.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda:0"
F32 = torch.float32
F64 = torch.float64
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}
BLOCK = 128


# --- the cases ---------------------------------------------------------------------------------------------------------
def listed():
    two_b, nine_b, big = dict(width=2304, inter=9216), dict(width=3584, inter=14336), dict(width=4608, inter=36864)
    experts = dict(kind="experts", width=2048, inter=1024, experts=32, top=4, activation="silu")
    return [
        # a decode step's rows between two layers of the 2B model: the smallest call
        dict(kind="rows", name="rows-decode-8", rows=8, cols=two_b["width"], type="bfloat16", stride=0),
        # a long prompt's rows at the 27B width
        dict(kind="rows", name="rows-prompt-8192", rows=8192, cols=big["width"], type="bfloat16", stride=0),
        # float32 rows that are a slice of wider ones and end inside a block
        dict(kind="rows", name="rows-odd-float", rows=1111, cols=1000, type="float32", stride=1600),
        # one sequence decodes: the product after the activation at the 2B sizes
        dict(kind="linear", name="linear-decode-1", rows=1, k=two_b["inter"], n=two_b["width"], type="bfloat16"),
        # eight sequences decode: the same at the 27B sizes
        dict(kind="linear", name="linear-decode-8", rows=8, k=big["inter"], n=big["width"], type="bfloat16"),
        # a short prompt in float32, with sizes that are multiples of nothing
        dict(kind="linear", name="linear-odd-float", rows=99, k=1000, n=777, type="float32"),
        # queries, keys and values of a prompt at the 2B sizes
        dict(kind="linear", name="linear-prompt-2048", rows=2048, k=two_b["width"], n=4096, type="bfloat16"),
        # the product after the activation of a long prompt at the 9B sizes
        dict(kind="linear", name="linear-prompt-8192", rows=8192, k=nine_b["inter"], n=nine_b["width"], type="bfloat16"),
        # a layer's feed-forward while eight sequences decode, 2B sizes
        dict(two_b, kind="feedforward", name="feedforward-decode-8", rows=8, activation="gelu_tanh"),
        # ... and of a prompt, 27B sizes: the largest call
        dict(big, kind="feedforward", name="feedforward-prompt-4096", rows=4096, activation="gelu_tanh"),
        # eight sequences decode through routed experts: most experts have one token or none
        dict(experts, name="experts-decode-8", rows=8, skew=0.0),
        # a prompt whose tokens prefer some experts
        dict(experts, name="experts-prompt-2048", rows=2048, skew=0.7),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _size(rng, lo, hi):
    """A width: often a multiple of 128 or 16, at times of nothing."""
    n, to = _log(rng, lo, hi), rng.choice([128, 128, 64, 16, 8, 1])
    return max(lo, n // to * to)


def draw(rng: random.Random):
    kind = rng.choice(["rows", "linear", "linear", "feedforward", "experts"])
    rows = _log(rng, 1, 8192)
    if kind == "rows":
        cols = _size(rng, 32, 36864)
        rows = min(rows, max(1, 40_000_000 // cols))
        return dict(kind="rows", rows=rows, cols=cols, type=rng.choice(["bfloat16", "bfloat16", "float32"]),
                    stride=rng.choice([0, 0, cols + 8, cols + 24]))
    if kind == "linear":
        k, n = _size(rng, 64, 36864), _size(rng, 64, 36864)
        while n * k > 340_000_000:
            k, n = _size(rng, 64, 36864), _size(rng, 64, 36864)
        rows = min(rows, max(1, 1_000_000_000_000 // (n * k)))
        return dict(kind="linear", rows=rows, k=k, n=n, type=rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"]))
    if kind == "feedforward":
        width, inter = _size(rng, 256, 4608), _size(rng, 256, 36864)
        rows = min(rows, max(1, 500_000_000_000 // (3 * width * inter)))
        return dict(kind="feedforward", rows=rows, width=width, inter=inter, activation=rng.choice(["gelu_tanh", "silu"]))
    experts = rng.choice([4, 8, 16, 32, 64])
    width, inter = _size(rng, 256, 4096), _size(rng, 128, 2048)
    return dict(kind="experts", rows=min(rows, 4096), width=width, inter=inter, experts=experts, top=rng.randint(1, min(6, experts)),
                activation=rng.choice(["silu", "gelu_tanh", "relu2"]), skew=rng.choice([0.0, 0.3, 0.7]))


# --- inputs ------------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _activations(g, rows, cols, dtype, stride=0):
    """Rows as a layer meets them: columns of unequal sizes, some of them far larger than the others."""
    size = torch.exp(0.5 * torch.randn(cols, generator=g, device=DEV))
    size = torch.where(torch.rand(cols, generator=g, device=DEV) < 0.005, size * 20.0, size)
    x = (torch.randn(rows, cols, generator=g, device=DEV) * size).to(dtype)
    if not stride:
        return x
    wide = torch.zeros(rows, stride, dtype=dtype, device=DEV)
    wide[:, :cols] = x
    return wide[:, :cols]


def _matrix(g, *shape):
    """A layer's matrix in the type that a checkpoint has it in."""
    w = torch.randn(*shape, generator=g, device=DEV, dtype=torch.bfloat16)
    return w.mul_(0.5 * shape[-1] ** -0.5)


def prepare(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    state = {"case": case}
    if kind == "rows":
        state["x"] = _activations(g, case["rows"], case["cols"], TYPES[case["type"]], case["stride"])
        return state
    if kind == "linear":
        state["x"] = _activations(g, case["rows"], case["k"], TYPES[case["type"]])
        matrices = {"w": _matrix(g, case["n"], case["k"])}
    elif kind == "feedforward":
        W, I = case["width"], case["inter"]
        state["x"] = _activations(g, case["rows"], W, torch.bfloat16)
        matrices = {"gate": _matrix(g, I, W), "up": _matrix(g, I, W), "down": _matrix(g, W, I)}
    else:
        W, I, E, T = case["width"], case["inter"], case["experts"], case["rows"]
        state["x"] = _activations(g, T, W, torch.bfloat16)
        liking = case["skew"] * 3.0 * torch.randn(E, generator=g, device=DEV)
        z = torch.randn(T, E, generator=g, device=DEV) + liking
        best, ids = torch.topk(z, case["top"], dim=1)
        state["ids"], state["weights"] = ids.to(torch.int32).contiguous(), torch.softmax(best, dim=1).contiguous()
        matrices = {"up": _matrix(g, E, I, W), "down": _matrix(g, E, W, I)}
        if case["activation"] != "relu2":
            matrices["gate"] = _matrix(g, E, I, W)
    # a program keeps its matrices in 8 bits: as the framework lays them out, or as numbers and exponents
    if own:
        from brolm_b200 import kernels
        for name in matrices:
            if name not in ("gate", "up"):
                state[name] = kernels.fp8_quantize(matrices[name])
        if "gate" in matrices:
            state["gate_up"] = kernels.fp8_gate_up(matrices["gate"], matrices["up"])
        elif "up" in matrices:
            state["up"] = kernels.fp8_quantize(matrices["up"])
    else:
        for name, w in matrices.items():
            state[name] = _round8(w)
    return state


# --- a pass ------------------------------------------------------------------------------------------------------------
def _round8(x):
    """Numbers of 8 bits and a power of two for each block of 128 of the last axis (the last one may be shorter)."""
    cols = x.shape[-1]
    blocks = (cols + BLOCK - 1) // BLOCK
    x = torch.nn.functional.pad(x, (0, blocks * BLOCK - cols)).unflatten(-1, (blocks, BLOCK))
    # the least power of two under which the largest is not beyond 448: of 448 = 1.75 * 2^8
    mantissa, exponent = torch.frexp(x.abs().amax(dim=-1, keepdim=True).float())        # m * 2^e, m from 0.5 to 1
    exponent = (exponent - 9 + (mantissa > 0.875)).clamp_(min=-127)
    q = torch.ldexp(x.float(), -exponent).to(torch.float8_e4m3fn)
    return q, exponent, cols


def _values(q, exponent, cols):
    return torch.ldexp(q.float(), exponent).flatten(-2)[..., :cols]


def _act(z, name):
    if name == "relu2":
        return torch.relu(z).square()
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))


def _plain(s):
    case, kind = s["case"], s["case"]["kind"]
    x = _values(*_round8(s["x"]))
    if kind == "rows":
        return x.to(s["x"].dtype)
    if kind == "linear":
        return (x @ _values(*s["w"]).T).to(s["x"].dtype)
    if kind == "feedforward":
        h = _act(x @ _values(*s["gate"]).T, case["activation"]) * (x @ _values(*s["up"]).T)
        return (_values(*_round8(h)) @ _values(*s["down"]).T).to(s["x"].dtype)
    # the pairs in the order of their experts, an expert's rows padded to those of the most wanted one
    T, top, E = case["rows"], case["top"], case["experts"]
    expert, order = torch.sort(s["ids"].flatten().long(), stable=True)
    counts = (expert[:, None] == torch.arange(E, device=DEV)).sum(dim=0)
    place = torch.arange(T * top, device=DEV) - (counts.cumsum(0) - counts)[expert]
    token = torch.div(order, top, rounding_mode="floor")
    rows = torch.zeros(E, int(counts.max()), case["width"], dtype=F32, device=DEV)
    rows[expert, place] = x[token]
    up = rows @ _values(*s["up"]).mT
    if "gate" in s:
        h = _act(rows @ _values(*s["gate"]).mT, case["activation"]) * up
    else:
        h = _act(up, case["activation"])
    back = (_values(*_round8(h)) @ _values(*s["down"]).mT)[expert, place] * s["weights"].flatten()[order, None]
    pairs = torch.empty(T * top, case["width"], dtype=F32, device=DEV)
    pairs[order] = back
    return pairs.unflatten(0, (T, top)).sum(dim=1).to(s["x"].dtype)


def run(s):
    if not own:
        return _plain(s)
    from brolm_b200 import kernels
    case, kind, x = s["case"], s["case"]["kind"], s["x"]
    if kind == "rows":
        y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        kernels.fp8_read(kernels.fp8_quantize(x), y)
    elif kind == "linear":
        y = torch.empty((x.shape[0], case["n"]), dtype=x.dtype, device=x.device)
        kernels.linear_fp8(x, s["w"], y)
    elif kind == "feedforward":
        y = torch.empty((x.shape[0], case["width"]), dtype=x.dtype, device=x.device)
        kernels.feedforward_fp8(x, s["gate_up"], s["down"], y, case["activation"])
    else:
        y = torch.empty((x.shape[0], case["width"]), dtype=x.dtype, device=x.device)
        up = s["up"] if case["activation"] == "relu2" else s["gate_up"]
        kernels.experts_fp8(x, s["ids"], s["weights"], up, s["down"], y, case["activation"])
    return y


def work(case):
    kind, M = case["kind"], case["rows"]
    size = TYPES[case.get("type", "bfloat16")].itemsize
    held = lambda rows, cols: rows * (cols + (cols + BLOCK - 1) // BLOCK)       # bytes of a matrix in 8 bits
    if kind == "rows":
        n = M * case["cols"]
        return {"bytes": float(2 * n * size + 2 * held(M, case["cols"])), "flops": float(3 * n)}
    if kind == "linear":
        N, K = case["n"], case["k"]
        return {"bytes": float(held(N, K) + size * M * (K + N)), "flops": 2.0 * M * N * K}
    W, I = case["width"], case["inter"]
    mats = 2 if case["activation"] == "relu2" else 3
    if kind == "feedforward":
        return {"bytes": float(2 * held(I, W) + held(W, I) + 4 * M * W), "flops": 6.0 * M * W * I}
    pairs, E = M * case["top"], case["experts"]
    # experts that some token is expected to choose, were all equally likely
    chosen = E * (1.0 - (1.0 - case["top"] / E) ** M)
    return {"bytes": chosen * ((mats - 1) * held(I, W) + held(W, I)) + 4.0 * M * W + 8.0 * pairs, "flops": 2.0 * mats * pairs * W * I}


# --- in 64 bits --------------------------------------------------------------------------------------------------------
def _nearest8(x):
    """The values that a tensor's rows stand for in 8 bits, block by block, by dividing and rounding in 64 bits."""
    cols = x.shape[-1]
    blocks = -(-cols // BLOCK)
    u = torch.zeros(*x.shape[:-1], blocks * BLOCK, dtype=F64, device=DEV)
    u[..., :cols] = x
    u = u.view(*x.shape[:-1], blocks, BLOCK)
    most = u.abs().amax(dim=-1, keepdim=True).clamp_(min=448.0 * 2.0 ** -127)
    scale = torch.exp2(torch.ceil(torch.log2(most / 448.0)))
    # the logarithm may be a hair off where the largest is 448 * 2^e itself
    scale = torch.where(most > 448.0 * scale, scale * 2.0, torch.where(most <= 224.0 * scale, scale / 2.0, scale))
    scale.clamp_(min=2.0 ** -127)
    u /= scale
    # from 2^-6 on, eight steps to the next power of two
    size = torch.floor(torch.log2(u.abs().clamp(min=2.0 ** -6)))
    size = torch.where(torch.exp2(size + 1) <= u.abs(), size + 1, size)
    step = torch.exp2(torch.where(torch.exp2(size) > u.abs().clamp(min=2.0 ** -6), size - 1, size) - 3.0)
    return (torch.round(u / step) * step * scale).flatten(-2)[..., :cols]


def exact(case, seed):
    g = _generator(seed)
    kind = case["kind"]
    if kind == "rows":
        return _nearest8(_activations(g, case["rows"], case["cols"], TYPES[case["type"]], case["stride"]))
    if kind == "linear":
        x = _nearest8(_activations(g, case["rows"], case["k"], TYPES[case["type"]]))
        return x @ _nearest8(_matrix(g, case["n"], case["k"])).T
    W, I, name = case["width"], case["inter"], case["activation"]

    def act(z):
        if name == "relu2":
            return torch.where(z > 0, z * z, torch.zeros_like(z))
        k = z if name == "silu" else 2.0 * (2.0 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)
        return z * torch.sigmoid(k)
    if kind == "feedforward":
        x = _nearest8(_activations(g, case["rows"], W, torch.bfloat16))
        gate, up, down = _matrix(g, I, W), _matrix(g, I, W), _matrix(g, W, I)
        h = act(x @ _nearest8(gate).T)
        h *= x @ _nearest8(up).T
        return _nearest8(h) @ _nearest8(down).T
    E, T = case["experts"], case["rows"]
    s = prepare(case, seed)
    x, ids, weights = _nearest8(s["x"]), s["ids"], s["weights"].to(F64)
    del s
    _activations(g, T, W, torch.bfloat16)                      # the same numbers once more, up to the matrices
    torch.randn(E, generator=g, device=DEV)
    torch.randn(T, E, generator=g, device=DEV)
    up, down = _matrix(g, E, I, W), _matrix(g, E, W, I)
    gate = _matrix(g, E, I, W) if name != "relu2" else None
    out = torch.zeros(T, W, dtype=F64, device=DEV)
    for e in range(E):
        chose = ids == e
        token = chose.any(dim=1).nonzero()[:, 0]
        if not len(token):
            continue
        weight = (weights * chose).sum(dim=1)[token]
        h = x[token] @ _nearest8(up[e]).T
        h = act(h) if gate is None else act(x[token] @ _nearest8(gate[e]).T) * h
        out[token] += weight[:, None] * (_nearest8(h) @ _nearest8(down[e]).T)
    return out
