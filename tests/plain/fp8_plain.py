"""Rows in 8-bit floating point and the products with them, in 64 bits: numbers one by one, blocks as a loop."""
from __future__ import annotations

import math

import torch

BLOCK = 128
# what e4m3 has: zeros, subnormal and normal numbers, no infinity
E4M3 = sorted({m * 2.0 ** -9 for m in range(8)} | {(1 + m / 8) * 2.0 ** e for e in range(-6, 9) for m in range(8) if (e, m) != (8, 7)})


def scale_of(most: float) -> float:
    """The least power of two from 2^-127 on with most <= 448 * it."""
    if not math.isfinite(most):
        return math.nan
    e = -127
    while most > 448.0 * 2.0 ** e:
        e += 1
    return 2.0 ** e


def nearest(u: torch.Tensor) -> torch.Tensor:
    """u (|u| <= 448) to the nearest number of e4m3, a tie to the one with an even mantissa (every second of the list)."""
    table = torch.tensor(E4M3, dtype=torch.float64, device=u.device)
    a = u.abs().double().contiguous()
    hi = torch.searchsorted(table, a).clamp_(max=len(E4M3) - 1)
    lo = torch.where(table[hi] > a, hi - 1, hi)
    down, up = a - table[lo], table[hi] - a
    pick = torch.where(down < up, lo, torch.where(up < down, hi, torch.where(lo % 2 == 0, lo, hi)))
    return torch.copysign(table[pick], u.double())


def values(x: torch.Tensor) -> torch.Tensor:
    """What the rows of x stand for in 8 bits, in 64 bits."""
    out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
    flat, res = x.double().reshape(-1, x.shape[-1]), out.view(-1, x.shape[-1])
    for a in range(0, x.shape[-1], BLOCK):
        piece = flat[:, a:a + BLOCK]
        scale = torch.tensor([scale_of(float(m)) for m in piece.abs().amax(dim=1).cpu()], dtype=torch.float64, device=x.device)[:, None]
        # a sum over the block: NaN if one of it is not finite
        bad = ~torch.isfinite(piece).all(dim=1, keepdim=True)
        safe = torch.where(bad, torch.ones_like(scale), scale)
        q = nearest(torch.where(bad, torch.zeros_like(piece), piece / safe)) * safe
        res[:, a:a + BLOCK] = torch.where(bad, torch.full_like(q, math.nan), q)
    return out


def act(z: torch.Tensor, name: str, limit: float = 0.0):
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "relu2":
        return z.clamp(min=0) ** 2
    if name == "none":
        return z
    return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)))


def gated(gate: torch.Tensor, up: torch.Tensor, name: str, limit: float = 0.0) -> torch.Tensor:
    if name == "clamped_gate":
        g, u = gate.clamp(max=limit), up.clamp(-limit, limit)
        return g * torch.sigmoid(1.702 * g) * (u + 1.0)
    return act(gate, name) * up


def experts(x, ids, weights, up, down, name, gate=None, scale_input=False, limit=0.0):
    """x, up, down, gate: values in 64 bits.  Every pair by itself; choices that are no expert's give nothing.  With
    ``scale_input`` the weight multiplies the pair's first sums and not its result.  Also returns how large a row's terms are."""
    out = torch.zeros(x.shape[0], down.shape[1], dtype=torch.float64, device=x.device)
    for t in range(x.shape[0]):
        for c in range(ids.shape[1]):
            e = int(ids[t, c])
            if not 0 <= e < up.shape[0]:
                continue
            w = float(weights[t, c])
            s = w if scale_input else 1.0
            h = (x[t] @ up[e].T) * s
            h = act(h, name) if gate is None else gated((x[t] @ gate[e].T) * s, h, name, limit)
            out[t] += (1.0 if scale_input else w) * (values(h[None])[0] @ down[e].T)
    return out
