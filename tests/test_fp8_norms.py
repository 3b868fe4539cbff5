"""Gains of models with matrices in 8-bit floating point, wherever a checkpoint's tensors lie."""
import pytest
import torch

import brolm_b200 as bb
from brolm_b200.parts.norm import RMSNorm
from tests.helpers import TINY

DEV = "cuda:0"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gains_come_to_lie_on_borders_of_16_bytes(dtype):
    room = torch.randn(257).to(dtype)
    assert room.data_ptr() % 16 == 0
    for first in (0, 1):
        n = RMSNorm(256, 1e-6)
        n.bind({"weight": room[first:first + 256]})
        n.to_fp8()
        assert n.weight.data_ptr() % 16 == 0 and torch.equal(n.weight, room[first:first + 256])
        assert (n.weight.data_ptr() == room.data_ptr()) is (first == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_model_whose_gains_lie_one_behind_the_other(dtype):
    """Gains as views of one room, none on a border of 16 bytes: the same logits as from tensors of their own."""
    cfg, _, _ = TINY["B"]
    kind = getattr(torch, dtype)
    g = torch.Generator().manual_seed(3)
    expected = bb.Model(bb.Gemma2Config(**cfg), dtype=dtype, device=DEV).expected_tensors()
    tensors = {n: (torch.randn(tuple(e.shape), generator=g) * 0.05).to(kind).to(DEV) for n, e in expected.items()}
    gains = [n for n in expected if "norm" in n]
    room, views, at = torch.zeros(sum(tensors[n].numel() + 2 for n in gains), dtype=kind, device=DEV), dict(tensors), 1
    for n in gains:
        size = tensors[n].numel()
        views[n] = room[at:at + size]
        views[n].copy_(tensors[n])
        assert views[n].data_ptr() % 16
        at += size + (2 if (at + size + 1) * kind.itemsize % 16 == 0 else 1)
    outs = []
    for given in (tensors, views):
        engine = bb.Engine(bb.Model(bb.Gemma2Config(**cfg), dtype=dtype, device=DEV, weight_dtype="fp8").load_weights(given), max_tokens=256)
        slots = engine.open(1)
        outs.append(torch.cat([engine.step(slots, [[5, 9, 2, 7]]).clone(), engine.step(slots, [[4]]).clone()]))
    assert torch.equal(outs[0], outs[1]) and outs[0].isfinite().all()
