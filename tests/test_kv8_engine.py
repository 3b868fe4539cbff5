"""What a cache in 8 bits refuses, and its bookkeeping, without a GPU."""
import pytest
import torch

import brolm_b200 as bb
from brolm_b200.cache import Cache, CacheError, KVSpec
from tests.helpers import TINY
from tests.papusun_helpers import CFG_S as PAPUSUN


def test_rings_have_room_for_the_page_that_is_being_filled():
    specs = [KVSpec(2, 16, None), KVSpec(2, 16, 100), KVSpec(2, 16, 64)]
    for piece, rings in ((1, (192, 128)), (30, (192, 192)), (65, (256, 192))):
        c = Cache(specs, 64 * 30, torch.bfloat16, "cpu", max_slots=3, int8=True, max_piece=piece, max_positions=1000)
        assert [g.ring for g in c.kv_groups] == [None, *rings]
        assert all(g.ring >= g.spec.window + piece + 64 - 2 for g in c.kv_groups[1:])
        assert [tuple(g.tables.tables.shape) for g in c.kv_groups] == [(3, 16), (3, rings[0] // 64), (3, rings[1] // 64)]
    plain = Cache(specs, 64 * 30, torch.bfloat16, "cpu", max_slots=3)
    assert [g.ring for g in plain.kv_groups] == [None, 128, 64]


def test_a_cache_in_8_bits_is_half_as_large():
    plain = Cache([KVSpec(4, 256, None)], 6400, torch.bfloat16, "cpu", max_slots=2)
    int8 = Cache([KVSpec(4, 256, None)], 6400, torch.bfloat16, "cpu", max_slots=2, int8=True)
    assert int8.kv_groups[0].k.dtype == int8.kv_groups[0].v.dtype == torch.int8
    assert int8.bytes() == plain.bytes() // 2 + 100 * 4 * 8


@pytest.mark.parametrize("spec", [KVSpec(1, 16, None, values=False), KVSpec(1, 16, None, v_dim=32), KVSpec(1, 16, None, chunk=64),
                                  KVSpec(1, 16, 64, keep_first=3)])
def test_layouts_that_8_bits_do_not_take(spec):
    with pytest.raises(CacheError, match="8 bits"):
        Cache([spec], 640, torch.bfloat16, "cpu", int8=True)


def test_counting_goes_on_as_it_was():
    c = Cache([KVSpec(1, 16, None), KVSpec(1, 16, 64)], 640, torch.bfloat16, "cpu", max_slots=2, int8=True)
    s = c.alloc_slot()
    c.reserve({s: 300})
    c.commit({s: 300})
    assert [len(g.pages[s]) for g in c.kv_groups] == [5, 2]
    with pytest.raises(CacheError):
        c.reserve({s: 700})
    c.free_slot(s)
    assert all(g.pool.free_pages == g.pool.num_pages for g in c.kv_groups)


def test_models_and_arguments_that_are_refused():
    model = bb.Model(bb.Gemma2Config(**TINY["A"][0]), dtype="float32", device="cpu")
    with pytest.raises(ValueError, match="cache_dtype"):
        model.new_cache(640, cache_dtype="int4")
    with pytest.raises(ValueError, match="max_piece"):
        model.new_cache(640, max_piece=4)
    with pytest.raises(CacheError, match="max_piece"):
        model.new_cache(640, cache_dtype="int8", max_piece=0)
    assert model.new_cache(640, cache_dtype="int8").int8 and not model.new_cache(640).int8
    other = bb.Model(bb.PapusunConfig.from_dict(PAPUSUN), dtype="float32", device="cpu")     # (delta rule, latent attention)
    with pytest.raises(ValueError, match="plain attention"):
        other.new_cache(640, cache_dtype="int8")



def test_limits_of_the_tables_are_said_before_a_step_is_begun():
    import os
    import re
    from brolm_b200.cache.cache import DeviceTables
    with open(os.path.join(os.path.dirname(__file__), "..", "brolm_b200", "csrc", "blocks.cu")) as fh:
        source = fh.read()
    assert [int(re.search(rf"MAX_{n} = (\d+)", source).group(1)) for n in ("ROWS", "SLOTS")] == [DeviceTables.MAX_ROWS, DeviceTables.MAX_SLOTS]
    spec = [KVSpec(1, 16, 32)]
    with pytest.raises(CacheError, match="65536 slots"):
        Cache(spec, 64, torch.bfloat16, "cpu", max_slots=65537, int8=True)
    assert Cache(spec, 64, torch.bfloat16, "cpu", max_slots=65537).max_slots == 65537
    assert Cache(spec, 64, torch.bfloat16, "cpu", max_slots=65536, int8=True).max_slots == 65536
    model = bb.Model(bb.Gemma2Config(**TINY["A"][0]), dtype="float32", device="cpu")
    e = bb.Engine(model, 64 * 4200, max_slots=4200, max_seq_len=64, cache_dtype="int8")
    slots = e.open(4097)
    free = [g.pool.free_pages for g in e.cache.kv_groups]
    with pytest.raises(bb.StepError, match="at most 4096"):
        e.step(slots, [[1]] * 4097)
    assert [g.pool.free_pages for g in e.cache.kv_groups] == free
