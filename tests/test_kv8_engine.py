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


@pytest.mark.parametrize("change,says", [
    (None, None), ("status", "too few free blocks"), ("held", "holds 3 pages on the device, 2 on the host"), ("count", "each once"),
    ("twice", "each once"), ("kv_len", "lengths"), ("positions", "positions"), ("padding", "positions"), ("rows", "group 1.*places"),
    ("spare", "group 0.*places")])
def test_what_the_device_made_of_a_step_against_the_hosts_counts(change, says):
    """The debug checks of such a cache, on tables that the plain restatement fills."""
    import numpy as np
    from brolm_b200.engine import debug
    from tests.plain import kv8_plain as plain
    c = Cache([KVSpec(1, 16, None), KVSpec(1, 16, 100)], 64 * 20, torch.bfloat16, "cpu", max_slots=4, int8=True, max_positions=640)
    slots = [c.alloc_slot() for _ in range(3)][::2]

    def step(old, new, tokens):
        c.reserve(dict(zip(slots, [a + n for a, n in zip(old, new)])))
        made = []
        for g in c.kv_groups:
            t = g.tables
            status, _, kv_len, pos, _, rows, tables, held, count = plain.extend(
                slots + [-1], old + [0], new + [1], t.tables.tolist(), t.held.tolist(), t.free.tolist(), int(t.free_count), 64, g.ring or 0, tokens)
            for x, y in ((t.tables, tables), (t.held, held), (t.free_count, [count]), (t.status, [status])):
                x.copy_(torch.tensor(y))
            made.append((np.array(kv_len), np.array(pos), np.array(rows)))
        return [made[0][0], made[0][1], [m[2] for m in made]]

    new_len = [300, 66]
    debug.check_tables(c, slots, [0, 0], new_len, *step([0, 0], new_len, 380))
    kv_len, positions, rows = step(new_len, [1, 1], 5)
    t = c.kv_groups[1].tables
    if change == "status":
        t.status.fill_(1)
    elif change == "held":
        t.held[slots[1]] += 1
    elif change == "count":
        t.free_count -= 1
    elif change == "twice":
        t.tables[slots[1], 0] = t.tables[slots[0], 0]
    elif change == "kv_len":
        kv_len[1] += 1
    elif change == "positions":
        positions[0] += 1
    elif change == "padding":
        positions[2] = 0
    elif change == "rows":
        rows[1][1] += 1
    elif change == "spare":
        rows[0][4] = 7
    args = (c, slots, new_len, [n + 1 for n in new_len], kv_len, positions, rows)
    if change is None:
        debug.check_tables(*args)
    else:
        with pytest.raises(debug.StepCheckError, match=says):
            debug.check_tables(*args)


def test_pages_that_the_kernels_do_not_take_are_refused_where_the_cache_is_made():
    spec = [KVSpec(1, 16, None)]
    with pytest.raises(CacheError, match="256 tokens"):
        Cache(spec, 640, torch.bfloat16, "cpu", page_size=320, int8=True)
    assert Cache(spec, 640, torch.bfloat16, "cpu", page_size=256, int8=True).page_size == 256
    assert Cache(spec, 640, torch.bfloat16, "cpu", page_size=320).page_size == 320
