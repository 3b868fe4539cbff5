"""The rings of the tcgen05 attention over the 8-bit cache (csrc/attn_kv8_tc.cu), as a model on the CPU.

A wait on an mbarrier tells a slot's uses apart by their parity alone: it passes when the phase before the current one has
the parity that is asked for, also where that phase is two uses too early.  The model runs the kernel's roles (two loading
warps, two groups of converting warps, the thread that issues the products) in random order, with loads that are now and then
very late, and looks at what every role finds where its wait has let it through.  The numbers of slots are those of the
kernel's source."""
import os
import random
import re

import pytest

SOURCE = os.path.join(os.path.dirname(__file__), "..", "brolm_b200", "csrc", "attn_kv8_tc.cu")


def constants():
    with open(SOURCE) as fh:
        text = fh.read()
    raws = int(re.search(r"KIND_RAWS = (\d+)", text).group(1))
    groups = int(re.search(r"CONVERT_GROUPS = (\d+)", text).group(1))
    a, b, c = map(int, re.search(r"SLOTS = HD == 256 \? (\d+) : HD == 128 \? (\d+) : (\d+);", text).groups())
    return raws, groups, {256: a, 128: b, 64: c}


class Bar:
    def __init__(self):
        self.phase = 0

    def arrive(self):
        self.phase += 1

    def passes(self, parity):
        return (self.phase - 1) & 1 == parity


def run(head, slots, raws, groups, tiles, seed, shared=0):
    """What went wrong, or None.  ``shared``: one ring of so many raw slots for keys and values, instead of one each."""
    rng = random.Random(seed)
    parts = head // 64
    raw_full, raw_empty = ([Bar() for _ in range(shared or 2 * raws)] for _ in range(2))
    unit_full, unit_empty = ([Bar() for _ in range(slots)] for _ in range(2))
    raw, unit, coming, wrong, now = {}, {}, [], [], 0

    def place(kind, t, p):                           # in the order of the products
        return ((0 if t == 0 else 2 * t - 1) if kind == "k" else min(2 * t + 2, 2 * tiles - 1)) * parts + p

    def raw_place(kind, t, p):                       # (slot, use)
        if shared:
            u = place(kind, t, p)
            return u % shared, u // shared
        i = t * parts + p
        return (0 if kind == "k" else raws) + i % raws, i // raws

    def load(kind):
        for t in range(tiles):
            for p in range(parts):
                s, use = raw_place(kind, t, p)
                while not raw_empty[s].passes((use & 1) ^ 1):
                    yield
                if raw_empty[s].phase < use:
                    wrong.append(("loaded over", kind, t, p))
                coming.append((now + (rng.choice([20, 400]) if rng.random() < 0.1 else 8), s, (kind, t, p)))
                yield

    def convert(group):
        order = [(kind, t, p) for j in range(-1, tiles) for kind, t in (("k", j + 1), ("v", j)) if 0 <= t < tiles for p in range(parts)
                 if (p % groups if parts > 1 else "kv".index(kind)) == group]
        for kind, t, p in order:
            s, use = raw_place(kind, t, p)
            while not raw_full[s].passes(use & 1):
                yield
            if raw.get(s) != (kind, t, p):
                wrong.append(("read", kind, t, p, raw.get(s)))
            for _ in range(30 if rng.random() < 0.05 else 1):
                yield
            u = place(kind, t, p)
            while not unit_empty[u % slots].passes((u // slots & 1) ^ 1):
                yield
            if unit_empty[u % slots].phase < u // slots:
                wrong.append(("stored over", kind, t, p))
            unit[u % slots] = (kind, t, p)
            yield
            raw_empty[s].arrive()
            unit_full[u % slots].arrive()

    def issue():
        order = [("k", 0)] + [x for j in range(tiles) for x in ((("k", j + 1),) if j + 1 < tiles else ()) + (("v", j),)]
        for u, (kind, t, p) in enumerate((kind, t, p) for kind, t in order for p in range(parts)):
            while not unit_full[u % slots].passes(u // slots & 1):
                yield
            if unit.get(u % slots) != (kind, t, p):
                wrong.append(("multiplied", kind, t, p, unit.get(u % slots)))
            yield
            unit_empty[u % slots].arrive()

    roles = [load("k"), load("v"), issue()] + [convert(g) for g in range(groups)]
    while roles and not wrong and now < 100_000:
        now += 1
        for x in [x for x in coming if x[0] <= now]:
            coming.remove(x)
            raw[x[1]] = x[2]
            raw_full[x[1]].arrive()
        role = rng.choice(roles)
        try:
            next(role)
        except StopIteration:
            roles.remove(role)
    return wrong[0] if wrong else ("stuck",) if roles else None


@pytest.mark.parametrize("head,tiles", [(64, 40), (64, 1), (128, 24), (128, 2), (256, 12), (256, 1)])
def test_nobody_passes_a_wait_too_early(head, tiles):
    raws, groups, slots = constants()
    assert [r for r in (run(head, slots[head], raws, groups, tiles, seed) for seed in range(60)) if r] == []


def test_the_model_sees_what_a_ring_of_seven_for_both_would_do():
    raws, groups, _ = constants()
    for head, tiles in ((64, 40), (128, 24)):
        assert any(run(head, 8, raws, groups, tiles, seed, shared=7) for seed in range(60))
