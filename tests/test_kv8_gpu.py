"""The 8-bit cache on the device against the plain restatement in 64 bits."""
import math
import random

import pytest
import torch

from brolm_b200 import kernels
from tests.plain import kv8_plain as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
I32 = torch.int32
NAN, INF = math.nan, math.inf


def ints(v):
    return torch.tensor(list(v), dtype=I32, device=DEV)


def same(a, b):
    """Equal numbers, NaN equal to NaN."""
    return a.shape == b.shape and bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


# --- tables ------------------------------------------------------------------------------------------------------------
class Tables:
    """The device's tables beside the plain ones; every step and every release is compared."""

    def __init__(self, S, W, N, block, ring, seed):
        self.block, self.ring = block, ring
        self.order = list(range(N))
        random.Random(seed).shuffle(self.order)
        self.free, self.count = list(self.order), N
        self.tables, self.held = [[0] * W for _ in range(S)], [0] * S
        self.dev = dict(tables=torch.zeros((S, W), dtype=I32, device=DEV), held=ints([0] * S), free=ints(self.free),
                        free_count=ints([N]))

    def step(self, slots, lengths, new, tokens):
        out = dict(cu_q=ints([7] * (len(slots) + 1)), kv_len=ints([7] * len(slots)), positions=ints([7] * tokens),
                   tok_seq=ints([7] * tokens), cache_rows=ints([7] * tokens), status=ints([7]))
        kernels.blocks_extend(ints(slots), ints(lengths), ints(new), *self.dev.values(), block=self.block, ring=self.ring, **out)
        want = plain.extend(slots, lengths, new, self.tables, self.held, self.free, self.count, self.block, self.ring, tokens)
        status, cu, kv_len, positions, seqs, rows, self.tables, self.held, self.count = want
        assert out["status"].tolist() == [status]
        for name, values in (("cu_q", cu), ("kv_len", kv_len), ("positions", positions), ("tok_seq", seqs), ("cache_rows", rows)):
            assert out[name].tolist() == values, name
        self.check()
        return status

    def release(self, slots):
        status = ints([7])
        kernels.blocks_release(ints(slots), *self.dev.values(), status=status)
        live = [s for s in slots if s != -1]
        bad = any(not 0 <= s < len(self.held) for s in live) or len(set(live)) != len(live)
        if not bad:
            for s in reversed(live):
                while self.held[s]:
                    self.held[s] -= 1
                    self.free[self.count] = self.tables[s][self.held[s]]
                    self.count += 1
        assert status.tolist() == [4 if bad else 0]
        self.check()

    def check(self):
        assert self.dev["tables"].tolist() == self.tables and self.dev["held"].tolist() == self.held
        assert self.dev["free_count"].tolist() == [self.count] and self.dev["free"].tolist() == self.free


@pytest.mark.parametrize("block,ring,S,W,N", [(32, 0, 5, 4, 17), (64, 192, 40, 3, 90), (128, 0, 200, 9, 900), (32, 32, 3, 1, 3)])
def test_tables_over_many_steps(block, ring, S, W, N):
    rng = random.Random(block + S)
    t = Tables(S, W, N, block, ring, S)
    lengths = [0] * S
    seen = set()
    for turn in range(25):
        slots = rng.sample(range(S), rng.randint(1, S))
        slots = [s if rng.random() < 0.9 else -1 for s in slots]
        new = [rng.choice([0, 1, 1, 1, rng.randint(0, 3 * block)]) for _ in slots]
        before = [lengths[s] if s >= 0 else rng.randint(-5, 5) for s in slots]
        tokens = max(0, sum(new) + rng.choice([0, 0, 1, 40, -1]))
        status = t.step(slots, before, new, tokens)
        seen.add(status)
        if status == 0:
            for s, n in zip(slots, new):
                if s >= 0:
                    lengths[s] += n
        if rng.random() < 0.4:
            gone = rng.sample(range(S), rng.randint(1, S)) + [-1]
            t.release(gone)
            for s in gone[:-1]:
                lengths[s] = 0
    assert 0 in seen and len(seen) > 1


def test_tables_of_many_rows_and_tokens():
    n, S = 2500, 3000
    rng = random.Random(1)
    t = Tables(S, 4, 6000, 32, 128, 3)
    slots = rng.sample(range(S), n)
    new = [rng.choice([1, 2, 31, 32, 33, 64, 300]) for _ in slots]
    free = list(t.free)
    if t.step(slots, [0] * n, new, sum(new)) != 0:
        new = [1] * n
        assert t.step(slots, [0] * n, new, n) == 0
    t.release(slots)
    assert t.free == free                          # the stack is as it was


def test_tables_of_a_step_that_all_sms_share():
    """Long prompts and short ones, padding between them, 40,000 tokens and more; once refused, once taken, once again."""
    new = [15000, 1, 0, 300, 20000, 64, 7000, 33]
    slots = [4, 0, 9, -1, 2, 7, 1, 5]
    t = Tables(12, 400, 850, 64, 0, 5)
    assert t.step(slots, [0] * 8, [700 * 64] + new[1:], 80000) == 2
    assert t.step(slots, [0] * 8, [390 * 64, 1, 0, 300, 390 * 64] + new[5:], 80000) == 1
    for _ in range(2):
        assert t.step(slots, [0] * 8, new, sum(new) + 100) == 0
    assert t.step([2, 4], [20000, 15000], [500, 24500], 40000) == 2
    assert t.step([2, 4], [20000, 15000], [500, 9000], 40000) == 0
    t.release(slots)
    r = Tables(6, 20, 100, 64, 1280, 6)
    assert r.step([3, 1, 0], [0, 100, 0], [30000, 10000, 1], 40001) == 0


@pytest.mark.parametrize("slots,lengths,new,tokens,status", [
    ([0, 1, 0], [0, 0, 0], [1, 1, 1], 3, 4), ([0, 9], [0, 0], [1, 1], 2, 4), ([0, -2], [0, 0], [1, 1], 2, 4),
    ([0, 1], [0, -1], [1, 1], 2, 4), ([0, 1], [0, 0], [1, -1], 2, 4), ([0, 1], [0, 0], [3, 4], 6, 3),
    ([0], [0], [97], 200, 2), ([0, 1, 2], [0, 0, 0], [96, 64, 65], 300, 1), ([0], [2 ** 31 - 5], [20], 30, 4),
    ([0, 1], [0, 0], [2 ** 31 - 1, 2 ** 31 - 1], 4, 3), ([0], [0], [0], 0, 0), ([], [], [], 5, 0)])
def test_steps_that_do_not_fit_change_nothing(slots, lengths, new, tokens, status):
    t = Tables(4, 3, 7, 32, 0, 0)
    t.step([3], [0], [10], 10)
    if max(new, default=0) > 2 ** 30 or max(lengths, default=0) > 2 ** 30:          # (too long for the plain lists)
        out = dict(cu_q=ints([7] * (len(slots) + 1)), kv_len=ints([7] * len(slots)), positions=ints([7] * tokens),
                   tok_seq=ints([7] * tokens), cache_rows=ints([7] * tokens), status=ints([7]))
        kernels.blocks_extend(ints(slots), ints(lengths), ints(new), *t.dev.values(), block=32, **out)
        t.check()
        assert int(out["status"]) >= 2 and out["positions"].tolist() == [-1] * tokens and not out["cu_q"].any()
    else:
        assert t.step(slots, lengths, new, tokens) == status
    t.release([0, 0])
    t.release([4])
    t.release([])


def test_the_same_step_again_takes_no_more_blocks():
    t = Tables(4, 8, 12, 32, 0, 0)
    for _ in range(3):
        assert t.step([2, 0], [33, 0], [40, 5], 50) == 0
    assert t.count == 12 - 3 - 1


# --- blocks ------------------------------------------------------------------------------------------------------------
class Cached:
    """Device blocks full of garbage beside plain ones, sequences with blocks in no order."""

    def __init__(self, B, W, G, P, D, ring=0, seed=0, spare=2):
        self.P, self.ring, self.G, self.D = P, ring, G, D
        n = B * W + spare
        g = torch.Generator().manual_seed(seed)
        self.table = torch.randperm(n, generator=g)[:B * W].view(B, W)
        self.pages = [torch.randint(-127, 128, (n, G, P, D), generator=g, dtype=torch.int8) for _ in range(2)]
        self.scales = [torch.full((n, G), NAN) for _ in range(2)]                 # (blocks that nobody began)
        self.dev = [p.to(DEV) for p in self.pages] + [s.to(DEV) for s in self.scales]
        self.pages = [p.double() for p in self.pages]
        self.scales = [s.double() for s in self.scales]
        self.tables = self.table.to(I32).to(DEV)
        self.lens = [0] * B

    def places(self, i, n):
        """Cache rows of the next n tokens of sequence i."""
        first = plain.first_kept(self.lens[i] + n, self.P, self.ring)
        out = []
        for p in range(self.lens[i], self.lens[i] + n):
            place = p % self.ring if self.ring else p
            out.append(int(self.table[i, place // self.P]) * self.P + place % self.P if p >= first else -1)
        return out

    def write(self, rows, new, k, v, bound=None):
        """k, v on the device; both sides."""
        at = [self.places(i, n) if i >= 0 else [-1] * n for i, n in zip(rows, new)]
        pos = [list(range(self.lens[i], self.lens[i] + n)) if i >= 0 else [-1] * n for i, n in zip(rows, new)]
        cu = [0]
        for n in new:
            cu.append(cu[-1] + n)
        kernels.kv8_write(k, v, ints(cu), ints(sum(pos, [])), ints(sum(at, [])), *self.dev, max_q_len=bound or max(new))
        for i, n in zip(rows, new):
            if i >= 0:
                self.lens[i] += n
        for x, pages, scales in zip((k, v), self.pages, self.scales):
            plain.write(x.cpu(), sum(at, []), pages, scales)

    def check(self):
        for d, p in zip(self.dev[2:], self.scales):
            assert same(d.cpu().double(), p)
        for d, p, s in zip(self.dev[:2], self.pages, self.scales):
            fine = ~torch.isnan(s)[:, :, None, None]
            assert bool(((d.cpu().double() == p) | ~fine).all())

    def values(self, which, i):
        """(first position, [n, G, D]) of all that sequence i still holds."""
        first = plain.first_kept(self.lens[i], self.P, self.ring)
        return first, plain.read(self.pages[which], self.scales[which], self.table[i], range(first, self.lens[i]), self.ring)


def rows_of(T, G, D, dtype, g, spread=2.0):
    x = torch.randn((T, G, D), generator=g) * torch.exp2(spread * torch.randn((T, 1, 1), generator=g))
    return x.to(dtype).to(DEV)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("G,P,D,ring", [(1, 32, 16, 0), (2, 64, 256, 0), (3, 128, 80, 0), (2, 32, 96, 96), (1, 256, 256, 0),
                                        (5, 64, 48, 64)])
def test_blocks_written_piece_by_piece(dtype, G, P, D, ring):
    B, W = 4, (ring // P if ring else max(2, 640 // P))
    c = Cached(B, W, G, P, D, ring, seed=D)
    g = torch.Generator().manual_seed(P + D)
    rng = random.Random(D)
    for turn in range(14):
        rows = rng.sample(range(B), rng.randint(1, B))
        room = [(10 ** 6 if ring else W * P) - c.lens[i] for i in rows]
        new = [min(r, rng.choice([0, 1, 1, 2, 7, P - 1, P, P + 1, 2 * P + 5])) for r in room]
        if turn % 3 == 2:
            new = [min(1, n) for n in new]
        if sum(new) == 0:
            continue
        k, v = (rows_of(sum(new), G, D, dtype, g) for _ in range(2))
        c.write(rows, new, k, v)
        c.check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_write_takes_rows_of_any_stride(dtype):
    """Parts of a fused projection, heads apart from each other, rows that begin off 16 bytes."""
    c = Cached(2, 3, 3, 32, 32, seed=1)
    g = torch.Generator().manual_seed(3)
    for cut in (0, 1, 5, 8):
        wide = rows_of(30, 8, 70, dtype, g)
        k, v = wide[:, 1:7:2, cut:cut + 32], wide[:, 2:8:2, 33:65]
        c.write([0, 1], [29, 1], k, v)
        c.write([1], [1], wide.reshape(30, -1)[3:4, 1:97].view(1, 3, 32), wide.reshape(30, -1)[5:6, 8:104].view(1, 3, 32))
        c.check()
        if c.lens[0] > 60:
            break


def test_write_at_the_ends_of_the_range():
    """Zeros, the largest and the smallest numbers, the limits of a scale, and halves between two steps."""
    rows = [0.0, 3.3895e38, 1e-45, 2.0 ** -127, 127 * 2.0 ** -126, 127.0, 127.00001, 254.0, 126.5, 0.5]
    c = Cached(len(rows), 1, 1, 32, 16, seed=2)
    for step in range(3):
        x = torch.zeros((len(rows), 1, 16))
        for i, r in enumerate(rows):
            x[i, 0, :5] = torch.tensor([r, -r, r / 2, r / 254, -r / 508])
            if step == 1:
                x[i] *= 0.01
        k = x.to(DEV)
        c.write(list(range(len(rows))), [1] * len(rows), k, -k)
        c.check()


@pytest.mark.parametrize("value", [NAN, INF, -INF])
def test_a_block_that_gets_a_number_that_is_not_finite(value):
    c = Cached(2, 4, 2, 32, 32, seed=4)
    g = torch.Generator().manual_seed(9)
    for new, where in (([40, 3], None), ([1, 1], (0, 1, 7)), ([1, 1], None), ([30, 30], None), ([5, 5], (1, 0, 0))):
        k, v = (rows_of(sum(new), 2, 32, torch.float32, g) for _ in range(2))
        if where:
            k[where] = value
        c.write([0, 1], new, k, v)
        c.check()
    assert torch.isnan(c.dev[2]).sum() >= 2 + 2       # this block, and at least the two that nobody began
    k, v = torch.empty((2, 75, 2, 32), device=DEV)
    kernels.kv8_read(ints([0, 75]), ints([77]), ints([0]), c.tables, *c.dev, k, v, max_q_len=75)
    want = c.values(0, 0)[1][2:]
    assert same(k.cpu().double(), want) and torch.isnan(want).any() and not torch.isnan(want).all()
    assert same(v.cpu().double(), c.values(1, 0)[1][2:])


def test_write_of_padding_and_wrong_places_writes_nothing():
    c = Cached(1, 2, 1, 32, 16)
    before = [d.clone() for d in c.dev]
    k = torch.ones((4, 1, 16), device=DEV)
    n = c.pages[0].shape[0]
    for bound in (1, 4):
        for cu, pos, at in (([0, 1, 2, 3, 4], [-1] * 4, [-1] * 4), ([0, 1, 2, 3, 4], [0] * 4, [-1, n * 32, 2 ** 31 - 1, -7]),
                            ([0, 0, 0, 0, 0], [0] * 4, [0] * 4)):
            kernels.kv8_write(k, k, ints(cu), ints(pos), ints(at), *c.dev, max_q_len=bound)
    assert all(same(a, b) for a, b in zip(before, c.dev))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ring", [0, 96])
def test_read_gives_back_what_is_held(dtype, ring):
    c = Cached(3, 3 if ring else 9, 2, 32, 48, ring, seed=5)
    g = torch.Generator().manual_seed(1)
    for new in ([1, 70, 33], [200, 1, 64]):
        c.write([0, 1, 2], new, rows_of(sum(new), 2, 48, dtype, g), rows_of(sum(new), 2, 48, dtype, g))
    asked = [201, 0, 98]                                       # 201 and 97 are held: one more reads as zero
    cu = ints([0, 201, 201, 299])
    wide = torch.full((300, 4, 64), 5.0, dtype=dtype, device=DEV)
    k, v = wide[:, ::2, :48], wide[:, 1::2, 16:]
    kernels.kv8_read(cu, ints(c.lens), ints([0, 1, 2]), c.tables, *c.dev, k[:299], v[:299], ring=ring, max_q_len=201)
    for which, got in ((0, k), (1, v)):
        at = 0
        for i, n in enumerate(asked):
            first, held = c.values(which, i)
            lead = torch.zeros((max(0, n - len(held)), 2, 48), dtype=torch.float64)
            want = torch.cat([lead, held[max(0, len(held) - n):]]) if n else lead[:0]
            assert same(got[at:at + n].cpu().double(), want.to(dtype).double())
            at += n
    assert bool((wide[299] == 5.0).all()) and bool((wide[:, ::2, 48:] == 5.0).all())


# --- attention ---------------------------------------------------------------------------------------------------------
def bound(dtype, ref, q, keys, values, scale):
    """How far a row may be from 64 bits.  Scores: products and sums in 32 bits, D of them, and an exponential of relative
    error below 2^-21, on scores of up to z = scale sum |q k|: 2^-21 (2 + z).  bfloat16 rounds the weights to 11 bits or
    more (2^-11 of the largest value; they sum to one) and the result to 8 (2^-8 with a margin for a result at the edge)."""
    z = scale * float((q.double().abs().amax() * keys.abs().sum(dim=2).amax())) if len(keys) else 0.0
    most = float(values.abs().max()) if len(values) else 0.0
    if dtype == torch.float32:
        return most * 2.0 ** -21 * (2.0 + z) + 2.0 ** -22 * ref.abs()
    return most * (2.0 ** -21 * (2.0 + z) + 2.0 ** -11) + 2.0 ** -8 * ref.abs()


def compare(c, dtype, rows, new, group, scale, cap, window, seed=0, q_spread=1.0, max_kv_len=None, q=None):
    """The newest tokens of the sequences ``rows`` (-1: a padding row) through the kernel and in 64 bits."""
    H = c.G * group
    g = torch.Generator().manual_seed(seed)
    T = sum(new)
    if q is None:
        wide = (torch.randn((T, H * c.D + 64), generator=g) * q_spread).to(dtype).to(DEV)
        q = wide[:, 32:32 + H * c.D]
    out = torch.full((T, H * c.D + 32), 9.0, dtype=dtype, device=DEV)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    lens = [c.lens[i] if i >= 0 else 0 for i in rows]
    kernels.attention_kv8(q, out[:, :H * c.D], ints(cu), ints(lens), ints(rows), c.tables, *c.dev, n_kv=c.G, group=group,
                          head_dim=c.D, scale=scale, cap=cap, window=window, ring=c.ring, batch=len(rows), max_q_len=max(new),
                          max_kv_len=max_kv_len or max(1, max(lens)))
    got = out[:, :H * c.D].cpu().double().view(T, H, c.D)
    assert bool((out[:, H * c.D:] == 9.0).all())
    qh = q.cpu().view(T, H, c.D)
    for r, i in enumerate(rows):
        first, keys = c.values(0, i) if i >= 0 else (0, torch.zeros((0, c.G, c.D), dtype=torch.float64))
        _, values = c.values(1, i) if i >= 0 else (0, keys)
        for j in range(new[r]):
            t = cu[r] + j
            ref = plain.attend(qh[t], keys, values, first, lens[r] - new[r] + j, scale, cap, window)
            assert bool((torch.isnan(ref) == torch.isnan(got[t])).all()), (r, j)
            fine = lambda x: torch.nan_to_num(x, nan=0.0)
            off = fine(got[t] - ref).abs() - bound(dtype, fine(ref), fine(qh[t].double()), fine(keys), fine(values), scale)
            assert float(off.max()) <= 0.0, (r, j, float(off.max()))
    return got


def filled(B, W, G, P, D, lens, ring=0, seed=0, dtype=torch.float32, spread=0.5):
    c = Cached(B, W, G, P, D, ring, seed)
    g = torch.Generator().manual_seed(seed + 1)
    c.write(list(range(B)), lens, rows_of(sum(lens), G, D, dtype, g, spread), rows_of(sum(lens), G, D, dtype, g, spread))
    return c


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,G,group,P", [(16, 2, 2, 32), (32, 1, 6, 64), (64, 2, 1, 64), (80, 2, 3, 32), (96, 1, 8, 128), (128, 2, 4, 64),
                                         (192, 1, 16, 32), (256, 4, 2, 64), (256, 1, 9, 256)])
def test_attention_of_one_token(dtype, D, G, group, P):
    lens = [1, 2, 31, 33, 64, 65, 200, 127]
    c = filled(len(lens), -(-256 // P), G, P, D, lens, seed=D + group)
    compare(c, dtype, [3, 0, -1, 6, 1, 2, 7, 4, 5], [1] * 9, group, D ** -0.5, 0.0, 0, q_spread=2.0)
    compare(c, dtype, list(range(8)), [1] * 8, group, D ** -0.5, 20.0, 0, q_spread=4.0)


@pytest.fixture(params=[False, True], ids=["mma", "tcgen05"])
def either(request, monkeypatch):
    """Steps of many rows on mma.sync, and on tcgen05 where it takes their sizes."""
    monkeypatch.setattr(kernels.kv8, "KV8_TC_WORK", 0.0 if request.param else math.inf)


@pytest.fixture
def on_tcgen05(monkeypatch):
    monkeypatch.setattr(kernels.kv8, "KV8_TC_WORK", 0.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,G,group,P", [(64, 2, 2, 64), (128, 1, 4, 32), (256, 2, 2, 64), (256, 1, 16, 64), (80, 1, 3, 32), (64, 1, 128, 32)])
@pytest.mark.parametrize("window", [0, 1, 50])
def test_attention_of_several_tokens(dtype, D, G, group, P, window, either):
    lens = [3, 70, 140, 1, 257]
    c = filled(len(lens), -(-288 // P), G, P, D, lens, seed=D + window)
    for new in ([3, 1, 5, 1, 2], [3, 70, 40, 1, 131]):
        compare(c, dtype, list(range(5)), new, group, D ** -0.5, 30.0 if window else 0.0, window, seed=sum(new))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 4, 67])
def test_attention_over_a_ring(dtype, new, either):
    P, window = 32, 41
    ring = (window + new + P - 2 + P - 1) // P * P
    c = filled(3, ring // P, 2, P, 64, [1, 33, 90], ring=ring, seed=new)
    g = torch.Generator().manual_seed(8)
    for _ in range(4):
        c.write([0, 1, 2], [new] * 3, rows_of(3 * new, 2, 64, dtype, g), rows_of(3 * new, 2, 64, dtype, g))
        compare(c, dtype, [2, 0, 1], [new] * 3, 2, 0.125, 0.0, window, seed=c.lens[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_attention_over_long_sequences_is_split_and_joined(dtype):
    c = filled(3, 48, 1, 64, 64, [3000, 5, 1500], seed=11)
    for bound_ in (3000, 3072, 100000):
        compare(c, dtype, [0, 1, 2], [1, 1, 1], 2, 0.125, 0.0, 0, max_kv_len=bound_)
    compare(c, dtype, [0], [1], 2, 0.125, 0.0, 0)
    compare(c, dtype, [0, 2], [1, 1], 2, 0.125, 0.0, 900)
    compare(c, dtype, [0, 2], [6, 3], 2, 0.125, 50.0, 0)


@pytest.fixture(params=[(1, -9), (1, -50), (2, -17), (8, -30)], ids=str)
def dealt(request, monkeypatch):
    """Clusters dealt out over the sequences by their lengths: as few as sequences, and more than they have tiles for."""
    monkeypatch.setattr(kernels.kv8, "KV8_TC_WORK", math.inf)
    monkeypatch.setattr(kernels.kv8, "kv8_shares", lambda *a: request.param)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,G,group", [(64, 2, 2), (256, 1, 5), (80, 1, 3)])
@pytest.mark.parametrize("window", [0, 300])
def test_attention_dealt_out_by_length(dtype, D, G, group, window, dealt):
    lens = [3, 900, 140, 1, 257, 64, 500]
    c = filled(len(lens), 15, G, 64, D, lens, seed=D + window)
    cap = 30.0 if window else 0.0
    compare(c, dtype, [4, -1, 0, 6, 1, 3, 2, 5, -1], [1] * 9, group, D ** -0.5, cap, window)
    compare(c, dtype, [1, 3, 5, 0, 2, -1, 6], [1, 1, 0, 3, 5, 1, 2], group, D ** -0.5, cap, window, seed=1)
    compare(c, dtype, [6, 2, 1], [20, 1, 33], group, D ** -0.5, cap, window, seed=2)
    compare(c, dtype, [1], [2], group, D ** -0.5, cap, window, seed=3)


@pytest.mark.parametrize("new", [1, 9])
def test_dealt_out_over_a_ring_with_blocks_that_are_not_numbers(new, dealt):
    ring = 160
    c = Cached(3, ring // 32, 2, 32, 64, ring, seed=4)
    g = torch.Generator().manual_seed(5)
    k, v = (rows_of(490, 2, 64, torch.float32, g, 0.5) for _ in range(2))
    k[40, 1, 3], v[483, 0, 9] = NAN, INF                     # (the first sequence's, long overwritten, and the last one's newest block)
    c.write([0, 1, 2], [400, 30, 60], k, v)
    for dtype in (torch.bfloat16, torch.float32):
        got = compare(c, dtype, [2, 0, 1], [new] * 3, 2, 0.125, 0.0, 100)
        assert torch.isnan(got[:new]).any() and not torch.isnan(got[new:]).any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sequences_of_very_different_lengths(dtype):
    """What the rule deals out by itself, up to as many sequences as it does."""
    lens = [1900, 40, 700, 1, 1300] + [11 * i + 1 for i in range(123)]
    assert kernels.kv8.kv8_shares(128, 1, 1, 9000, 32, 148)[1] < 0
    c = filled(len(lens), 30, 1, 64, 32, lens, seed=12)
    for rows in (list(range(128)), list(range(20)), [3, 0], [0, 1, 2, 3, 4, -1]):
        compare(c, dtype, rows, [1] * len(rows), 2, 0.2, 0.0, 0, max_kv_len=9000)
    compare(c, dtype, [0, 1, 2, 4], [1, 7, 9, 2], 2, 0.2, 20.0, 600, max_kv_len=9000)
    c.lens[1] = 0                                            # (a length of zero: its token sees nothing)
    compare(c, dtype, [0, 1, 2, 4], [1, 1, 1, 1], 2, 0.2, 0.0, 0, max_kv_len=9000)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 3, 80])
def test_blocks_that_a_token_does_not_see_change_nothing(dtype, new, either):
    """A NaN block before the window, or behind the token, must not reach it; one that it sees makes it NaN."""
    for value, at in ((NAN, 10), (INF, 140), (NAN, 295)):
        c = Cached(2, 10, 2, 32, 64, seed=6)
        g = torch.Generator().manual_seed(2)
        k, v = (rows_of(600, 2, 64, torch.float32, g, 0.5) for _ in range(2))
        k[at, 0, 3] = value
        v[300 + at, 1, 5] = value
        c.write([0, 1], [300, 300], k, v)
        got = compare(c, dtype, [0, 1], [new, new], 2, 0.125, 0.0, 100)
        assert not torch.isnan(got).all()
        got = compare(c, dtype, [0, 1], [new, new], 2, 0.125, 25.0, 0)
        assert torch.isnan(got).any() and not torch.isnan(got).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 40])
def test_attention_where_numbers_are_of_all_sizes(dtype, new, either):
    """Keys and values whose blocks differ by powers of ten, queries that are very large or small, scores that leave one
    key all the weight."""
    c = Cached(2, 6, 1, 32, 64, seed=7)
    g = torch.Generator().manual_seed(3)
    for step in range(6):
        k, v = (rows_of(64, 1, 64, torch.float32, g, 0.5) for _ in range(2))
        c.write([0, 1], [32, 32], k * 10.0 ** (step % 3 - 1), v * 10.0 ** (5 - 3 * step))
    q = (torch.randn((2 * new, 128), generator=g)).to(dtype).to(DEV)
    for size in (1.0, 30.0, 1e-30, 0.0):
        compare(c, dtype, [0, 1], [new, new], 2, 0.125, 0.0, 0, q=q * size)
    compare(c, dtype, [0, 1], [new, new], 2, 1e-20, 0.0, 0, q=q * 1e18)
    compare(c, dtype, [0, 1], [new, new], 2, 0.125, 5.0, 0, q=q * 1e4)


@pytest.mark.parametrize("new", [1, 5, 33])
def test_a_query_that_is_not_a_number(new):
    c = filled(2, 3, 2, 32, 32, [70, 50], seed=3)
    g = torch.Generator().manual_seed(4)
    for dtype in (torch.bfloat16, torch.float32):
        q = torch.randn((2 * new, 4 * 32), generator=g).to(dtype).to(DEV)
        q[0, 40] = NAN                                      # one head of one token
        out = torch.empty_like(q)
        kernels.attention_kv8(q, out, ints([0, new, 2 * new]), ints([70, 50]), ints([0, 1]), c.tables, *c.dev, n_kv=2, group=2,
                              head_dim=32, scale=0.2, cap=0.0, window=0, ring=0, batch=2, max_q_len=new, max_kv_len=70)
        bad = torch.isnan(out)
        assert bool(bad[0, 32:64].all()) and int(bad.sum()) == 32


@pytest.mark.parametrize("new", [1, 33, 200])
def test_cache_of_more_than_31_bits_of_bytes(new, on_tcgen05):
    """Blocks whose bytes lie beyond 2^31, of a sequence and of its neighbours' heads."""
    G, P, D = 16, 64, 256
    N = (1 << 31) // (G * P * D) + 40
    dev = [torch.empty((N, G, P, D), dtype=torch.int8, device=DEV) for _ in range(2)] + \
          [torch.full((N, G), NAN, device=DEV) for _ in range(2)]
    blocks = [N - 1, 3, N - 30, N - 2]
    g = torch.Generator().manual_seed(5)
    k, v = (rows_of(200, G, D, torch.bfloat16, g, 0.3) for _ in range(2))
    at = [blocks[p // P] * P + p % P for p in range(200)]
    kernels.kv8_write(k, v, ints([0, 200]), ints(range(200)), ints(at), *dev, max_q_len=200)
    small = [torch.zeros((4, G, P, D), dtype=torch.float64) for _ in range(2)]
    scales = [torch.zeros((4, G), dtype=torch.float64) for _ in range(2)]
    for x, p, s in zip((k, v), small, scales):
        plain.write(x.cpu(), list(range(200)), p, s)
    tables = ints(blocks).view(1, 4)
    ko, vo = torch.empty((2, 200, G, D), dtype=torch.bfloat16, device=DEV)
    kernels.kv8_read(ints([0, 200]), ints([200]), ints([0]), tables, *dev, ko, vo, max_q_len=200)
    keys, values = (plain.read(p, s, range(4), range(200)) for p, s in zip(small, scales))
    assert same(ko.cpu().double(), keys) and same(vo.cpu().double(), values)
    q = torch.randn((new, G * D), generator=g).bfloat16().to(DEV)
    out = torch.empty_like(q)
    kernels.attention_kv8(q, out, ints([0, new]), ints([200]), ints([0]), tables, *dev, n_kv=G, group=1, head_dim=D,
                          scale=1 / 16, cap=0.0, window=0, ring=0, batch=1, max_q_len=new, max_kv_len=200)
    for j in (0, new - 1):
        qj = q[j].cpu().view(G, D)
        ref = plain.attend(qj, keys, values, 0, 200 - new + j, 1 / 16, 0.0, 0)
        off = (out[j].cpu().double().view(G, D) - ref).abs() - bound(torch.bfloat16, ref, qj, keys, values, 1 / 16)
        assert float(off.max()) <= 0.0


def test_everything_on_a_stream_of_its_own_and_twice_the_same_bits():
    """A step's four calls one after the other on a stream that is not the default, without a wait between them."""
    G, P, D, group, B = 2, 64, 128, 4, 3
    g = torch.Generator().manual_seed(6)
    lens, N = [500, 64, 129], 20
    results = []
    for _ in range(2):
        side = torch.cuda.Stream()
        g.manual_seed(6)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            state = dict(tables=torch.zeros((B, 9), dtype=I32, device=DEV), held=ints([0] * B), free=ints(range(N)), free_count=ints([N]))
            cache = [torch.zeros((N, G, P, D), dtype=torch.int8, device=DEV) for _ in range(2)] + \
                    [torch.zeros((N, G), device=DEV) for _ in range(2)]
            out = []
            for before, new in (([0] * B, lens), (lens, [1] * B), ([n + 1 for n in lens], [1, 20, 3])):
                T = sum(new)
                step = dict(cu_q=ints([0] * (B + 1)), kv_len=ints([0] * B), positions=ints([0] * T), tok_seq=ints([0] * T),
                            cache_rows=ints([0] * T), status=ints([0]))
                slots = ints([2, 0, 1])
                kernels.blocks_extend(slots, ints(before), ints(new), *state.values(), block=P, **step)
                x = torch.randn((T, (group + 2) * G * D), generator=g).bfloat16().to(DEV)
                H = group * G * D
                kernels.kv8_write(x[:, H:H + G * D].view(T, G, D), x[:, H + G * D:].view(T, G, D), step["cu_q"], step["positions"],
                                  step["cache_rows"], *cache, max_q_len=max(new))
                o = torch.empty((T, H), dtype=torch.bfloat16, device=DEV)
                kernels.attention_kv8(x[:, :H], o, step["cu_q"], step["kv_len"], slots, state["tables"], *cache, n_kv=G, group=group,
                                      head_dim=D, scale=D ** -0.5, cap=0.0, window=0, ring=0, batch=B, max_q_len=max(new), max_kv_len=520)
                out.append(o)
        side.synchronize()
        results.append(out)
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert all(bool(torch.isfinite(o).all()) for o in results[0])


def test_launchers_refuse_sizes():
    c = Cached(1, 2, 1, 32, 16)
    odd = [torch.zeros((3, 1, 32, 24), dtype=torch.int8, device=DEV)] * 2 + c.dev[2:]
    k = torch.zeros((1, 1, 24), device=DEV)
    for cache, x in ((odd, k),):
        with pytest.raises(kernels.KernelError, match="size"):
            kernels.kv8_write(x, x, ints([0, 1]), ints([0]), ints([0]), *[a[:3].contiguous() for a in cache], max_q_len=1)
    block = [torch.zeros((3, 1, 48, 16), dtype=torch.int8, device=DEV)] * 2 + [d[:3].contiguous() for d in c.dev[2:]]
    q = torch.zeros((1, 16), device=DEV)
    with pytest.raises(kernels.KernelError, match="size"):
        kernels.attention_kv8(q, q.clone(), ints([0, 1]), ints([1]), ints([0]), c.tables, *block, n_kv=1, group=1, head_dim=16, scale=1.0,
                              cap=0.0, window=0, ring=0, batch=1, max_q_len=1, max_kv_len=1)
    with pytest.MonkeyPatch.context() as m:                  # fewer clusters than sequences
        m.setattr(kernels.kv8, "kv8_shares", lambda *a: (1, -1))
        with pytest.raises(kernels.KernelError, match="size"):
            kernels.attention_kv8(q.repeat(2, 1), q.repeat(2, 1), ints([0, 1, 2]), ints([1, 1]), ints([0, 0]), c.tables, *c.dev, n_kv=1, group=1,
                                  head_dim=16, scale=1.0, cap=0.0, window=0, ring=0, batch=2, max_q_len=1, max_kv_len=1)
    k = torch.zeros((2, 1, 16), device=DEV)
    off = torch.zeros(40, device=DEV)[1:33].view(2, 1, 16)
    with pytest.raises(kernels.KernelError, match="aligned"):
        kernels.kv8_read(ints([0, 2]), ints([2]), ints([0]), c.tables, *c.dev, off, k, max_q_len=2)
    with pytest.raises(kernels.KernelError, match="size"):
        kernels.blocks_extend(ints([0]), ints([0]), ints([1]), c.tables, ints([0]), ints([0]), ints([1]), block=32, ring=40,
                              cu_q=ints([0, 0]), kv_len=ints([0]), positions=ints([0]), tok_seq=ints([0]), cache_rows=ints([0]),
                              status=ints([0]))


# --- pieces of prompts on tcgen05 --------------------------------------------------------------------------------------
@pytest.mark.parametrize("D,G,group,P,cap", [(64, 2, 3, 32, 0.0), (128, 1, 5, 96, 30.0), (256, 2, 2, 64, 50.0), (256, 1, 1, 256, 0.0),
                                             (128, 3, 4, 128, 3.0)])
def test_pieces_of_prompts(D, G, group, P, cap, on_tcgen05):
    """More rows than a block of threads has, row tiles that end inside a token's heads, sequences that bring little or
    nothing (their rows of the tile are empty), lengths that end inside a tile, a window that begins inside one."""
    lens = [300, 1, 129, 0, 515, 128]
    c = filled(len(lens), -(-576 // P), G, P, D, [max(1, n) for n in lens], seed=D + P)
    c.lens[3] = 0
    for new, window in (([150, 1, 129, 0, 70, 128], 0), ([1, 0, 60, 0, 200, 33], 100), ([80, 1, 0, 0, 300, 1], 1)):
        compare(c, torch.bfloat16, list(range(6)), new, group, D ** -0.5, cap, window, seed=sum(new), q_spread=2.0)
    compare(c, torch.bfloat16, [4, -1, 0], [100, 3, 90], group, D ** -0.5, cap, 0)
    for window in (31, 130):
        compare(c, torch.bfloat16, [4, 0], [100, 128], group, D ** -0.5, cap, window)


def test_a_piece_over_a_ring_of_unusual_blocks(on_tcgen05):
    P, window, new = 96, 50, 70
    ring = (window + new + P - 2 + P - 1) // P * P
    c = filled(2, ring // P, 2, P, 128, [1, 90], ring=ring, seed=new)
    g = torch.Generator().manual_seed(8)
    for _ in range(5):
        c.write([0, 1], [new] * 2, rows_of(2 * new, 2, 128, torch.bfloat16, g), rows_of(2 * new, 2, 128, torch.bfloat16, g))
        compare(c, torch.bfloat16, [1, 0], [new] * 2, 3, 0.1, 0.0, window, seed=c.lens[0])


def test_queries_and_results_of_a_piece_that_begin_off_sixteen_bytes(on_tcgen05):
    c = filled(1, 4, 2, 64, 64, [200], seed=2)
    wide = torch.randn((100, 300)).bfloat16().to(DEV)
    for at in (1, 4, 8):
        out = torch.full((100, 300), 7.0, dtype=torch.bfloat16, device=DEV)
        args = dict(n_kv=2, group=2, head_dim=64, scale=0.125, cap=0.0, window=0, ring=0, batch=1, max_q_len=100, max_kv_len=200)
        rest = (ints([0, 100]), ints([200]), ints([0]), c.tables, *c.dev)
        kernels.attention_kv8(wide[:, at:at + 256], out[:, at:at + 256], *rest, **args)
        q, plain_out = wide[:, at:at + 256].contiguous(), torch.empty((100, 256), dtype=torch.bfloat16, device=DEV)
        kernels.attention_kv8(q, plain_out, *rest, **args)
        assert torch.equal(out[:, at:at + 256], plain_out)
        assert bool((out[:, :at] == 7.0).all()) and bool((out[:, at + 256:] == 7.0).all())


def test_a_query_of_a_piece_that_is_not_a_number(on_tcgen05):
    c = filled(1, 3, 1, 64, 64, [150], seed=3)
    q = torch.randn((90, 2 * 64)).bfloat16().to(DEV)
    q[17, 70] = INF
    out = torch.empty_like(q)
    kernels.attention_kv8(q, out, ints([0, 90]), ints([150]), ints([0]), c.tables, *c.dev, n_kv=1, group=2, head_dim=64, scale=0.1,
                          cap=0.0, window=0, ring=0, batch=1, max_q_len=90, max_kv_len=150)
    bad = torch.isnan(out)
    assert bool(bad[17, 64:].all()) and int(bad.sum()) == 64


def test_a_piece_whose_values_scales_lie_2_to_the_100_apart(on_tcgen05):
    """Blocks of values of size 1, 2^-70 and 2^-110 beside each other: rows that see only small ones keep their bits, and rows
    that see large ones lose nothing by them."""
    c = Cached(1, 6, 1, 32, 64, seed=7)
    g = torch.Generator().manual_seed(3)
    for step in range(6):
        k, v = (rows_of(32, 1, 64, torch.float32, g, 0.2) for _ in range(2))
        c.write([0], [32], k, v * 2.0 ** (-110, -70, -110, 0, -70, 0)[step])
    compare(c, torch.bfloat16, [0], [100], 1, 0.125, 0.0, 20)        # windows of 20: most rows see one or two blocks
    compare(c, torch.bfloat16, [0], [192], 1, 0.125, 0.0, 0)


@pytest.mark.parametrize("D", [16, 48, 80, 96, 112, 192, 240])
def test_pieces_of_heads_between_the_sizes(D, on_tcgen05, monkeypatch):
    """Heads whose rows end inside a copied box, or a whole box before the last."""
    c = filled(2, 10, 3, 32, D, [310, 200], seed=D)
    compare(c, torch.bfloat16, [1, 0], [140, 75], 3, D ** -0.5, 30.0, 0)
    compare(c, torch.bfloat16, [0], [200], 1, D ** -0.5, 0.0, 150)
    monkeypatch.setattr(kernels.kv8, "kv8_tc_spans", lambda *a: (2, 3))
    compare(c, torch.bfloat16, [0, 1], [129, 130], 2, D ** -0.5, 0.0, 0)


@pytest.mark.parametrize("shared", [(0, 3), (1, 2), (5, 4), (7, 30)], ids=str)
@pytest.mark.parametrize("D,window", [(64, 0), (256, 0), (128, 90)])
def test_a_piece_some_of_whose_tiles_are_shared(D, window, shared, on_tcgen05, monkeypatch):
    """The first tiles with a block each, the others' keys shared by several; tokens before a sequence's first, and a query
    that is not a number, on both sides."""
    monkeypatch.setattr(kernels.kv8, "kv8_tc_spans", lambda *a: shared)
    c = filled(3, 12, 2, 64, D, [700, 150, 333], seed=D)
    compare(c, torch.bfloat16, [0], [260], 2, D ** -0.5, 25.0, window)                       # (ten tiles)
    compare(c, torch.bfloat16, [2, 0, 1], [130, 70, 150], 2, D ** -0.5, 0.0, window)         # (eighteen)
    c.lens[1] = 60                                           # of 150 new tokens 90 come before the first
    compare(c, torch.bfloat16, [1], [150], 3, D ** -0.5, 0.0, window)
    c.lens[1] = 150
    q = torch.randn((260, 4 * D), generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    q[3, 5] = q[200, 3 * D] = NAN
    out = torch.empty_like(q)
    kernels.attention_kv8(q, out, ints([0, 260]), ints([700]), ints([0]), c.tables, *c.dev, n_kv=2, group=2, head_dim=D, scale=0.1, cap=0.0,
                          window=window, ring=0, batch=1, max_q_len=260, max_kv_len=700)
    bad = torch.isnan(out)
    assert bool(bad[3, :D].all()) and bool(bad[200, 3 * D:].all()) and int(bad.sum()) == 2 * D


@pytest.mark.parametrize("code", [8, 9, 15])
def test_a_piece_whose_wait_runs_out(code, on_tcgen05):
    """The softmax warps' waits for a score tile and for the lookups never end: the launch gives up, says so, and the next
    one is right."""
    c = filled(1, 10, 2, 64, 128, [600], seed=5)
    q = torch.randn((200, 4 * 128)).bfloat16().to(DEV)

    def run():
        out = torch.empty_like(q)
        kernels.attention_kv8(q, out, ints([0, 200]), ints([600]), ints([0]), c.tables, *c.dev, n_kv=2, group=2, head_dim=128,
                              scale=0.09, cap=0.0, window=0, ring=0, batch=1, max_q_len=200, max_kv_len=600)
        torch.cuda.synchronize()
        return out

    good = run()
    assert kernels.attention_kv8_tc_status(reset=True) == 0
    kernels.wait_control("attn_kv8_tc", cycles=8_000_000, stall_code=code)
    try:
        run()
        assert kernels.attention_kv8_tc_status(reset=True) == code and kernels.attention_kv8_tc_status() == 0
    finally:
        kernels.wait_control("attn_kv8_tc", 0, 0)
    assert torch.equal(run(), good) and kernels.attention_kv8_tc_status() == 0


# --- sums of weights beside values of other sizes ------------------------------------------------------------------------
def small_beside_large(sizes, dtype=torch.float32):
    """A sequence of blocks of 64 tokens whose values are about 1 times ``sizes``, one after the other."""
    c = Cached(1, len(sizes), 1, 64, 64, seed=7)
    g = torch.Generator().manual_seed(3)
    for size in sizes:
        k, v = (rows_of(64, 1, 64, torch.float32, g, 0.2) for _ in range(2))
        c.write([0], [64], k, (v.abs() + 1.0) * size)
    return c


@pytest.mark.parametrize("shared", [None, (0, 1), (0, 3), (1, 2)], ids=str)
@pytest.mark.parametrize("new", [1, 5, 100])
def test_many_values_of_zero_before_values_that_are_not(new, shared, either, monkeypatch):
    """Blocks of zeros have the least scale there is, 2^-126: their weights count in the sum all the same, however many come
    before the first value, and whatever its size."""
    if shared:
        monkeypatch.setattr(kernels.kv8, "kv8_tc_spans", lambda *a: shared)
    for sizes in ([0.0] * 40 + [1.0], [0.0] * 20 + [1.0] + [0.0] * 20 + [2.0 ** 12] * 2, [1.0] + [0.0] * 30 + [2.0 ** 40, 0.0, 0.0]):
        c = small_beside_large(sizes)
        for dtype in (torch.bfloat16, torch.float32):
            got = compare(c, dtype, [0], [new], 2, 0.125, 0.0, 0)
            assert not torch.isnan(got).any()


@pytest.mark.parametrize("shared", [None, (0, 1), (0, 2)], ids=str)
def test_rows_that_see_small_values_alone_keep_them(shared, either, monkeypatch):
    """Rows of one tile under a window of 20: those that see values of 2^-60 alone are as near to 64 bits, beside what they
    see, as those that see values of 2^70 (or of both)."""
    if shared:
        monkeypatch.setattr(kernels.kv8, "kv8_tc_spans", lambda *a: shared)
    c = small_beside_large([2.0 ** -60, 2.0 ** 70, 2.0 ** -60, 2.0 ** -60, 2.0 ** 70])
    n, new = 320, 250
    for dtype in (torch.bfloat16, torch.float32):
        q = torch.randn((new, 64), generator=torch.Generator().manual_seed(5)).to(dtype).to(DEV)
        out = torch.empty_like(q)
        kernels.attention_kv8(q, out, ints([0, new]), ints([n]), ints([0]), c.tables, *c.dev, n_kv=1, group=1, head_dim=64, scale=0.125,
                              cap=0.0, window=20, ring=0, batch=1, max_q_len=new, max_kv_len=n)
        keys, values = c.values(0, 0)[1], c.values(1, 0)[1]
        for j in range(new):
            p = n - new + j
            lo = max(0, p - 19)
            qj = q[j].cpu().view(1, 64)
            ref = plain.attend(qj, keys, values, 0, p, 0.125, 0.0, 20)
            off = (out[j].cpu().double().view(1, 64) - ref).abs() - bound(dtype, ref, qj, keys[lo:p + 1], values[lo:p + 1], 0.125)
            assert float(off.max()) <= 0.0, (dtype, j, float(off.max()))


@pytest.mark.parametrize("dtype,new", [(torch.bfloat16, 1), (torch.float32, 1), (torch.bfloat16, 10), (torch.float32, 10),
                                       (torch.bfloat16, 40)])
def test_a_sequence_of_more_than_2_to_the_30_tokens(dtype, new, on_tcgen05):
    """Without a window the newest token sees the first ones.  The first 4,096 keys lie in one block's worth of numbers and
    all others in another's; scores of 15 and 0 give the first e^15 2^12 of e^15 2^12 + 2^30 parts of the weight, values of 1
    and -1 so 0.8515.  (Sums of so many equal numbers lose up to 2^-25 of themselves with each: 2^18 of them, a warp's or a
    thread's share, 2^-7.)"""
    P, D, n = 256, 16, (1 << 30) + 4096
    key = torch.zeros((2 * P, 1, D), device=DEV)
    key[:P, 0, 0] = 15.0
    value = torch.ones((2 * P, 1, D), device=DEV)
    value[P:] = -1.0
    dev = [torch.zeros((2, 1, P, D), dtype=torch.int8, device=DEV) for _ in range(2)] + [torch.zeros((2, 1), device=DEV) for _ in range(2)]
    kernels.kv8_write(key, value, ints([0, 2 * P]), ints(range(2 * P)), ints(range(2 * P)), *dev, max_q_len=2 * P)
    table = torch.ones((1, n // P), dtype=I32, device=DEV)
    table[0, :4096 // P] = 0
    q = torch.zeros((new, D), dtype=dtype, device=DEV)
    q[:, 0] = 1.0
    out = torch.empty_like(q)
    kernels.attention_kv8(q, out, ints([0, new]), ints([n]), ints([0]), table, *dev, n_kv=1, group=1, head_dim=D, scale=1.0, cap=0.0,
                          window=0, ring=0, batch=1, max_q_len=new, max_kv_len=n)
    share = math.exp(15.0) * 4096 / (math.exp(15.0) * 4096 + 2.0 ** 30)
    off = (out.cpu().double() - (2.0 * share - 1.0)).abs().max()
    assert kernels.attention_kv8_tc_status() == 0 and float(off) <= 2.0 ** -7 + 2.0 ** -8
    k, v = torch.empty((2, 3, 1, D), device=DEV)
    kernels.kv8_read(ints([0, 3]), ints([n]), ints([0]), table, *dev, k, v, max_q_len=3)
    assert bool((v == -1.0).all()) and not k.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("new", [1, 5, 70])
@pytest.mark.parametrize("P", [32, 128])
def test_blocks_that_are_not_the_caches_are_passed_over(dtype, new, P, either):
    """Ids outside the cache, and places beyond the table's width: nobody's keys are seen there."""
    c = filled(3, -(-512 // P), 2, P, 64, [500, 300, 64], seed=9)
    n, group, scale = c.pages[0].shape[0], 2, 0.125
    table = c.tables.clone()
    gone = [set(), set(), set()]
    for i, e, bad in ((0, 1, -1), (0, 3, n), (1, 0, 2 ** 31 - 1), (1, 2, -2 ** 31), (2, 0, -1)):
        if P == 128 or i < 2:
            table[i, e] = bad
            gone[i].add(e)
    if P == 32:
        table[2, :2] = n + 5                                 # (a sequence that has nothing left)
        gone[2] = {0, 1}
    for width in (table.shape[1], 384 // P):
        q = torch.randn((3 * new, 4 * 64), generator=torch.Generator().manual_seed(new)).to(dtype).to(DEV)
        out = torch.full_like(q, 9.0)
        kernels.attention_kv8(q, out, ints([0, new, 2 * new, 3 * new]), ints(c.lens), ints([0, 1, 2]), table[:, :width].contiguous(), *c.dev,
                              n_kv=2, group=group, head_dim=64, scale=scale, cap=0.0, window=0, ring=0, batch=3, max_q_len=new,
                              max_kv_len=500)
        k, v = (torch.empty((sum(c.lens), 2, 64), device=DEV) for _ in range(2))
        kernels.kv8_read(ints([0, 500, 800, 864]), ints(c.lens), ints([0, 1, 2]), table[:, :width].contiguous(), *c.dev, k, v, max_q_len=500)
        at = 0
        for i, length in enumerate(c.lens):
            keys, values = c.values(0, i)[1], c.values(1, i)[1]
            here = torch.tensor([p // P not in gone[i] and p // P < width for p in range(length)])
            assert same(k[at:at + length].cpu().double(), torch.where(here[:, None, None], keys, 0.0))
            at += length
            for j in range(new):
                p = length - new + j
                sees = here.nonzero()[:, 0][here.nonzero()[:, 0] <= p]
                qj = q[i * new + j].cpu().view(4, 64)
                ref = plain.attend(qj, keys[sees], values[sees], 0, len(sees) - 1, scale, 0.0, 0) if p >= 0 else torch.zeros(4, 64).double()
                off = (out[i * new + j].cpu().double().view(4, 64) - ref).abs() - bound(dtype, ref, qj, keys, values, scale)
                assert float(off.max()) <= 0.0, (width, i, j, float(off.max()))


@pytest.mark.parametrize("tokens", [8, 40000])
def test_the_first_refusal_is_kept_until_someone_has_seen_it(tokens):
    """Behind one launch and behind the steps that all SMs share; calls that are fine in between, and the release."""
    t = Tables(4, 3, 7, 32, 0, 0)
    refused = ints([0])

    def step(slots, lengths, new):
        out = dict(cu_q=ints([7] * (len(slots) + 1)), kv_len=ints([7] * len(slots)), positions=ints([7] * tokens),
                   tok_seq=ints([7] * tokens), cache_rows=ints([7] * tokens), status=ints([7]))
        kernels.blocks_extend(ints(slots), ints(lengths), ints(new), *t.dev.values(), block=32, refused=refused, **out)
        return int(out["status"]), int(refused)

    def release(slots):
        status = ints([7])
        kernels.blocks_release(ints(slots), *t.dev.values(), status=status, refused=refused)
        return int(status), int(refused)

    assert step([0], [0], [5]) == (0, 0) and release([1]) == (0, 0)
    assert step([0, 1], [5, 0], [1, 97 if tokens > 100 else 2 ** 20]) == (2 if tokens > 100 else 3, 2 if tokens > 100 else 3)
    assert step([0], [5], [1])[0] == 0 and release([0, 9])[0] == 4 and release([0])[0] == 0
    assert int(refused) == (2 if tokens > 100 else 3)
    refused.zero_()
    assert release([2, 2]) == (4, 4) and step([0], [0], [1]) == (0, 4)
    for wrong in (ints([0, 0]), torch.zeros(1, device=DEV)):
        with pytest.raises(kernels.KernelError, match="refused"):
            kernels.blocks_release(ints([0]), *t.dev.values(), status=ints([0]), refused=wrong)


def test_read_gives_no_more_of_a_row_than_it_is_told():
    c = Cached(2, 5, 2, 32, 48, seed=5)
    g = torch.Generator().manual_seed(1)
    c.write([0, 1], [130, 90], rows_of(220, 2, 48, torch.float32, g), rows_of(220, 2, 48, torch.float32, g))
    for most in (1, 37, 90, 130):
        k, v = torch.full((2, 220, 2, 48), 5.0, device=DEV)
        kernels.kv8_read(ints([0, 130, 220]), ints([130, 90]), ints([0, 1]), c.tables, *c.dev, k, v, max_q_len=most)
        for which, got in ((0, k), (1, v)):
            for i, (at, n) in enumerate(((0, 130), (130, 90))):
                want = c.values(which, i)[1]
                want[:max(0, n - most)] = 0.0
                assert same(got[at:at + n].cpu().double(), want)


@pytest.mark.parametrize("tokens", [200, 40000])
def test_block_ids_that_no_cache_has_give_no_places(tokens):
    """Ids whose places pass 31 bits, or come before the first, must not come back as another block's."""
    ids = [5, 2 ** 27, -1, -2 ** 27, 2 ** 31 - 1, 2 ** 26 - 1, -2 ** 31]
    free = ints(reversed(ids))
    state = dict(tables=torch.zeros((2, 8), dtype=I32, device=DEV), held=ints([0, 0]), free=free, free_count=ints([len(ids)]))
    for before, n in ((0, 200), (200, 24)):                       # taken from the stack, then found in the table
        out = dict(cu_q=ints([7, 7]), kv_len=ints([7]), positions=ints([7] * tokens), tok_seq=ints([7] * tokens),
                   cache_rows=ints([7] * tokens), status=ints([7]))
        kernels.blocks_extend(ints([1]), ints([before]), ints([n]), *state.values(), block=32, **out)
        want = [ids[p // 32] * 32 + p % 32 if ids[p // 32] in (5, 2 ** 26 - 1) else -1 for p in range(before, before + n)]
        assert int(out["status"]) == 0 and out["cache_rows"][:n].tolist() == want


@pytest.mark.parametrize("tokens", [3000, 120000])
def test_lengths_that_go_on_in_place(tokens):
    """`kv_len` is `lengths`: many rows, so that some blocks of threads still read while others write."""
    n, block = 4000, 32
    rng = random.Random(tokens)
    new = [rng.choice([0, 1, 1]) if tokens < 4000 else rng.choice([1, 20, 40]) for _ in range(n)]
    new = [0 if sum(new[:i]) > tokens - 50 else m for i, m in enumerate(new)] if sum(new) > tokens else new
    slots = [i if rng.random() < 0.95 else -1 for i in rng.sample(range(n), n)]
    state = dict(tables=torch.zeros((n, 12), dtype=I32, device=DEV), held=ints([0] * n), free=ints(range(30000)), free_count=ints([30000]))
    lengths, want = ints([5] * n), [5] * n
    out = dict(cu_q=ints([0] * (n + 1)), positions=ints([0] * tokens), tok_seq=ints([0] * tokens), cache_rows=ints([0] * tokens), status=ints([7]))
    for turn in range(4):
        kernels.blocks_extend(ints(slots), lengths, ints(new), *state.values(), block=block, kv_len=lengths, **out)
        want = [w + m if s >= 0 else 0 for w, m, s in zip(want, new, slots)]
        assert int(out["status"]) == 0 and lengths.tolist() == want
        held = [0] * n
        for w, s in zip(want, slots):
            if s >= 0:
                held[s] = -(-w // block)
        assert state["held"].tolist() == held and int(state["free_count"]) == 30000 - sum(held)
        pos = [p for w, m, s in zip(want, new, slots) for p in (range(w - m, w) if s >= 0 else [-1] * m)]
        assert out["positions"][:len(pos)].tolist() == pos
    before = lengths.clone()
    kernels.blocks_extend(ints(slots), lengths, ints([10000] + new[1:]), *state.values(), block=block, kv_len=lengths, **out)
    assert int(out["status"]) > 0 and not lengths.any() and bool(before.any())
