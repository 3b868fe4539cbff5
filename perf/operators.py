"""The cache in 8 bits, the block tables it lives by, and the attention over it, as timed cases.

A case is one pass through one of four operators (``kind``):

* ``tables``: ``kernels.blocks_extend``: a step's requests take the cache blocks that their new tokens need from a stack of
  free ones, and every token of the step gets its position, its request and its place in the cache; with ``release`` the
  requests end in the same pass and ``kernels.blocks_release`` takes their blocks back.
* ``append``: ``kernels.kv8_write``: new keys and values go into blocks of 8-bit numbers with a scale for each block and
  head, blocks that were begun before among them; then ``kernels.kv8_read`` gives back all that the cache holds.
* ``read``: ``kernels.kv8_read`` alone, over long sequences: what a program does that hands a sequence on, or looks at it.
* ``attend``: ``kernels.attention_kv8``: one new token a sequence (decoding), a few (several drafted tokens looked at in
  one step), or a long piece of a prompt, whose keys and values are already in the cache.

The cache: ``[blocks][kv heads][tokens of a block][entries]`` numbers of 8 bits and float32 scales ``[blocks][kv heads]``,
a number standing for q * scale; a sequence's blocks are the first entries of its row of ``tables``.  The scale of a block
and head is the least power of two, 2^-126 at least, under which none of its numbers is beyond 127; it never shrinks while a
block fills, and when it grows the numbers that were there are rounded to it.  A block that gets a number that is not finite
has the scale NaN.  With a ring, position p lives at place p % ring, and the newest ring / block blocks are kept.
"""
from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda:0"
F32 = torch.float32
F64 = torch.float64
I32 = torch.int32
TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# --- the cases ---------------------------------------------------------------------------------------------------------
def _lengths(b, lo, hi):
    """b lengths from lo to hi, spread over their logarithm and then stirred, the same ones every time."""
    if b == 1:
        return [hi]
    out = [round(lo * (hi / lo) ** (i / (b - 1))) for i in range(b)]
    return [out[(i * 7 + 3) % b] for i in range(b)] if b % 7 else out


def _texts(values):
    return " ".join(str(int(v)) for v in values)


def _numbers(text):
    return [int(v) for v in text.split()]


def listed():
    two_b = dict(n_kv=4, group=2, dim=256, scale=256 ** -0.5, cap=50.0, type="bfloat16", block=64)
    nine_b = dict(two_b, n_kv=8)
    tables = dict(kind="tables", block=64, ring=0, release=False)
    return [
        # a decode step of 64 requests among 256 slots: the smallest call, once a step and cache group
        dict(tables, name="tables-decode-64", requests=64, slots=256, before=_texts(_lengths(64, 65, 8192)), new=_texts([1] * 64)),
        # a batch of 16 prompts of 128 to 6,144 tokens arrives and, answered, leaves again
        dict(tables, name="tables-prompts-16", requests=16, slots=64, before=_texts([0] * 16), new=_texts(_lengths(16, 128, 6144)),
             release=True),
        # 300 short prompts at once into a windowed layer's ring
        dict(tables, name="tables-prompts-300-ring", requests=300, slots=512, before=_texts([0] * 300),
             new=_texts(_lengths(300, 5, 2000)), block=32, ring=1056, release=True),
        # one token more for each of 64 short sequences
        dict(two_b, kind="append", name="append-decode-64", ring=0, before=_texts(_lengths(64, 1, 250)), new=_texts([1] * 64)),
        # a whole prompt
        dict(two_b, kind="append", name="append-prompt-2048", ring=0, before="0", new="2048"),
        # float32, ragged pieces of prompts that begin inside blocks, a ring that wraps
        dict(kind="append", name="append-pieces-float", n_kv=2, group=2, dim=96, type="float32", block=32, ring=320,
             before="17 0 300 95 1021", new="611 5 33 1 290"),
        # 16 sequences handed on to 16-bit kernels
        dict(nine_b, kind="read", name="read-16", ring=0, before=_texts(_lengths(16, 128, 6144))),
        # one sequence, the smallest attention of a program
        dict(two_b, kind="attend", name="attend-decode-1", window=0, ring=0, lens="1280", new="1"),
        # decoding at batch 8 and context 8,192
        dict(two_b, kind="attend", name="attend-decode-8", window=0, ring=0, lens=_texts([8192] * 8), new=_texts([1] * 8)),
        # very unequal sequences under a window
        dict(nine_b, kind="attend", name="attend-decode-16-window", window=4096, ring=4160, lens=_texts(_lengths(16, 129, 6145)),
             new=_texts([1] * 16)),
        # float32, five drafted tokens each, four heads on a kv head, odd lengths
        dict(kind="attend", name="attend-drafts-float", n_kv=4, group=4, dim=128, scale=128 ** -0.5, cap=30.0, type="float32",
             block=64, window=0, ring=0, lens="4001 77 1999 13 640 2750", new=_texts([5] * 6)),
        # the last piece of a long prompt
        dict(nine_b, kind="attend", name="attend-piece-2048", window=0, ring=0, lens="14336", new="2048"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng: random.Random):
    kind = rng.choice(["tables", "append", "read", "attend", "attend", "attend"])
    block = rng.choice([32, 64, 64, 128])
    if kind == "tables":
        n = _log(rng, 1, 300)
        ring = rng.choice([0, 0, block * rng.randint(2, 70)])
        fresh = rng.random() < 0.5
        most = max(8, min(6144, 150_000 // n))
        before = [0] * n if fresh else [_log(rng, 1, 8192) for _ in range(n)]
        new = [_log(rng, 1, most) for _ in range(n)] if fresh else [rng.choice([0, 1, 1, 1, 2, 5]) for _ in range(n)]
        new[0] = max(1, new[0])
        return dict(kind="tables", requests=n, slots=n + rng.randint(0, 200), before=_texts(before), new=_texts(new), block=block,
                    ring=ring, release=fresh)
    heads = dict(n_kv=rng.choice([1, 2, 4, 4, 8, 16]), group=rng.choice([1, 2, 2, 4, 6, 8]),
                 dim=rng.choice([16, 32, 64, 80, 96, 128, 192, 256]), type=rng.choice(["bfloat16", "bfloat16", "float32"]), block=block)
    row = heads["n_kv"] * heads["dim"]                       # numbers of a token's keys
    if kind in ("append", "read"):
        b = _log(rng, 1, 64)
        most = max(16, min(8192, 16_000_000 // (row * b)))
        total = [_log(rng, 2, most) for _ in range(b)]
        if kind == "read":
            return dict(heads, kind="read", ring=0, before=_texts(total))
        new = [1 if rng.random() < 0.3 else rng.randint(1, t) for t in total]
        if rng.random() < 0.4:
            new = [1] * b
        ring = rng.choice([0, 0, block * rng.randint(2, 20)])
        return dict(heads, kind="append", ring=ring, before=_texts(t - n for t, n in zip(total, new)), new=_texts(new))
    case = dict(heads, kind="attend", scale=heads["dim"] ** -0.5, cap=rng.choice([0.0, 30.0, 50.0]))
    style = rng.choice(["decode", "decode", "drafts", "piece"])
    b = _log(rng, 1, 4 if style == "piece" else 64)
    most = max(32, min(16384, 120_000_000 // (row * b)))
    lens = [_log(rng, 2, most) for _ in range(b)] if rng.random() < 0.6 else [_log(rng, max(2, most // 8), most)] * b
    if style == "decode":
        new = [1] * b
    elif style == "drafts":
        new = [min(l, rng.randint(1, 8)) for l in lens]
    else:
        fits = 150e9 / (4.0 * row * heads["group"] * b)      # (token, key) pairs of a sequence
        new = [max(1, min(l, _log(rng, 16, 1024), int(fits / l))) for l in lens]
    window = rng.choice([0, 0, _log(rng, 8, 4096)])
    ring = (window + max(new) + 2 * block - 2) // block * block if window else 0
    return dict(case, window=window, ring=ring, lens=_texts(lens), new=_texts(new))


# --- a state's parts ---------------------------------------------------------------------------------------------------
def _int(values):
    return torch.tensor(list(values), dtype=I32, device=DEV)


def _sums(values):
    return [0] + np.cumsum(np.asarray(values, dtype=np.int64)).tolist()


def _need(n, block, ring):
    """Blocks that a sequence of n tokens holds."""
    return (min(n, ring or n) + block - 1) // block


def _first_kept(n, block, ring):
    """The oldest position that a sequence of n tokens still has in its ring."""
    return max(0, ((n - 1) // block - ring // block + 1) * block) if ring and n else 0


def _blocks_of(lengths, block, ring, gen):
    """Every sequence's row of the tables, blocks in no order, and how many blocks there are."""
    need = [max(1, _need(n, block, ring)) for n in lengths]
    n_blocks = sum(need) + 3
    order = torch.randperm(n_blocks, generator=gen, device=DEV).to(I32)
    tables = torch.zeros((len(need), max(need)), dtype=I32, device=DEV)
    at = 0
    for i, n in enumerate(need):
        tables[i, :n] = order[at:at + n]
        at += n
    return tables, n_blocks


def _pages(n_blocks, case, gen):
    """Blocks full of numbers: keys or values of deviation about 1."""
    G, P, D = case["n_kv"], case["block"], case["dim"]
    q = torch.randn((n_blocks, G, P, D), generator=gen, device=DEV).mul_(40.0).round_().clamp_(-127.0, 127.0).to(torch.int8)
    scale = torch.exp2(torch.randint(-6, -4, (n_blocks, G), generator=gen, device=DEV).to(F32))
    return q, scale


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(1_000_003 * seed + 17)
    kind, block = case["kind"], case["block"]
    ring = case.get("ring", 0)
    if kind == "tables":
        before, new = _numbers(case["before"]), _numbers(case["new"])
        n, S = case["requests"], case["slots"]
        after = [a + b for a, b in zip(before, new)]
        width = max(1, max(_need(x, block, ring) for x in after)) + 1
        held_of = [_need(x, block, ring) for x in before]
        total = sum(_need(x, block, ring) for x in after) + 16
        order = torch.randperm(total, generator=gen, device=DEV).to(I32)
        slots = torch.randperm(S, generator=gen, device=DEV)[:n].to(I32)
        tables = torch.zeros((S, width), dtype=I32, device=DEV)
        held = torch.zeros(S, dtype=I32, device=DEV)
        held[slots.long()] = _int(held_of)
        at = _int(_sums(held_of)[:-1])
        cols = torch.arange(width, device=DEV)
        mine = cols[None, :] < _int(held_of)[:, None]
        tables[slots.long()] = torch.where(mine, order[(at[:, None] + cols[None, :]).clamp_(max=total - 1).long()], tables[slots.long()])
        left = total - sum(held_of)
        free = torch.zeros(total, dtype=I32, device=DEV)
        free[:left] = order[sum(held_of):]
        T = sum(new)
        return dict(case=case, slots=slots, lengths=_int(before), new=_int(new), tables=tables, held=held, free=free,
                    free_count=_int([left]), cu_q=torch.zeros(n + 1, dtype=I32, device=DEV),
                    kv_len=torch.zeros(n, dtype=I32, device=DEV), positions=torch.zeros(T, dtype=I32, device=DEV),
                    tok_seq=torch.zeros(T, dtype=I32, device=DEV), cache_rows=torch.zeros(T, dtype=I32, device=DEV),
                    status=torch.zeros(1, dtype=I32, device=DEV))
    if kind == "attend":
        lens, new = _numbers(case["lens"]), _numbers(case["new"])
    else:
        before = _numbers(case["before"])
        new = _numbers(case["new"]) if kind == "append" else [0] * len(before)
        lens = [a + b for a, b in zip(before, new)]
    tables, n_blocks = _blocks_of(lens, block, ring, gen)
    k_pages, k_scale = _pages(n_blocks, case, gen)
    v_pages, v_scale = _pages(n_blocks, case, gen)
    dt = TYPES[case["type"]]
    B, T, G, D = len(lens), sum(new), case["n_kv"], case["dim"]
    state = dict(case=case, lens=lens, new=new, kv_len=_int(lens), slots=torch.arange(B, dtype=I32, device=DEV), tables=tables,
                 k_pages=k_pages, v_pages=v_pages, k_scale=k_scale, v_scale=v_scale)
    if kind == "attend":
        q = torch.randn((T, G * case["group"] * D), generator=gen, device=DEV).mul_(1.5).to(dt)
        state.update(cu_q=_int(_sums(new)), q=q)
        return state
    kept = [n - _first_kept(n, block, ring) for n in lens]
    state.update(cu_r=_int(_sums(kept)), rows=sum(kept), longest=max(kept))
    if kind == "append":
        # rows of a fused projection's result: the keys and values are parts of a wider row
        qkv = torch.randn((T, (case["group"] + 2) * G * D), generator=gen, device=DEV)
        qkv.mul_(torch.exp(0.5 * torch.randn((T, 1), generator=gen, device=DEV)))
        qkv = qkv.to(dt)
        H = case["group"] * G * D
        places = []
        host_tables = tables.cpu().numpy()
        for i, (a, n) in enumerate(zip(lens, new)):
            pos = np.arange(a - n, a)
            place = pos % ring if ring else pos
            rows = host_tables[i][place // block].astype(np.int64) * block + place % block
            places.append(np.where(pos < _first_kept(a, block, ring), -1, rows))
        state.update(k=qkv[:, H:H + G * D].view(T, G, D), v=qkv[:, H + G * D:].view(T, G, D), cu_q=_int(_sums(new)),
                     positions=_int(np.concatenate([np.arange(a - n, a) for a, n in zip(lens, new)]).tolist()),
                     cache_rows=_int(np.concatenate(places).tolist()))
    return state


# --- one pass ----------------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(s):
    from brolm_b200 import kernels
    case = s["case"]
    kind = case["kind"]
    if kind == "tables":
        kernels.blocks_extend(s["slots"], s["lengths"], s["new"], s["tables"], s["held"], s["free"], s["free_count"],
                              block=case["block"], ring=case["ring"], cu_q=s["cu_q"], kv_len=s["kv_len"], positions=s["positions"],
                              tok_seq=s["tok_seq"], cache_rows=s["cache_rows"], status=s["status"])
        if case["release"]:
            kernels.blocks_release(s["slots"], s["tables"], s["held"], s["free"], s["free_count"], status=s["status"])
        return _tables_out(s)
    cache = (s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
    if kind == "attend":
        out = torch.empty_like(s["q"])
        kernels.attention_kv8(s["q"], out, s["cu_q"], s["kv_len"], s["slots"], s["tables"], *cache, n_kv=case["n_kv"],
                              group=case["group"], head_dim=case["dim"], scale=case["scale"], cap=case["cap"], window=case["window"],
                              ring=case["ring"], batch=len(s["lens"]), max_q_len=max(s["new"]), max_kv_len=max(s["lens"]))
        return out
    if kind == "append":
        kernels.kv8_write(s["k"], s["v"], s["cu_q"], s["positions"], s["cache_rows"], *cache, max_q_len=max(s["new"]))
    k = torch.empty((s["rows"], case["n_kv"], case["dim"]), dtype=TYPES[case["type"]], device=DEV)
    v = torch.empty_like(k)
    kernels.kv8_read(s["cu_r"], s["kv_len"], s["slots"], s["tables"], *cache, k, v, ring=case["ring"], max_q_len=s["longest"])
    return k, v


def _tables_out(s):
    return {n: s[n] for n in ("cu_q", "kv_len", "positions", "tok_seq", "cache_rows", "status", "tables", "held", "free_count", "free")}


def _run_plain(s):
    kind = s["case"]["kind"]
    if kind == "tables":
        _extend_plain(s)
        if s["case"]["release"]:
            _release_plain(s)
        return _tables_out(s)
    if kind == "attend":
        return _attend_plain(s)
    if kind == "append":
        _write_plain(s, s["k"], s["k_pages"], s["k_scale"])
        _write_plain(s, s["v"], s["v_pages"], s["v_scale"])
    return _read_plain(s, s["k_pages"], s["k_scale"]), _read_plain(s, s["v_pages"], s["v_scale"])


def _extend_plain(s):
    """(These requests always fit; a step that does not fit changes nothing and says so in ``status``.)"""
    P, R = s["case"]["block"], s["case"]["ring"]
    slots = s["slots"].long()
    after = s["lengths"] + s["new"]
    need = ((after.clamp(max=R) if R else after) + P - 1) // P
    had = s["held"][slots]
    extra = (need - had).clamp_(min=0)
    first = torch.cumsum(extra, 0) - extra
    W = s["tables"].shape[1]
    cols = torch.arange(W, device=DEV)[None, :]
    fresh = (cols >= had[:, None]) & (cols < need[:, None])
    pick = (s["free_count"] - 1 - (first[:, None] + cols - had[:, None])).clamp_(0, s["free"].numel() - 1)
    rows = torch.where(fresh, s["free"][pick.long()], s["tables"][slots])
    s["tables"][slots] = rows
    s["held"][slots] = torch.maximum(had, need)
    s["free_count"].sub_(extra.sum())
    ends = torch.cumsum(s["new"], 0)
    s["cu_q"][1:] = ends
    s["cu_q"][:1] = 0
    s["kv_len"].copy_(after)
    T = s["positions"].numel()
    t = torch.arange(T, device=DEV)
    seq = torch.searchsorted(ends, t, right=True)
    pos = s["lengths"][seq] + t - s["cu_q"][seq]
    place = pos % R if R else pos
    at = rows[seq, place // P] * P + place % P
    if R:
        at = torch.where(pos // P + R // P > (after[seq] - 1) // P, at, -1)
    s["positions"].copy_(pos)
    s["tok_seq"].copy_(seq)
    s["cache_rows"].copy_(at)
    s["status"].zero_()


def _release_plain(s):
    slots = s["slots"].long()
    had = s["held"][slots]
    W = s["tables"].shape[1]
    # the last request's last block goes back first
    cols = torch.arange(W - 1, -1, -1, device=DEV)
    rows = s["tables"][slots].flip(0, 1)
    mine = cols[None, :] < had.flip(0)[:, None]
    back = torch.cumsum(mine.reshape(-1), 0) - 1 + s["free_count"]
    keep = torch.where(mine.reshape(-1), back, s["free"].numel())
    longer = torch.cat([s["free"], s["free"].new_zeros(1)])
    longer[keep.long()] = torch.where(mine, rows, 0).reshape(-1)
    s["free"].copy_(longer[:-1])
    s["free_count"].add_(had.sum())
    s["held"][slots] = 0
    s["status"].zero_()


def _write_plain(s, x, pages, scales):
    """New rows x [tokens, kv heads, entries] into the blocks."""
    P = pages.shape[2]
    keep = s["cache_rows"] >= 0
    at = torch.where(keep, s["cache_rows"], 0)
    block = at // P
    x = x.to(F32)
    N, G = scales.shape
    # the largest number that every block and head gets, and whether the block is begun anew
    most = torch.where(keep[:, None], x.abs().amax(dim=2), 0.0)
    amax = torch.zeros_like(scales).scatter_reduce_(0, block.long()[:, None].expand(-1, G), most, "amax")
    begun = torch.zeros(N, device=DEV).scatter_reduce_(0, block.long(), (keep & (at % P == 0)).to(F32), "amax") > 0
    got = torch.zeros(N, device=DEV).scatter_reduce_(0, block.long(), keep.to(F32), "amax") > 0
    m, e = torch.frexp(amax)
    fit = torch.ldexp(torch.ones_like(amax), torch.where(m <= 127.0 / 128.0, e - 7, e - 6).clamp_(min=-126))
    fit = torch.where(torch.isfinite(amax), fit, float("nan"))
    new = torch.where(begun[:, None], fit, torch.maximum(fit, scales))
    new = torch.where(got[:, None], new, scales)
    # what was there is rounded to the scale that grew
    grew = (new != scales) & ~begun[:, None] & got[:, None]
    ratio = torch.where(grew, scales / new, 1.0)
    touched = grew.any(dim=1).nonzero()[:, 0]
    pages[touched] = (pages[touched].to(F32) * ratio[touched][:, :, None, None]).round().to(torch.int8)
    scales.copy_(new)
    q = (x / new[block.long()][:, :, None]).round().to(torch.int8)
    t = keep.nonzero()[:, 0]
    pages[block.long()[t], :, (at % P).long()[t]] = q[t]


def _places(s, i, first, last):
    """(block, place in it) of positions first..last-1 of sequence i."""
    P, R = s["case"]["block"], s["case"]["ring"]
    pos = torch.arange(first, last, device=DEV)
    place = pos % R if R else pos
    return pos, s["tables"][i][place // P].long(), place % P


def _read_plain(s, pages, scales):
    out = []
    for i, n in enumerate(s["lens"]):
        _, b, at = _places(s, i, _first_kept(n, s["case"]["block"], s["case"]["ring"]), n)
        out.append(pages[b, :, at].to(F32) * scales[b][:, :, None])
    return torch.cat(out).to(TYPES[s["case"]["type"]])


def _attend_plain(s):
    case = s["case"]
    G, g, D, W, cap = case["n_kv"], case["group"], case["dim"], case["window"], case["cap"]
    out = torch.empty_like(s["q"])
    row0 = 0
    for i, (n, m) in enumerate(zip(s["lens"], s["new"])):
        lo = max(0, n - m - W + 1) if W else 0
        pos, b, at = _places(s, i, lo, n)
        k = (s["k_pages"][b, :, at].to(F32) * s["k_scale"][b][:, :, None]).transpose(0, 1)          # [G, keys, D]
        v = (s["v_pages"][b, :, at].to(F32) * s["v_scale"][b][:, :, None]).transpose(0, 1)
        step = max(1, (1 << 28) // (G * g * (n - lo)))
        for a in range(0, m, step):
            c = min(m, a + step)
            q = s["q"][row0 + a:row0 + c].to(F32).view(c - a, G, g, D).permute(1, 0, 2, 3).reshape(G, (c - a) * g, D)
            z = torch.matmul(q, k.transpose(1, 2)) * case["scale"]
            if cap > 0:
                z = cap * torch.tanh(z / cap)
            at_q = torch.arange(n - m + a, n - m + c, device=DEV).repeat_interleave(g)[:, None]
            sees = pos[None, :] <= at_q
            if W:
                sees = sees & (at_q - pos[None, :] < W)
            z = z.masked_fill(~sees, float("-inf"))
            z = torch.exp(z - z.amax(dim=2, keepdim=True))
            o = torch.matmul(z, v) / z.sum(dim=2, keepdim=True)
            out[row0 + a:row0 + c] = o.view(G, c - a, g, D).permute(1, 0, 2, 3).reshape(c - a, G * g * D).to(out.dtype)
        row0 += m
    return out


# --- the work of a pass ------------------------------------------------------------------------------------------------
def _pairs(n, m, window):
    """(token, key) pairs that the last m tokens of n see, and how many keys one of them sees."""
    pos = np.arange(n - m, n, dtype=np.int64)
    sees = np.minimum(pos + 1, window) if window else pos + 1
    return int(sees.sum()), n - (max(0, n - m - window + 1) if window else 0)


def work(case):
    kind, P, R = case["kind"], case["block"], case.get("ring", 0)
    if kind == "tables":
        before, new = _numbers(case["before"]), _numbers(case["new"])
        taken = sum(_need(a + b, P, R) - _need(a, P, R) for a, b in zip(before, new))
        n, T = len(before), sum(new)
        # slot, length, new and held in; lengths, sums and held out; three numbers a token; a block read and written
        return {"bytes": 4.0 * (4 * n + 3 * n + 3 * T + (4 if case["release"] else 2) * taken), "flops": 0.0}
    size = TYPES[case["type"]].itemsize
    row = case["n_kv"] * case["dim"]
    if kind == "attend":
        lens, new = _numbers(case["lens"]), _numbers(case["new"])
        seen = [_pairs(n, m, case["window"]) for n, m in zip(lens, new)]
        keys = sum(k for _, k in seen)
        q = sum(new) * row * case["group"] * size
        return {"bytes": float(2 * keys * row + 2 * q + 8 * case["n_kv"] * sum((k + P - 1) // P for _, k in seen)),
                "flops": 4.0 * row * case["group"] * sum(p for p, _ in seen)}
    before = _numbers(case["before"])
    new = _numbers(case["new"]) if kind == "append" else [0] * len(before)
    held = [n - _first_kept(n, P, R) for n in (a + b for a, b in zip(before, new))]
    kept = sum(min(n, h) for n, h in zip(new, held))
    write = kept * 2 * row * (size + 1)                      # read once, written once as 8 bits
    read = 2 * row * sum(held) * (1 + size)
    return {"bytes": float(write + read), "flops": float(2 * row * (2 * kept + sum(held)))}


# --- in 64 bits --------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "tables":
        return _exact_tables(s)
    if case["kind"] == "attend":
        if work(case)["flops"] > 2e12:
            return None
        return _exact_attend(s)
    P, R, G = case["block"], case["ring"], case["n_kv"]
    done = []
    for pages, scales, x in ((s["k_pages"], s["k_scale"], s.get("k")), (s["v_pages"], s["v_scale"], s.get("v"))):
        values = pages.to(F64) * scales.to(F64)[:, :, None, None]
        scales = scales.to(F64)
        if x is not None:
            rows = s["cache_rows"].cpu().numpy()
            start = 0
            for m in s["new"]:
                t = start
                while t < start + m:
                    if rows[t] < 0:
                        t += 1
                        continue
                    b, p = divmod(int(rows[t]), P)
                    n = min(P - p, start + m - t)
                    piece = x[t:t + n].to(F64).transpose(0, 1)                         # [G, n, D]
                    most = piece.abs().amax(dim=(1, 2)).clamp_(min=127.0 * 2.0 ** -126)
                    _, e = torch.frexp(most / 127.0)
                    # 2^(e-1) <= most / 127 < 2^e: the lower one only where it is reached exactly
                    step = torch.ldexp(torch.ones(G, dtype=F64, device=DEV), e)
                    step = torch.where(127.0 * step / 2 == most, step / 2, step)
                    if p:
                        step = torch.maximum(step, scales[b])
                        values[b, :, :p] = torch.round(values[b, :, :p] / step[:, None, None]) * step[:, None, None]
                    scales[b] = step
                    values[b, :, p:p + n] = torch.round(piece / step[:, None, None]) * step[:, None, None]
                    t += n
                start += m
        out = []
        for i, n in enumerate(s["lens"]):
            row = s["tables"][i].cpu().tolist()
            p = _first_kept(n, P, R)
            while p < n:
                place = p % R if R else p
                c = min(P - place % P, n - p)
                out.append(values[row[place // P], :, place % P:place % P + c].transpose(0, 1))
                p += c
        done.append(torch.cat(out))
    return tuple(done)


def _exact_tables(s):
    """By hand, one block at a time."""
    case = s["case"]
    P, R = case["block"], case["ring"]
    h = {n: s[n].cpu().numpy().astype(np.int64) for n in ("slots", "lengths", "new", "tables", "held", "free", "free_count")}
    count = int(h["free_count"][0])
    cu, positions, seqs, rows = [0], [], [], []
    for i, slot in enumerate(h["slots"]):
        n = int(h["lengths"][i] + h["new"][i])
        while h["held"][slot] < _need(n, P, R):
            count -= 1
            h["tables"][slot, h["held"][slot]] = h["free"][count]
            h["held"][slot] += 1
        pos = np.arange(h["lengths"][i], n)
        place = pos % R if R else pos
        at = h["tables"][slot][place // P] * P + place % P
        rows.append(np.where(pos >= _first_kept(n, P, R), at, -1))
        positions.append(pos)
        seqs.append(np.full(len(pos), i))
        cu.append(cu[-1] + len(pos))
    if case["release"]:
        for slot in h["slots"][::-1]:
            while h["held"][slot] > 0:
                h["held"][slot] -= 1
                h["free"][count] = h["tables"][slot, h["held"][slot]]
                count += 1
    ints = lambda a: torch.from_numpy(np.asarray(a, dtype=np.int32)).to(DEV)
    return {"cu_q": ints(cu), "kv_len": ints(h["lengths"] + h["new"]), "positions": ints(np.concatenate(positions)),
            "tok_seq": ints(np.concatenate(seqs)), "cache_rows": ints(np.concatenate(rows)), "status": ints([0]),
            "tables": ints(h["tables"]), "held": ints(h["held"]), "free_count": ints([count]), "free": ints(h["free"])}


def _exact_attend(s):
    case = s["case"]
    G, g, D, P, R = case["n_kv"], case["group"], case["dim"], case["block"], case["ring"]
    out = torch.empty(s["q"].shape, dtype=F64, device=DEV)
    heads = s["q"].to(F64).view(-1, G * g, D)
    row0 = 0
    for i, (n, m) in enumerate(zip(s["lens"], s["new"])):
        key = torch.arange(n, device=DEV)
        place = torch.remainder(key, R) if R else key
        where = s["tables"][i].index_select(0, torch.div(place, P, rounding_mode="floor")).long()
        inside = torch.remainder(place, P)
        for h in range(G * g):
            k = s["k_pages"][:, h // g][where, inside].to(F64).mul_(s["k_scale"][where, h // g].to(F64)[:, None])
            v = s["v_pages"][:, h // g][where, inside].to(F64).mul_(s["v_scale"][where, h // g].to(F64)[:, None])
            for a in range(0, m, 1024):
                c = min(m, a + 1024)
                z = (heads[row0 + a:row0 + c, h] @ k.T) * case["scale"]
                if case["cap"]:
                    z = torch.tanh(z / case["cap"]) * case["cap"]
                back = torch.arange(n - m + a, n - m + c, device=DEV)[:, None] - key[None, :]
                seen = (back >= 0) & (back < (case["window"] or n + 1))
                w = torch.softmax(torch.where(seen, z, float("-inf")), dim=1)
                out[row0 + a:row0 + c].view(c - a, G * g, D)[:, h] = w @ v
        row0 += m
    return out
