"""Python face of the 8-bit cache: block tables built on the device, blocks written, read and attended to.

A cache layer is four tensors: ``k_pages`` and ``v_pages``, int8 [blocks, kv heads, tokens of a block, head_dim], and
``k_scale`` and ``v_scale``, float32 [blocks, kv heads].  A number q of a block stands for ``q * scale``; the scale is the
least power of two (2^-126 at least) under which nothing that the block of that head was given is beyond 127.  A scale
never shrinks while its block fills; when it grows, the numbers that were there are rounded to it.  A block that gets a
number that is not finite has the scale NaN, and all that sees it gets NaN, until it is begun anew.  Blocks hold 32, 64 or
another multiple of 32 tokens, up to 256; heads have a multiple of 16 entries, up to 256.

A sequence (a *slot*) holds a row of ``tables``, the ids of its blocks in the order of their places.  Position p lives at
place p, or, with ``ring`` (a multiple of the block), at ``p % ring``: the newest ``ring / block`` blocks are then kept, the
one that is being filled among them, so a window of W keys under steps of up to n tokens needs
``ring >= W + n + block - 2``.

The functions launch on the current stream, like all of this package; they wait for nothing and keep nothing.  Ids that
come from the device (slots, block ids, cache rows) and lie outside the tensors are passed over, never followed.
"""
from __future__ import annotations

import functools
import struct
from ctypes import c_char_p, c_int
from typing import Optional

import torch

from . import KernelError, _check, _fn, _sms, device_sms, library_loaded, load_library

# what the tables' status word says
BLOCKS_STATUS = {0: "ok", 1: "too few free blocks (or a stack that does not fit)", 2: "a row of the tables is too narrow",
                 3: "the step has more tokens than the outputs have places",
                 4: "a slot is out of range or named twice, or a length is negative"}

_I8, _I32, _F32 = torch.int8, torch.int32, torch.float32
_CODES = {torch.float32: 0, torch.bfloat16: 1}

# A call of these operators is a few microseconds on the device, so what the host does for it counts.  Their launchers take
# one struct, packed here as C lays it out (converting a pointer and 35 numbers one by one costs ctypes 3.4 us a call,
# packing them 0.4 and passing the one pointer 0.3), and the checks of the arguments are one expression each; which of
# them failed is found out only then.
_EXTEND = struct.Struct("@15P8i")
_RELEASE = struct.Struct("@8P4i")
_WRITE = struct.Struct("@10P4q8i")
_READ = struct.Struct("@11P4q11i")
_ATTN = struct.Struct("@14P17i2f")
_ATTN_TC = struct.Struct("@13P16i2f")
_functions: dict = {}
# (a call gets here with tensors of the device, so that there is one has been found out)
_raw_stream, _device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice
_NO_CPU = "brolm_b200 kernels run on CUDA tensors only; there is no CPU path"


def _call(lib: str, name: str, packed: bytes, what: str) -> None:
    f = _functions.get(name)
    if f is None:
        f = _functions[name] = _fn(lib, name, [c_char_p])
    _check(f(packed), what)


def _refuse_ints(what: str, **named) -> None:
    """Raise for the first of ``name=(tensor, entries or None)`` that is not a contiguous int32 tensor on the device."""
    for name, (t, n) in named.items():
        if t.dtype != _I32 or not t.is_contiguous():
            raise KernelError(f"{what}: {name} must be a contiguous int32 tensor")
        if n is not None and t.numel() != n:
            raise KernelError(f"{what}: {name} has {t.numel()} entries, not {n}")
        if not t.is_cuda:
            raise KernelError(_NO_CPU)


def _odd_ints(t: torch.Tensor, n: int) -> bool:
    return t.dtype is not _I32 or t.numel() != n or not t.is_contiguous() or not t.is_cuda


def blocks_extend(slots: torch.Tensor, lengths: torch.Tensor, new: torch.Tensor, tables: torch.Tensor, held: torch.Tensor,
                  free: torch.Tensor, free_count: torch.Tensor, *, block: int, cu_q: torch.Tensor, kv_len: torch.Tensor,
                  positions: torch.Tensor, tok_seq: torch.Tensor, cache_rows: torch.Tensor, status: torch.Tensor,
                  ring: int = 0, settle: bool = False, refused: Optional[torch.Tensor] = None) -> None:
    """A step's block tables and slot map, on the device.  All tensors are int32.

    Row i of the step goes on with slot ``slots[i]`` (-1: padding), which holds ``lengths[i]`` tokens, by ``new[i]``.  The
    blocks that its tokens need beyond ``held[slot]`` come from the top of the stack ``free[:free_count]``, rows in order,
    and are entered behind those that ``tables[slot]`` holds.  Written: ``cu_q`` [rows + 1] (sums of ``new``), ``kv_len``
    [rows] (0 for padding), and for every token, rows back to back, ``positions``, ``tok_seq`` (its row) and ``cache_rows``
    (block * block size + place, -1 where the ring does not keep the token); places beyond the last token get -1, 0, -1.
    ``kv_len`` may be ``lengths``, which then go on in place; the other outputs are tensors of their own.

    ``settle``: kernels launched behind this call may read what it writes (all but the tables and ``cache_rows``, which are
    read after the wait) before they wait for the launch before them; the kernels of this package that read a step's
    positions, sums and lengths do so, since the host used to write them.  It costs an empty launch.

    A step that does not fit changes neither ``tables``, ``held`` nor the stack: its outputs read as padding and ``status``
    holds a key of ``BLOCKS_STATUS``.  ``refused``, one number where given, then gets that key, too, unless it holds one:
    whoever queues steps without looking at each one's status finds the first refusal there, and sets it back to 0.  The
    same step again takes no more blocks.  Up to 4,096 rows and 65,536 slots."""
    what = "blocks_extend"
    n, T = slots.numel(), positions.numel()
    if tables.dim() != 2:
        raise KernelError(f"{what}: tables must be [slots, width]")
    S, W = tables.shape
    N = free.numel()
    if _odd_ints(slots, n) or _odd_ints(lengths, n) or _odd_ints(new, n) or _odd_ints(tables, S * W) or _odd_ints(held, S) or \
            _odd_ints(free, N) or _odd_ints(free_count, 1) or _odd_ints(cu_q, n + 1) or _odd_ints(kv_len, n) or \
            _odd_ints(positions, T) or _odd_ints(tok_seq, T) or _odd_ints(cache_rows, T) or _odd_ints(status, 1) or \
            (refused is not None and _odd_ints(refused, 1)):
        _refuse_ints(what, slots=(slots, n), lengths=(lengths, n), new=(new, n), tables=(tables, None), held=(held, S), free=(free, N),
                     free_count=(free_count, 1), cu_q=(cu_q, n + 1), kv_len=(kv_len, n), positions=(positions, T),
                     tok_seq=(tok_seq, T), cache_rows=(cache_rows, T), status=(status, 1),
                     refused=(status if refused is None else refused, 1))
    _call("blocks", "brolm_blocks_extend", _EXTEND.pack(
        slots.data_ptr(), lengths.data_ptr(), new.data_ptr(), tables.data_ptr(), held.data_ptr(), free.data_ptr(),
        free_count.data_ptr(), cu_q.data_ptr(), kv_len.data_ptr(), positions.data_ptr(), tok_seq.data_ptr(),
        cache_rows.data_ptr(), status.data_ptr(), 0 if refused is None else refused.data_ptr(), _raw_stream(_device()), n, S, W, N, block,
        ring, T, 1 if settle else 0), what)


def blocks_release(slots: torch.Tensor, tables: torch.Tensor, held: torch.Tensor, free: torch.Tensor, free_count: torch.Tensor, *,
                   status: torch.Tensor, refused: Optional[torch.Tensor] = None) -> None:
    """Give the blocks of ``slots`` (-1: left out) back to the stack, the last row's last block first, so that releasing
    the rows of an extend restores the order it found.  ``status`` and ``refused`` as in ``blocks_extend``; a wrong slot
    changes nothing."""
    what = "blocks_release"
    if tables.dim() != 2:
        raise KernelError(f"{what}: tables must be [slots, width]")
    S, W = tables.shape
    n, N = slots.numel(), free.numel()
    if _odd_ints(slots, n) or _odd_ints(tables, S * W) or _odd_ints(held, S) or _odd_ints(free, N) or _odd_ints(free_count, 1) or \
            _odd_ints(status, 1) or (refused is not None and _odd_ints(refused, 1)):
        _refuse_ints(what, slots=(slots, n), tables=(tables, None), held=(held, S), free=(free, N), free_count=(free_count, 1),
                     status=(status, 1), refused=(status if refused is None else refused, 1))
    _call("blocks", "brolm_blocks_release", _RELEASE.pack(
        slots.data_ptr(), tables.data_ptr(), held.data_ptr(), free.data_ptr(), free_count.data_ptr(), status.data_ptr(),
        0 if refused is None else refused.data_ptr(), _raw_stream(_device()), n, S, W, N), what)


def _cache(what: str, k_pages, v_pages, k_scale, v_scale) -> tuple:
    shape = k_pages.shape
    if len(shape) != 4 or k_pages.dtype is not _I8 or v_pages.dtype is not _I8:
        raise KernelError(f"{what}: the pages must be int8 [blocks, kv heads, block, head_dim]")
    if v_pages.shape != shape or not k_pages.is_contiguous() or not v_pages.is_contiguous():
        raise KernelError(f"{what}: key and value pages must be contiguous and of one shape")
    n_blocks, n_kv, _, _ = shape
    scales = (n_blocks, n_kv)
    if k_scale.dtype is not _F32 or v_scale.dtype is not _F32 or k_scale.shape != scales or v_scale.shape != scales or \
            not k_scale.is_contiguous() or not v_scale.is_contiguous():
        raise KernelError(f"{what}: the scales must be contiguous float32 [blocks, kv heads]")
    return shape


def _two(what: str, names: str, a: torch.Tensor, b: torch.Tensor, n_kv: int, dim: int) -> tuple:
    """(tokens, element type code, strides of both) of two tensors [tokens, n_kv, dim] of one element type."""
    dt = a.dtype
    sa, sb = a.stride(), b.stride()
    shape = a.shape
    if len(shape) != 3 or b.shape != shape or shape[1] != n_kv or shape[2] != dim or sa[2] != 1 or sb[2] != 1:
        raise KernelError(f"{what}: {names} must be [tokens, {n_kv}, {dim}], as many tokens both, with rows of consecutive entries")
    if b.dtype is not dt or dt not in _CODES:
        raise KernelError(f"{what}: {names} must both be float32 or both bfloat16, not {dt} and {b.dtype}")
    return shape[0], _CODES[dt], sa[0], sa[1], sb[0], sb[1]


def kv8_write(k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, positions: torch.Tensor, cache_rows: torch.Tensor,
              k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, *,
              max_q_len: int) -> None:
    """New keys and values ``k``, ``v`` [tokens, kv heads, head_dim] (float32 or bfloat16, any strides between tokens and
    heads) into the cache, at ``cache_rows`` (``blocks_extend``).  ``cu_q`` says where the step's rows begin, ``positions``
    where their first tokens lie (-1: padding, not written); ``max_q_len``: no row brings more tokens than that.  The tokens
    that go to one block take its scale together; a block whose first place is among them is begun anew."""
    what = "kv8_write"
    n_blocks, n_kv, block, dim = _cache(what, k_pages, v_pages, k_scale, v_scale)
    T, code, k0, k1, v0, v1 = _two(what, "k and v", k, v, n_kv, dim)
    rows = cu_q.numel() - 1
    if max_q_len < 1 or rows < 0:
        raise KernelError(f"{what}: max_q_len and the entries of cu_q must be at least 1")
    if not (k.is_cuda and v.is_cuda and k_pages.is_cuda and v_pages.is_cuda and k_scale.is_cuda and v_scale.is_cuda):
        raise KernelError(_NO_CPU)
    if _odd_ints(cu_q, rows + 1) or _odd_ints(positions, T) or _odd_ints(cache_rows, T):
        _refuse_ints(what, cu_q=(cu_q, None), positions=(positions, T), cache_rows=(cache_rows, T))
    _call("kv8", "brolm_kv8_write", _WRITE.pack(
        k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), positions.data_ptr(), cache_rows.data_ptr(), k_pages.data_ptr(),
        v_pages.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), _raw_stream(_device()), k0, v0, k1, v1, code, T, rows, n_kv, dim, block,
        n_blocks, max_q_len), what)


def kv8_read(cu_q: torch.Tensor, kv_len: torch.Tensor, slots: torch.Tensor, tables: torch.Tensor, k_pages: torch.Tensor,
             v_pages: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor, *,
             max_q_len: int, ring: int = 0) -> None:
    """The newest ``cu_q[i + 1] - cu_q[i]`` tokens of every row as numbers: ``k_out``, ``v_out`` [tokens, kv heads,
    head_dim], float32 or bfloat16 (both hold them exactly), on 16 bytes, with strides between tokens and heads that are
    multiples of 16 bytes.  Tokens before a sequence's first, that the ring no longer holds, or that come before the row's
    newest ``max_q_len``, read as zero."""
    what = "kv8_read"
    n_blocks, n_kv, block, dim = _cache(what, k_pages, v_pages, k_scale, v_scale)
    T, code, k0, k1, v0, v1 = _two(what, "k_out and v_out", k_out, v_out, n_kv, dim)
    rows = cu_q.numel() - 1
    if tables.dim() != 2 or max_q_len < 1 or rows < 0:
        raise KernelError(f"{what}: tables must be [slots, width], max_q_len and the entries of cu_q at least 1")
    S, W = tables.shape
    if not (k_out.is_cuda and v_out.is_cuda and k_pages.is_cuda and v_pages.is_cuda and k_scale.is_cuda and v_scale.is_cuda):
        raise KernelError(_NO_CPU)
    if _odd_ints(cu_q, rows + 1) or _odd_ints(kv_len, rows) or _odd_ints(slots, rows) or _odd_ints(tables, S * W):
        _refuse_ints(what, cu_q=(cu_q, None), kv_len=(kv_len, rows), slots=(slots, rows), tables=(tables, None))
    _call("kv8", "brolm_kv8_read", _READ.pack(
        cu_q.data_ptr(), kv_len.data_ptr(), slots.data_ptr(), tables.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
        k_scale.data_ptr(), v_scale.data_ptr(), k_out.data_ptr(), v_out.data_ptr(), _raw_stream(_device()), k0, v0, k1, v1, code, T, rows, n_kv,
        dim, block, n_blocks, S, W, ring, max_q_len), what)


KV8_TILE, KV8_WARPS, KV8_CLUSTER = 32, 4, 8       # keys of a tile, warps of a block, blocks that join their results themselves
KV8_DEALT = 128                                   # sequences of a launch whose clusters are dealt out by length


@functools.lru_cache(maxsize=256)
def kv8_shares(batch: int, n_kv: int, row_tiles: int, keys: int, head_dim: int, sms: int, many: bool = False,
               per_sm: int = 3) -> tuple[int, int]:
    """How many blocks share the keys of one (sequence, kv head, tile of query rows): (blocks of a cluster, clusters), or
    (blocks of a cluster, -n): n clusters of a (kv head, tile of query rows) are dealt out over the sequences by their lengths
    on the device.  ``many``: more than eight query rows of a kv head, whose tiles take twice as long.

    Two blocks run on an SM (``per_sm`` of heads of up to 64 entries), and there are as many shares as give every SM its blocks,
    but none whose four warps would not have a tile of keys each.  A cluster lies inside one group of SMs, so clusters of
    three to eight leave up to an eighth of the places empty; where one too many is asked for, it runs alone at the end (48
    items of 2,000 keys, float32: 28.6 us as 6 x 1, of which 45 fit, 19.7 as 5 x 1; 12 of 4,000 at 4 kv heads of 256, one
    query row each: 35.8 and 23.3).  Up to eight join their results inside the launch; more are joined by a second one, which
    pays from about 100 tiles on where eight shares leave SMs without a block (1 sequence of 8,192 keys, 4 kv heads of 256:
    18.3 us as 8 x 1, 11.1 as 8 x 8; 2 of 2,000: 8.6 as 8 x 1, 10.2 as 8 x 2; 24 items of 4,000, float32, heads of 64: 12.9 as
    8 x 1, 20.8 as 8 x 2).

    Where the longest sequence's warps would have more than eight tiles each, what counts is that sequence, and dealing pays:
    24 sequences of 100 to 4,000 keys, 4 kv heads of 256, 32.5 us as 3 x 1, 18.3 dealt; 16 of 129 to 6,145 under a window of
    4,096, 8 kv heads, 33 and 26.5; 4 of 1,000 to 12,000, 4 kv heads, 21.8 and 17.2.  It costs 1.5 to 2.5 us (finding out, and
    the second launch) where all are equally long (24 of 3,000, 8 kv heads of 128: 35.0 and 37.9), and more than it brings
    where there are few clusters to deal (48 sequences of 3,000 on 74: 57.9 and 64.7).  What is dealt out is one round of
    blocks (two rounds: 24.2 us for the first), in clusters of so many that a sequence has about eight parts to join.

    With more sequences, where an item would have no more than two shares, the longest ones' blocks would run alone at the
    end: such steps are cut into rounds of blocks that the SMs take as they come free, if the shares stay long enough (24
    tiles) and fill their rounds (40 sequences of 100 to 3,000 keys, 8 kv heads: 52.9 us as 1 x 1, 43.7 as 1 x 2)."""
    places = (per_sm if head_dim <= 64 else 2) * sms
    heads = n_kv * row_tiles
    items = max(1, batch * heads)
    tiles = max(1, -(-keys // KV8_TILE))

    def fit(cluster):                             # clusters of a (kv head, tile of rows) that run at a time
        return (places if cluster <= 2 else places * 7 // 8) // (cluster * heads)
    want = min(places // items, -(-tiles // KV8_WARPS))
    if want > 2:
        want = max(2, min(want, places * 7 // 8 // items))
    if batch > 1 and tiles * (2 if many else 1) > 8 * KV8_WARPS * max(1, min(want, KV8_CLUSTER)):
        for cluster in (1, 2, 4, 8):
            if fit(cluster) <= 8 * batch or cluster == 8:
                break
        if batch <= KV8_DEALT and fit(cluster) >= 1.5 * batch:
            return cluster, -fit(cluster)
    if want <= 2:
        if batch > 1 and items < 4 * places:
            for k in (2, 3, 4):
                rounds = k * items / places
                if rounds > 1.5 and tiles >= 24 * k and rounds >= 0.8 * -(-k * items // places):
                    return 1, k
        return max(1, want), 1
    if want <= KV8_CLUSTER:
        return want, 1
    return KV8_CLUSTER, (want // KV8_CLUSTER if tiles >= 96 and items * KV8_CLUSTER < sms else 1)


def _parts(n: int, head_dim: int, device, plans: int = 0) -> tuple:
    """Room for n parts of rows and for ``plans`` pairs of whole numbers: the tensor that holds it, and where the sums, their
    (maximum, weight) and the pairs begin."""
    parts = torch.empty(n * (head_dim + 2) + 2 * plans, dtype=_F32, device=device)
    at = parts.data_ptr()
    return parts, at, at + 4 * n * head_dim, at + 4 * n * (head_dim + 2)


@functools.lru_cache(maxsize=256)
def kv8_tc_spans(tokens: int, batch: int, n_kv: int, group: int, max_q_len: int, keys: int, head_dim: int, sms: int) -> tuple[int, int]:
    """How many of the tiles of 128 query rows have a block each on tcgen05, and how many blocks share the keys of each of the
    others: one block runs on an SM, so what counts is how many rounds of blocks there are and how long a block's share is.
    In tiles of 128 keys (about 2.6 us each at 256 entries, counted as 3): a block begins and ends in three, and joining costs another three and
    what the parts take to memory and back.  Where the last round would be far from full, its tiles alone are shared
    (on 14,336 keys, 8 kv heads of 256, two query heads each, us with a block for a tile / four / the last round's
    shared as the rule has it: 1,280 tokens, 160 tiles on 148 SMs, 570 / 453 / 351 by 12; 1,700, 216 tiles, 571 / 555 / 470 by 2;
    2,048, 256 tiles, 569 / 655 / 580 by 4).  The model is 2 % off in the last of these: where the last round is three quarters
    full, a block a tile is as good or a little better, and it counts what sharing costs too low."""
    items = batch * n_kv * -(-max_q_len * group // 128)
    tiles = -(-keys // 128)
    traffic = tokens * n_kv * group * head_dim * 8 / 6.5e12 / (3e-6 * head_dim / 256)

    def cost(choice):
        whole, k = choice
        t = -(-whole // sms) * (tiles + 3)
        if k > 1:
            t += -(-(items - whole) * k // sms) * (-(-tiles // k) + 3) + 3 + k * traffic * (items - whole) / items
        return t
    most = min(32, tiles // 2)
    full = items // sms * sms
    choices = [(items, 1)] + [(0, k) for k in range(2, most + 1)]
    if tokens == batch * max_q_len and 0 < full < items:
        choices += [(full, k) for k in range(2, most + 1)]
    return min(choices, key=cost)


# From how many rows of a kv head (tokens x query heads), and from how many of rows x kv heads x keys x entries (64 at least),
# a step of bfloat16 runs on tcgen05, whose blocks take 128 rows and heads of 64, 128 or 256 entries, smaller ones filled up
# with zeros.  8 kv heads, two query heads each, us on mma.sync / tcgen05.  256 entries: 32 tokens on 1,000 keys (1.3e8) 14.6 /
# 19.1, 128 on 300 (1.6e8) 18.0 / 21.7, 16 on 4,096 (2.7e8) 20.6 / 20.8, 64 on 4,096 (1.1e9) 40.1 / 26.9, 4 x 64 on 1,000
# (1.0e9) 40.0 / 28.5, 1,024 on 8,192 (3.4e10) 803 / 179, and of 192 736 / 178, of 96 472 / 157, of 32 343 / 137.
KV8_TC_ROWS, KV8_TC_WORK = 32, 2.5e8


def attention_kv8_tc_status(reset: bool = False) -> int:
    """0 if no bounded wait inside the tcgen05 attention over the 8-bit cache ever ran out; otherwise its code.  Synchronises."""
    if not library_loaded("attn_kv8_tc"):
        return 0                   # its kernels never ran: nothing is built or loaded for the question
    f = load_library("attn_kv8_tc").brolm_attn_kv8_tc_status
    f.argtypes = [c_int]
    f.restype = c_int
    return f(1 if reset else 0)


def attention_kv8(q: torch.Tensor, out: torch.Tensor, cu_q: torch.Tensor, kv_len: torch.Tensor, slots: torch.Tensor,
                  tables: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, *, n_kv: int, group: int, head_dim: int, scale: float, cap: float, window: int,
                  ring: int, batch: int, max_q_len: int, max_kv_len: int) -> None:
    """The newest ``cu_q[i + 1] - cu_q[i]`` tokens of every row i against the ``kv_len[i]`` that its slot holds, themselves
    among them (``kv8_write`` comes first).  ``q`` and ``out`` [tokens, n_kv * group * head_dim], float32 or bfloat16, query
    head h reads kv head h // group; ``scale``, ``cap`` (<= 0: none) and ``window`` (0: all keys) as everywhere.  A token
    that sees no key (a padding row's) gets zeros; places of ``out`` that are no row's (all of them, behind a step that the
    tables refused) stay as they are.  ``max_q_len`` and ``max_kv_len`` bound the rows' new tokens and lengths."""
    what = "attention_kv8"
    n_blocks, G, block, dim = _cache(what, k_pages, v_pages, k_scale, v_scale)
    if G != n_kv or dim != head_dim:
        raise KernelError(f"{what}: the pages hold {G} heads of {dim}, not {n_kv} of {head_dim}")
    shape, dt = q.shape, q.dtype
    q0, o0 = q.stride(), out.stride()
    if len(shape) != 2 or shape[1] != n_kv * group * head_dim or out.shape != shape or q0[1] != 1 or o0[1] != 1:
        raise KernelError(f"{what}: q and out must be [tokens, {n_kv * group * head_dim}] with rows of consecutive entries")
    if out.dtype is not dt or dt not in _CODES:
        raise KernelError(f"{what}: q and out must both be float32 or both bfloat16, not {dt} and {out.dtype}")
    if tables.dim() != 2 or max_q_len < 1:
        raise KernelError(f"{what}: tables must be [slots, width] and max_q_len at least 1")
    if ring and (window <= 0 or ring < window + max_q_len + block - 2):
        raise KernelError(f"{what}: a ring of {ring} does not keep what {max_q_len} new tokens see under a window of {window}: "
                          f"it takes window + tokens + {block} - 2")
    S, W = tables.shape
    if not (q.is_cuda and out.is_cuda and k_pages.is_cuda and v_pages.is_cuda and k_scale.is_cuda and v_scale.is_cuda):
        raise KernelError(_NO_CPU)
    if _odd_ints(cu_q, batch + 1) or _odd_ints(kv_len, batch) or _odd_ints(slots, batch) or _odd_ints(tables, S * W):
        _refuse_ints(what, cu_q=(cu_q, batch + 1), kv_len=(kv_len, batch), slots=(slots, batch), tables=(tables, None))
    T = shape[0]
    sms = _sms.get(_device()) or device_sms()
    rows = max_q_len * group
    keys = min(max_kv_len, window + max_q_len) if window > 0 else max_kv_len
    if rows >= KV8_TC_ROWS and dt is torch.bfloat16 and n_blocks * n_kv * block < 1 << 31 and \
            float(T) * group * n_kv * keys * max(head_dim, 64) >= KV8_TC_WORK:
        whole, spans = kv8_tc_spans(T, batch, n_kv, group, max_q_len, keys, head_dim, sms)
        part_o = part_ml = 0
        if spans > 1:
            parts, part_o, part_ml, _ = _parts((batch * n_kv * -(-rows // 128) - whole) * spans * 128, head_dim, q.device)
        _call("attn_kv8_tc", "brolm_attn_kv8_tc", _ATTN_TC.pack(
            q.data_ptr(), out.data_ptr(), cu_q.data_ptr(), kv_len.data_ptr(), slots.data_ptr(), tables.data_ptr(), k_pages.data_ptr(),
            v_pages.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), part_o, part_ml, _raw_stream(_device()), q0[0], o0[0], T, batch, n_kv, group,
            head_dim, block, n_blocks, S, W, ring, window, max_q_len, whole, spans, scale, cap), what)
        return
    shares, spans = kv8_shares(batch, n_kv, 1 if rows <= 8 else -(-rows // 16), keys, head_dim, sms, rows > 8,
                               3 if rows <= (4 if dt is _F32 else 8) else 2)
    part_o = part_ml = plan = 0
    if spans > 1:
        parts, part_o, part_ml, _ = _parts(T * n_kv * group * spans, head_dim, q.device)
    elif spans < 0:
        tile = 2 if rows <= 2 else 4 if rows <= 4 else 8 if rows <= 8 else 16
        parts, part_o, part_ml, plan = _parts(-spans * n_kv * -(-rows // tile) * tile, head_dim, q.device, T * n_kv * group)
    _call("attn_kv8", "brolm_attn_kv8", _ATTN.pack(
        q.data_ptr(), out.data_ptr(), cu_q.data_ptr(), kv_len.data_ptr(), slots.data_ptr(), tables.data_ptr(), k_pages.data_ptr(),
        v_pages.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), part_o, part_ml, plan, _raw_stream(_device()), q0[0], o0[0], _CODES[dt], T, batch,
        n_kv, group, head_dim, block, n_blocks, S, W, ring, window, max_q_len, shares, spans, scale, cap), what)
