"""Python face of the 8-bit cache: block tables built on the device, blocks written, read and attended to.

A cache layer is four tensors: ``k_pages`` and ``v_pages``, int8 [blocks, kv heads, tokens of a block, head_dim], and
``k_scale`` and ``v_scale``, float32 [blocks, kv heads].  A number q of a block stands for ``q * scale``; the scale is the
least power of two (2^-126 at least) under which nothing that the block of that head was given is beyond 127.  A scale
never shrinks while its block fills; when it grows, the numbers that were there are rounded to it.  A block that gets a
number that is not finite has the scale NaN, and all that sees it gets NaN, until it is begun anew.

A sequence (a *slot*) holds a row of ``tables``, the ids of its blocks in the order of their places.  Position p lives at
place p, or, with ``ring`` (a multiple of the block), at ``p % ring``: the newest ``ring / block`` blocks are then kept, the
one that is being filled among them, so a window of W keys under steps of up to n tokens needs
``ring >= W + n + block - 2``.

The functions launch on the current stream, like all of this package; they wait for nothing and keep nothing.  Ids that
come from the device (slots, block ids, cache rows) and lie outside the tensors are passed over, never followed.
"""
from __future__ import annotations

import struct
from ctypes import c_char_p, c_float, c_int, c_longlong, c_void_p
from typing import Optional

import torch

from . import KernelError, _check, _code, _fn, _ptr, _stream, device_sms

# what the tables' status word says
BLOCKS_STATUS = {0: "ok", 1: "too few free blocks (or a stack that does not fit)", 2: "a row of the tables is too narrow",
                 3: "the step has more tokens than the outputs have places",
                 4: "a slot is out of range or named twice, or a length is negative"}


# The launchers of these libraries take one struct, packed here as C lays it out: converting a pointer and 35 numbers
# one by one costs ctypes 3.4 us a call, packing them 0.4 and passing the one pointer 0.3.
_ATTN = struct.Struct("@13P17i2f")
_functions: dict = {}


def _call(lib: str, name: str, packed: bytes, what: str) -> None:
    f = _functions.get(name)
    if f is None:
        f = _functions[name] = _fn(lib, name, [c_char_p])
    _check(f(packed), what)


def _ints(what: str, *named) -> None:
    for name, t, n in named:
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise KernelError(f"{what}: {name} must be a contiguous int32 tensor")
        if n is not None and t.numel() != n:
            raise KernelError(f"{what}: {name} has {t.numel()} entries, not {n}")


def _state(what: str, tables, held, free, free_count) -> None:
    if tables.dim() != 2:
        raise KernelError(f"{what}: tables must be [slots, width]")
    _ints(what, ("tables", tables, None), ("held", held, tables.shape[0]), ("free", free, None), ("free_count", free_count, 1))


def blocks_extend(slots: torch.Tensor, lengths: torch.Tensor, new: torch.Tensor, tables: torch.Tensor, held: torch.Tensor,
                  free: torch.Tensor, free_count: torch.Tensor, *, block: int, cu_q: torch.Tensor, kv_len: torch.Tensor,
                  positions: torch.Tensor, tok_seq: torch.Tensor, cache_rows: torch.Tensor, status: torch.Tensor,
                  ring: int = 0) -> None:
    """A step's block tables and slot map, on the device.  All tensors are int32.

    Row i of the step goes on with slot ``slots[i]`` (-1: padding), which holds ``lengths[i]`` tokens, by ``new[i]``.  The
    blocks that its tokens need beyond ``held[slot]`` come from the top of the stack ``free[:free_count]``, rows in order,
    and are entered behind those that ``tables[slot]`` holds.  Written: ``cu_q`` [rows + 1] (sums of ``new``), ``kv_len``
    [rows] (0 for padding), and for every token, rows back to back, ``positions``, ``tok_seq`` (its row) and ``cache_rows``
    (block * block size + place, -1 where the ring does not keep the token); places beyond the last token get -1, 0, -1.

    A step that does not fit changes neither ``tables``, ``held`` nor the stack: its outputs read as padding and ``status``
    holds a key of ``BLOCKS_STATUS``.  The same step again takes no more blocks.  Up to 4,096 rows and 65,536 slots."""
    what = "blocks_extend"
    _state(what, tables, held, free, free_count)
    n, T = slots.numel(), positions.numel()
    _ints(what, ("slots", slots, None), ("lengths", lengths, n), ("new", new, n), ("cu_q", cu_q, n + 1), ("kv_len", kv_len, n),
          ("positions", positions, None), ("tok_seq", tok_seq, T), ("cache_rows", cache_rows, T), ("status", status, 1))
    f = _fn("blocks", "brolm_blocks_extend", [c_void_p] * 13 + [c_int] * 7 + [c_void_p])
    _check(f(_ptr(slots), _ptr(lengths), _ptr(new), _ptr(tables), _ptr(held), _ptr(free), _ptr(free_count), _ptr(cu_q), _ptr(kv_len),
             _ptr(positions), _ptr(tok_seq), _ptr(cache_rows), _ptr(status), n, tables.shape[0], tables.shape[1], free.numel(),
             block, ring, T, _stream()), what)


def blocks_release(slots: torch.Tensor, tables: torch.Tensor, held: torch.Tensor, free: torch.Tensor, free_count: torch.Tensor, *,
                   status: torch.Tensor) -> None:
    """Give the blocks of ``slots`` (-1: left out) back to the stack, the last row's last block first, so that releasing
    the rows of an extend restores the order it found.  ``status`` as in ``blocks_extend``; a wrong slot changes nothing."""
    what = "blocks_release"
    _state(what, tables, held, free, free_count)
    _ints(what, ("slots", slots, None), ("status", status, 1))
    f = _fn("blocks", "brolm_blocks_release", [c_void_p] * 6 + [c_int] * 4 + [c_void_p])
    _check(f(_ptr(slots), _ptr(tables), _ptr(held), _ptr(free), _ptr(free_count), _ptr(status), slots.numel(), tables.shape[0],
             tables.shape[1], free.numel(), _stream()), what)


def _cache(what: str, k_pages, v_pages, k_scale, v_scale) -> tuple:
    if k_pages.dim() != 4 or k_pages.dtype != torch.int8 or v_pages.dtype != torch.int8:
        raise KernelError(f"{what}: the pages must be int8 [blocks, kv heads, block, head_dim]")
    if v_pages.shape != k_pages.shape or not k_pages.is_contiguous() or not v_pages.is_contiguous():
        raise KernelError(f"{what}: key and value pages must be contiguous and of one shape")
    for s in (k_scale, v_scale):
        if s.dtype != torch.float32 or s.shape != k_pages.shape[:2] or not s.is_contiguous():
            raise KernelError(f"{what}: the scales must be contiguous float32 [blocks, kv heads]")
    return tuple(k_pages.shape)


def _rows3(what: str, name: str, x: torch.Tensor, n_kv: int, dim: int) -> None:
    if x.dim() != 3 or x.shape[1:] != (n_kv, dim) or x.stride(2) != 1:
        raise KernelError(f"{what}: {name} must be [tokens, {n_kv}, {dim}] with rows of consecutive entries")


def kv8_write(k: torch.Tensor, v: torch.Tensor, cu_q: torch.Tensor, positions: torch.Tensor, cache_rows: torch.Tensor,
              k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, *,
              max_q_len: int) -> None:
    """New keys and values ``k``, ``v`` [tokens, kv heads, head_dim] (float32 or bfloat16, any strides between tokens and
    heads) into the cache, at ``cache_rows`` (``blocks_extend``).  ``cu_q`` says where the step's rows begin, ``positions``
    where their first tokens lie (-1: padding, not written); ``max_q_len``: no row brings more tokens than that.  The tokens
    that go to one block take its scale together; a block whose first place is among them is begun anew."""
    what = "kv8_write"
    n_blocks, n_kv, block, dim = _cache(what, k_pages, v_pages, k_scale, v_scale)
    _rows3(what, "k", k, n_kv, dim)
    _rows3(what, "v", v, n_kv, dim)
    T = k.shape[0]
    if v.shape[0] != T or v.dtype != k.dtype:
        raise KernelError(f"{what}: k and v must have as many tokens and one element type")
    if max_q_len < 1:
        raise KernelError(f"{what}: max_q_len must be at least 1")
    _ints(what, ("cu_q", cu_q, None), ("positions", positions, T), ("cache_rows", cache_rows, T))
    f = _fn("kv8", "brolm_kv8_write", [c_void_p, c_longlong, c_longlong] * 2 + [c_int] + [c_void_p] * 7 + [c_int] * 7 + [c_void_p])
    _check(f(_ptr(k), k.stride(0), k.stride(1), _ptr(v), v.stride(0), v.stride(1), _code(k), _ptr(cu_q), _ptr(positions),
             _ptr(cache_rows), _ptr(k_pages), _ptr(v_pages), _ptr(k_scale), _ptr(v_scale), T, cu_q.numel() - 1, n_kv, dim, block,
             n_blocks, max_q_len, _stream()), what)


def kv8_read(cu_q: torch.Tensor, kv_len: torch.Tensor, slots: torch.Tensor, tables: torch.Tensor, k_pages: torch.Tensor,
             v_pages: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, k_out: torch.Tensor, v_out: torch.Tensor, *,
             max_q_len: int, ring: int = 0) -> None:
    """The newest ``cu_q[i + 1] - cu_q[i]`` tokens of every row (at most ``max_q_len`` of each) as numbers: ``k_out``,
    ``v_out`` [tokens, kv heads, head_dim], float32 or bfloat16 (both hold them exactly).  Tokens before a sequence's first,
    or that the ring no longer holds, read as zero."""
    what = "kv8_read"
    n_blocks, n_kv, block, dim = _cache(what, k_pages, v_pages, k_scale, v_scale)
    _rows3(what, "k_out", k_out, n_kv, dim)
    _rows3(what, "v_out", v_out, n_kv, dim)
    if v_out.shape[0] != k_out.shape[0] or v_out.dtype != k_out.dtype:
        raise KernelError(f"{what}: k_out and v_out must have as many tokens and one element type")
    rows = cu_q.numel() - 1
    if tables.dim() != 2 or max_q_len < 1:
        raise KernelError(f"{what}: tables must be [slots, width] and max_q_len at least 1")
    _ints(what, ("cu_q", cu_q, None), ("kv_len", kv_len, rows), ("slots", slots, rows), ("tables", tables, None))
    f = _fn("kv8", "brolm_kv8_read", [c_void_p] * 8 + [c_void_p, c_longlong, c_longlong] * 2 + [c_int] * 10 + [c_void_p])
    _check(f(_ptr(cu_q), _ptr(kv_len), _ptr(slots), _ptr(tables), _ptr(k_pages), _ptr(v_pages), _ptr(k_scale), _ptr(v_scale),
             _ptr(k_out), k_out.stride(0), k_out.stride(1), _ptr(v_out), v_out.stride(0), v_out.stride(1), _code(k_out),
             k_out.shape[0], rows, n_kv, dim, block, n_blocks, tables.shape[0], tables.shape[1], ring, _stream()), what)


KV8_TILE, KV8_WARPS, KV8_CLUSTER = 32, 4, 8       # keys of a tile, warps of a block, blocks that join their results themselves


def kv8_shares(batch: int, n_kv: int, row_tiles: int, keys: int, sms: Optional[int] = None) -> tuple[int, int]:
    """How many blocks share the keys of one (sequence, kv head, tile of query rows): (blocks of a cluster, clusters).

    Two blocks run on an SM; there are as many as give every SM its two, but none whose four warps would not have a tile
    of keys each.  More than a cluster's eight are joined by a second launch: only where they shorten a long run."""
    sms = sms or device_sms()
    tiles = max(1, -(-keys // KV8_TILE))
    want = min(2 * sms // max(1, batch * n_kv * row_tiles), -(-tiles // KV8_WARPS))
    if want <= KV8_CLUSTER:
        return max(1, want), 1
    if tiles <= 8 * KV8_CLUSTER * KV8_WARPS:
        return KV8_CLUSTER, 1
    return KV8_CLUSTER, want // KV8_CLUSTER


def attention_kv8(q: torch.Tensor, out: torch.Tensor, cu_q: torch.Tensor, kv_len: torch.Tensor, slots: torch.Tensor,
                  tables: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, *, n_kv: int, group: int, head_dim: int, scale: float, cap: float, window: int,
                  ring: int, batch: int, max_q_len: int, max_kv_len: int) -> None:
    """The newest ``cu_q[i + 1] - cu_q[i]`` tokens of every row i against the ``kv_len[i]`` that its slot holds, themselves
    among them (``kv8_write`` comes first).  ``q`` and ``out`` [tokens, n_kv * group * head_dim], float32 or bfloat16, query
    head h reads kv head h // group; ``scale``, ``cap`` (<= 0: none) and ``window`` (0: all keys) as everywhere.  A token
    that sees no key (padding) gets zeros.  ``max_q_len`` and ``max_kv_len`` bound the rows' new tokens and lengths."""
    what = "attention_kv8"
    n_blocks, G, block, dim = _cache(what, k_pages, v_pages, k_scale, v_scale)
    if (G, dim) != (n_kv, head_dim):
        raise KernelError(f"{what}: the pages hold {G} heads of {dim}, not {n_kv} of {head_dim}")
    for name, x in (("q", q), ("out", out)):
        if x.dim() != 2 or x.shape[1] != n_kv * group * head_dim or x.stride(1) != 1:
            raise KernelError(f"{what}: {name} must be [tokens, {n_kv * group * head_dim}] with rows of consecutive entries")
    if q.dtype != out.dtype or q.shape[0] != out.shape[0]:
        raise KernelError(f"{what}: q and out must have as many tokens and one element type")
    if tables.dim() != 2 or max_q_len < 1:
        raise KernelError(f"{what}: tables must be [slots, width] and max_q_len at least 1")
    if ring and (window <= 0 or ring < window + max_q_len + block - 2):
        raise KernelError(f"{what}: a ring of {ring} does not keep what {max_q_len} new tokens see under a window of {window}: "
                          f"it takes window + tokens + {block} - 2")
    _ints(what, ("cu_q", cu_q, batch + 1), ("kv_len", kv_len, batch), ("slots", slots, batch), ("tables", tables, None))
    rows = max_q_len * group
    keys = min(max_kv_len, window + max_q_len) if window > 0 else max_kv_len
    shares, spans = kv8_shares(batch, n_kv, -(-rows // (8 if rows <= 8 else 16)), keys)
    part_o = part_ml = 0
    if spans > 1:
        n = q.shape[0] * n_kv * group * spans
        parts = torch.empty(n * (head_dim + 2), dtype=torch.float32, device=q.device)
        part_o = parts.data_ptr()
        part_ml = part_o + 4 * n * head_dim
    _call("attn_kv8", "brolm_attn_kv8", _ATTN.pack(
        _ptr(q), _ptr(out), _ptr(cu_q), _ptr(kv_len), _ptr(slots), _ptr(tables), _ptr(k_pages), _ptr(v_pages), _ptr(k_scale),
        _ptr(v_scale), part_o, part_ml, _stream(), q.stride(0), out.stride(0), _code(q), q.shape[0], batch, n_kv, group, head_dim,
        block, n_blocks, tables.shape[0], tables.shape[1], ring, window, max_q_len, shares, spans, scale, cap), what)
