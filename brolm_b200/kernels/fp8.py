"""Python face of the products with matrices in 8-bit floating point: rows rounded to 8 bits and read back, products, a gated
feed-forward, routed experts.

A number is e4m3 (a sign, four bits of exponent, three of mantissa; largest 448) times a power of two that 128 consecutive
numbers of a row share: the least from 2^-127 on under which none of them is beyond 448 times it.  Rounding is to nearest, ties
to even.  A block with a number that is not finite is NaN as a whole, and so is what is computed from it.  Both sides of a
product are such rows; products are exact, sums are float32.

``Fp8Matrix`` holds rows in the order the kernels want them: ``fp8_quantize`` makes one from rows or a matrix, or from a stack
of experts' matrices; ``fp8_gate_up`` from the two matrices of a gated feed-forward, whose rows then alternate.  A matrix in
use as a weight may be read before what runs ahead of the product in its stream has ended, except for ``fp8_quantize`` itself;
it is made once and kept.

The functions launch on the current stream, like all of this package, and wait for nothing.
"""
from __future__ import annotations

import dataclasses
from ctypes import c_float, c_int, c_longlong, c_void_p
from typing import Optional

import torch

from . import ACTIVATIONS, EXPERT_ACTS, KernelError, _check, _fn, _ptr, _stream, device_sms, library_loaded, load_library

BLOCK = 128              # numbers that share a scale
_TILE = 512              # bytes of scales of 128 rows and four blocks
_CODES = {torch.float32: 0, torch.bfloat16: 1}
_PIECE = 16              # blocks of K that a float32 result is summed over before the sum goes to registers


@dataclasses.dataclass
class Fp8Matrix:
    """Rows of 8-bit numbers.  ``shape``: (rows, columns) or (experts, rows, columns).  ``gated``: the rows of a gate and of its
    partner alternate, so that a product has half as many results as there are rows."""
    values: torch.Tensor         # uint8 [rows of all experts, columns rounded up to 16]
    scales: torch.Tensor         # uint8 [rows / 128, columns / 512, 512]
    shape: tuple
    gated: bool = False

    @property
    def rows(self) -> int:
        return self.shape[-2]

    @property
    def cols(self) -> int:
        return self.shape[-1]

    @property
    def outputs(self) -> int:
        """How many results a row's product with this matrix has."""
        return self.shape[-2] // 2 if self.gated else self.shape[-2]

    @property
    def group_rows(self) -> int:
        """Rows that an expert's matrix takes."""
        return self.values.shape[0] // self.shape[0] if len(self.shape) == 3 else self.shape[0]

    @property
    def device(self) -> torch.device:
        return self.values.device

    @property
    def nbytes(self) -> int:
        return self.values.numel() + self.scales.numel()


def _round_up(n: int, m: int) -> int:
    return (n + m - 1) // m * m


def _empty(shape: tuple, device, gated: bool = False, scale_rows: Optional[int] = None) -> Fp8Matrix:
    rows, cols = shape[-2:]
    # an expert's matrix begins with a tile of scales
    total = rows if len(shape) == 2 else shape[0] * _round_up(rows, 128)
    values = torch.empty((total, _round_up(cols, 16)), dtype=torch.uint8, device=device)
    scales = torch.empty((((scale_rows or total) + 127) // 128, (cols + 511) // 512, _TILE), dtype=torch.uint8, device=device)
    return Fp8Matrix(values, scales, tuple(shape), gated)


def _rows(what: str, x: torch.Tensor) -> torch.Tensor:
    if x.dtype not in _CODES:
        raise KernelError(f"{what}: element type {x.dtype} is not float32 or bfloat16")
    if not x.is_cuda:
        raise KernelError("brolm_b200 kernels run on CUDA tensors only; there is no CPU path")
    if x.device.index != torch.cuda.current_device():
        raise KernelError(f"{what}: a tensor lives on {x.device}, the current device is cuda:{torch.cuda.current_device()}")
    if x.stride(-1) != 1 and x.shape[-1] > 1:
        raise KernelError(f"{what}: rows must be packed (strides {tuple(x.stride())})")
    return x


_Q_ARGS = [c_int, c_void_p, c_longlong, c_void_p, c_longlong, c_void_p, c_longlong, c_int, c_int, c_int, c_int, c_void_p]


def _quantize(x: torch.Tensor, m: Fp8Matrix, early: int) -> None:
    rows = x.shape[0]
    group = m.shape[-2] if len(m.shape) == 3 else max(rows, 1)
    f = _fn("fp8_rows", "brolm_fp8_quantize", _Q_ARGS)
    _check(f(_CODES[x.dtype], x.data_ptr(), x.stride(0), m.values.data_ptr(), m.values.stride(0), m.scales.data_ptr(), rows, x.shape[1],
             group, m.group_rows if len(m.shape) == 3 else group, early, _stream()), "fp8_quantize")


def fp8_quantize(x: torch.Tensor) -> Fp8Matrix:
    """x [rows, columns] or [experts, rows, columns], float32 or bfloat16, packed rows (any stride between them; a stack of
    experts contiguous) -> the same in 8 bits."""
    x = _rows("fp8_quantize", x)
    if x.dim() not in (2, 3) or x.shape[-1] == 0:
        raise KernelError(f"fp8_quantize: rows or a stack of matrices, not a tensor of shape {tuple(x.shape)}")
    if x.dim() == 3 and not x.is_contiguous():
        raise KernelError("fp8_quantize: a stack of matrices must be contiguous")
    m = _empty(tuple(x.shape), x.device)
    if x.numel():
        _quantize(x.view(-1, x.shape[-1]) if x.dim() == 3 else x, m, 0)
    return m


def fp8_gate_up(gate: torch.Tensor, up: torch.Tensor) -> Fp8Matrix:
    """The two matrices of a gated feed-forward, or of a stack of experts, in 8 bits, their rows one after the other in turn."""
    if gate.shape != up.shape or gate.dtype != up.dtype or gate.device != up.device:
        raise KernelError(f"fp8_gate_up: two matrices of a kind are wanted, not {tuple(gate.shape)} {gate.dtype} and {tuple(up.shape)} {up.dtype}")
    m = fp8_quantize(torch.stack((gate, up), dim=-2).flatten(-3, -2))
    m.gated = True
    return m


def fp8_read(m: Fp8Matrix, out: torch.Tensor) -> None:
    """out (the matrix's shape, float32 or bfloat16, packed rows; a stack contiguous) = the values that ``m`` stands for."""
    out = _rows("fp8_read", out)
    if tuple(out.shape) != tuple(m.shape) or (out.dim() == 3 and not out.is_contiguous()):
        raise KernelError(f"fp8_read: a matrix of shape {tuple(m.shape)} goes into such a tensor, not into {tuple(out.shape)}")
    if m.device != out.device:
        raise KernelError("fp8_read: the matrix and the result live on two devices")
    if not out.numel():
        return
    y = out.view(-1, out.shape[-1]) if out.dim() == 3 else out
    group = m.shape[-2] if len(m.shape) == 3 else y.shape[0]
    f = _fn("fp8_rows", "brolm_fp8_read", [c_int, c_void_p, c_longlong, c_void_p, c_void_p, c_longlong, c_longlong, c_int, c_int, c_int, c_void_p])
    _check(f(_CODES[y.dtype], m.values.data_ptr(), m.values.stride(0), m.scales.data_ptr(), y.data_ptr(), y.stride(0), y.shape[0], m.cols, group,
             m.group_rows if len(m.shape) == 3 else group, _stream()), "fp8_read")


# --- products ----------------------------------------------------------------
STREAM_ROWS = 128        # up to as many rows W is streamed; more are tiles of 256 x 256


def fp8_slices(tiles: int, nkb: int, sms: int) -> int:
    """Into how many slices K is cut for a product of few rows, ``tiles`` tiles of 128 rows of W and ``nkb`` blocks of K."""
    best = 1
    for s in range(2, 9):
        per = (nkb + s - 1) // s
        if per >= 2 and (s - 1) * per < nkb and tiles * s <= sms:
            best = s
    return best


def _out_check(what: str, out: torch.Tensor, rows: int, cols: int) -> None:
    _rows(what, out)
    if tuple(out.shape) != (rows, cols):
        raise KernelError(f"{what}: the result has the shape {(rows, cols)}, not {tuple(out.shape)}")


def _act_code(what: str, w: Fp8Matrix, activation: str) -> int:
    table = ACTIVATIONS if w.gated else EXPERT_ACTS
    if activation not in table:
        raise KernelError(f"{what}: unknown activation '{activation}' for {'gated' if w.gated else 'plain'} rows (known: {sorted(table)})")
    return table[activation]


def _to8(what: str, x, cols: int) -> Fp8Matrix:
    if isinstance(x, Fp8Matrix):
        if len(x.shape) != 2 or x.cols != cols:
            raise KernelError(f"{what}: rows of {cols} numbers are wanted, not {tuple(x.shape)}")
        return x
    x = _rows(what, x)
    if x.dim() != 2 or x.shape[1] != cols:
        raise KernelError(f"{what}: rows of {cols} numbers are wanted, not {tuple(x.shape)}")
    m = _empty(tuple(x.shape), x.device)
    if x.shape[0]:
        _quantize(x, m, 1)
    return m


def _product(x: Fp8Matrix, w: Fp8Matrix, out, act: int, limit: float) -> None:
    M, K, N = x.rows, x.cols, w.outputs
    if not M or not N:
        return
    to8 = isinstance(out, Fp8Matrix)
    if M <= STREAM_ROWS and not to8:
        slices = fp8_slices((w.rows + 127) // 128, (K + 127) // 128, device_sms())
        f = _fn("fp8_stream", "brolm_fp8_stream", [c_void_p, c_longlong, c_void_p, c_void_p, c_longlong, c_void_p, c_void_p, c_longlong, c_int, c_int, c_int,
                                                   c_int, c_int, c_int, c_float, c_int, c_void_p])
        _check(f(x.values.data_ptr(), x.values.stride(0), x.scales.data_ptr(), w.values.data_ptr(), w.values.stride(0), w.scales.data_ptr(), out.data_ptr(),
                 out.stride(0), 1 if out.dtype == torch.float32 else 0, M, N, K, 1 if w.gated else 0, act, limit, slices, _stream()), "linear_fp8")
        return
    y, kind = (out.values, 2) if to8 else (out, 1 if out.dtype == torch.float32 else 0)
    f = _fn("fp8_gemm", "brolm_fp8_gemm", [c_void_p, c_longlong, c_void_p, c_void_p, c_longlong, c_void_p, c_void_p, c_longlong, c_void_p, c_int, c_int, c_int,
                                           c_int, c_int, c_int, c_float, c_int, c_void_p])
    _check(f(x.values.data_ptr(), x.values.stride(0), x.scales.data_ptr(), w.values.data_ptr(), w.values.stride(0), w.scales.data_ptr(), y.data_ptr(), y.stride(0),
             out.scales.data_ptr() if to8 else None, kind, M, N, K, 1 if w.gated else 0, act, limit, _PIECE, _stream()), "linear_fp8")


def linear_fp8(x, w: Fp8Matrix, out: torch.Tensor, activation: str = "none", limit: float = 0.0) -> None:
    """out [rows, w.outputs] (float32 or bfloat16) = act(x w^T).  x [rows, columns]: float32 or bfloat16, which is rounded to 8
    bits first, or such rows.  With a plain matrix ``activation`` is "none" or "relu2" (the square of relu), with a gated one one
    of ``ACTIVATIONS``: act(gate) * partner."""
    if len(w.shape) != 2:
        raise KernelError("linear_fp8: a stack of experts' matrices goes to experts_fp8")
    act = _act_code("linear_fp8", w, activation)
    x8 = _to8("linear_fp8", x, w.cols)
    _out_check("linear_fp8", out, x8.rows, w.outputs)
    _product(x8, w, out, act, float(limit))


def feedforward_fp8(x, gate_up: Fp8Matrix, down: Fp8Matrix, out: torch.Tensor, activation: str = "gelu_tanh", limit: float = 0.0) -> None:
    """out [rows, down.rows] = (act(x Wg^T) * (x Wu^T)) Wd^T; what goes into the second product is rounded to 8 bits, too."""
    if len(gate_up.shape) != 2 or len(down.shape) != 2 or down.gated or gate_up.outputs != down.cols:
        raise KernelError(f"feedforward_fp8: matrices of shapes {tuple(gate_up.shape)} and {tuple(down.shape)} do not follow one another")
    act = _act_code("feedforward_fp8", gate_up, activation)
    x8 = _to8("feedforward_fp8", x, gate_up.cols)
    M, inter = x8.rows, gate_up.outputs
    _out_check("feedforward_fp8", out, M, down.rows)
    if M <= STREAM_ROWS:
        h = torch.empty((M, inter), dtype=torch.float32, device=out.device)
        _product(x8, gate_up, h, act, float(limit))
        h8 = _to8("feedforward_fp8", h, inter)
    else:
        h8 = _empty((M, inter), out.device)
        _product(x8, gate_up, h8, act, float(limit))
    _product(h8, down, out, 0, 0.0)


# --- routed experts -----------------------------------------------------------
def experts_fp8_rows(pairs: int, experts: int) -> int:
    """How many rows a tile of an expert's pairs has."""
    mean = pairs / max(experts, 1)
    for rows in (16, 32, 64, 128):
        if mean <= 0.75 * rows:
            return rows
    return 256


def experts_fp8_pairs(x: torch.Tensor, ids: torch.Tensor, up: Fp8Matrix, down: Fp8Matrix, out: torch.Tensor, activation: str = "silu",
                      limit: float = 0.0, scale: Optional[torch.Tensor] = None) -> None:
    """Every (token, choice) pair through its expert: out float32 [top, tokens, down.rows], a pair's result at [its choice, its
    token].  ``ids`` int32 [tokens, top]: a number that is no expert's has no result (its place stays as it was).  ``up`` a stack
    [experts, ...], gated or not, ``down`` the stack of the second matrices; ``scale`` float32 [tokens, top] multiplies a pair's
    sums before the activation."""
    what = "experts_fp8"
    x = _rows(what, x)
    if len(up.shape) != 3 or len(down.shape) != 3 or down.gated or up.shape[0] != down.shape[0] or up.outputs != down.cols:
        raise KernelError(f"{what}: stacks of shapes {tuple(up.shape)} and {tuple(down.shape)} do not follow one another")
    if x.dim() != 2 or x.shape[1] != up.cols:
        raise KernelError(f"{what}: rows of {up.cols} numbers are wanted, not {tuple(x.shape)}")
    T = x.shape[0]
    if ids.dim() != 2 or ids.shape[0] != T or ids.dtype != torch.int32 or not ids.is_contiguous():
        raise KernelError(f"{what}: ids are a packed int32 [tokens, top]")
    E, top, dev = up.shape[0], ids.shape[1], x.device
    if tuple(out.shape) != (top, T, down.rows) or out.dtype != torch.float32 or not out.is_contiguous():
        raise KernelError(f"{what}: the pairs' results are a packed float32 {(top, T, down.rows)}")
    if scale is not None and (scale.dtype != torch.float32 or scale.shape != ids.shape or not scale.is_contiguous()):
        raise KernelError(f"{what}: the pairs' scales are a packed float32 [tokens, top]")
    for t in (ids, up, down, out, scale):
        if t is not None and t.device != dev:
            raise KernelError(f"{what}: tensors on {dev} and {t.device}")
    act = _act_code(what, up, activation)
    P, K, inter, N = T * top, x.shape[1], up.outputs, down.rows
    if not P or not E or not N:
        return
    rows = experts_fp8_rows(P, E)
    pad = _round_up(rows, 128)
    most = (P + rows - 1) // rows + min(E, P)
    lists = torch.empty(2 * P + E + 1 + 2 * most, dtype=torch.int32, device=dev)
    at = lists.data_ptr()
    perm, place, offsets, group, row0 = at, at + 4 * P, at + 8 * P, at + 8 * P + 4 * (E + 1), at + 8 * P + 4 * (E + 1 + most)
    stream = _stream()
    f = _fn("fp8_rows", "brolm_fp8_group", [c_void_p, c_int, c_int, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_int, c_void_p])
    _check(f(ids.data_ptr(), P, E, rows, perm, place, offsets, group, row0, most, stream), what)
    gather = _fn("fp8_rows", "brolm_fp8_gather", [c_int, c_void_p, c_longlong, c_void_p, c_void_p, c_int, c_void_p, c_longlong, c_void_p, c_int, c_int, c_void_p])
    a = _empty((P, K), dev, scale_rows=most * pad)
    _check(gather(_CODES[x.dtype], x.data_ptr(), x.stride(0), perm, place, top, a.values.data_ptr(), a.values.stride(0), a.scales.data_ptr(), P, K, stream), what)
    s = scale.data_ptr() if scale is not None else None
    h8 = _empty((P, inter), dev, scale_rows=most * pad)
    if rows <= STREAM_ROWS:
        f = _fn("fp8_stream", "brolm_fp8_experts_stream", [c_void_p, c_longlong, c_void_p, c_void_p, c_longlong, c_void_p, c_void_p, c_longlong, c_int, c_int,
                                                           c_int, c_int, c_int, c_int, c_int, c_int, c_float, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                                           c_int, c_int, c_int, c_int, c_int, c_void_p])

        def product(m, w, y, ldy, n, k, code, sc, last):
            _check(f(m.values.data_ptr(), m.values.stride(0), m.scales.data_ptr(), w.values.data_ptr(), w.values.stride(0), w.scales.data_ptr(), y, ldy, 1, P, n, k,
                     E, w.group_rows, 1 if w.gated else 0, code, float(limit), group, row0, offsets, perm, sc, last, top, T, rows, most, stream), what)
        h = torch.empty((P, inter), dtype=torch.float32, device=dev)
        product(a, up, h.data_ptr(), inter, inter, K, act, s, 0)
        _check(gather(0, h.data_ptr(), inter, perm, place, 0, h8.values.data_ptr(), h8.values.stride(0), h8.scales.data_ptr(), P, inter, stream), what)
        product(h8, down, out.data_ptr(), N, N, inter, 0, None, 1)
        return
    f = _fn("fp8_gemm", "brolm_fp8_experts_gemm", [c_void_p, c_longlong, c_void_p, c_void_p, c_longlong, c_void_p, c_void_p, c_longlong, c_void_p, c_int, c_int,
                                                   c_int, c_int, c_int, c_int, c_int, c_int, c_float, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p,
                                                   c_int, c_int, c_int, c_int, c_void_p])

    def product(m, w, y, ldy, ys, kind, n, k, code, sc, last):
        _check(f(m.values.data_ptr(), m.values.stride(0), m.scales.data_ptr(), w.values.data_ptr(), w.values.stride(0), w.scales.data_ptr(), y, ldy, ys, kind, P, n,
                 k, E, w.group_rows, 1 if w.gated else 0, code, float(limit), _PIECE, group, row0, offsets, perm, sc, last, top, T, most, stream), what)
    product(a, up, h8.values.data_ptr(), h8.values.stride(0), h8.scales.data_ptr(), 2, inter, K, act, s, 0)
    product(h8, down, out.data_ptr(), N, None, 1, N, inter, 0, None, 1)


def experts_fp8(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, up: Fp8Matrix, down: Fp8Matrix, out: torch.Tensor, activation: str = "silu",
                limit: float = 0.0, scale_input: bool = False) -> None:
    """out [tokens, down.rows] (float32 or bfloat16) = the sum over a token's choices of ``weights`` times its expert's result, in
    the order of the choices; a number in ``ids`` that is no expert's adds nothing.  With ``scale_input`` the weight multiplies
    the sums before the activation and not the result."""
    what = "experts_fp8"
    if weights.shape != ids.shape or weights.dtype != torch.float32 or not weights.is_contiguous() or weights.device != x.device:
        raise KernelError(f"{what}: weights are a packed float32 [tokens, top] beside the tokens")
    T, top = ids.shape
    _out_check(what, out, T, down.rows)
    y = torch.empty((top, T, down.rows), dtype=torch.float32, device=out.device)
    experts_fp8_pairs(x, ids, up, down, y, activation, limit, weights if scale_input else None)
    if not T or not down.rows:
        return
    f = _fn("fp8_rows", "brolm_fp8_combine", [c_void_p, c_void_p, c_void_p, c_int, c_int, c_int, c_int, c_void_p, c_longlong, c_int, c_void_p])
    _check(f(y.data_ptr(), ids.data_ptr(), None if scale_input else weights.data_ptr(), top, up.shape[0], T, down.rows, out.data_ptr(), out.stride(0),
             1 if out.dtype == torch.float32 else 0, _stream()), what)


def fp8_stream_status(reset: bool = False) -> int:
    """0 if no bounded wait of the products of few rows ever ran out; otherwise its code.  Synchronises."""
    return _status("fp8_stream", reset)


def fp8_gemm_status(reset: bool = False) -> int:
    """0 if no bounded wait of the products of many rows ever ran out; otherwise its code.  Synchronises."""
    return _status("fp8_gemm", reset)


def _status(lib: str, reset: bool) -> int:
    if not library_loaded(lib):
        return 0
    f = getattr(load_library(lib), f"brolm_{lib}_status")
    f.argtypes = [c_int]
    f.restype = c_int
    return f(1 if reset else 0)
