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
