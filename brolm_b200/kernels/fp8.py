"""Python face of the products with matrices in 8-bit floating point: rows rounded to 8 bits and read back, products, a gated
feed-forward, routed experts.

A number is e4m3 (a sign, four bits of exponent, three of mantissa; largest 448) times a power of two that 128 consecutive
numbers of a row share: the least from 2^-127 on under which none of them is beyond 448 times it.  Rounding is to nearest, ties
to even (numbers beyond 240 * 2^120 may become 2^128, which a float32 reads as infinity).  A block with a number that is not
finite is NaN as a whole, and so is what is computed from it.  Both sides of a product are such rows; products are exact, sums
are float32.

``Fp8Matrix`` holds rows in the order the kernels want them: ``fp8_quantize`` makes one from rows or a matrix, or from a stack
of experts' matrices; ``fp8_gate_up`` from the two matrices of a gated feed-forward, whose rows then alternate.  A matrix is made
once and kept, on the stream that is current when the object is made.  Its products wait for what runs ahead of them until one has
been launched on that stream (captured ones count for nothing and, captured before that, stay so); from then on they may read
the matrix before what runs ahead of them has ended.

The functions launch on the current stream, like all of this package, and wait for nothing.  All that is kept from call to call is
whether a matrix has had that product.
"""
from __future__ import annotations

import functools
import struct
from ctypes import c_char_p, c_int, c_void_p, cast
from typing import Optional

import torch

from . import ACTIVATIONS, EXPERT_ACTS, KernelError, _check, _fn, add_launches, device_sms, library_loaded, load_library

BLOCK = 128              # numbers that share a scale
_TILE = 512              # bytes of scales of 128 rows and four blocks
_BF16, _F32 = torch.bfloat16, torch.float32
_CODES = {_F32: 0, _BF16: 1}
_OUT = {_BF16: 0, _F32: 1}
_FUSED = {_BF16: 1, _F32: 2}
_NO_CPU = "brolm_b200 kernels run on CUDA tensors only; there is no CPU path"
_new_matrix = object.__new__
_raw_stream, _device = torch._C._cuda_getCurrentRawStream, torch._C._cuda_getDevice

# A product of few rows is a few microseconds on the device, so what the host does for it counts: the launchers take one
# struct, packed here as C lays it out, and the checks of a call's arguments are one expression; which of them failed is found
# out only then.
_ROWS = struct.Struct("@4P3q5i")
_PRODUCT = struct.Struct("@7P3q8ifi5P7i2Pqiii")
_EXPERTS = struct.Struct("@13P5q14if")
_NORM = struct.Struct("@7Pq3i4f")
_functions: dict = {}
_launchers: dict = {}        # by name, as other launchers are given them


def _call(lib: str, name: str, packed: bytes, what: str) -> None:
    f = _functions.get(name)
    if f is None:
        f = _functions[name] = _fn(lib, name, [c_char_p])
    _check(f(packed), what)


def _launcher(lib: str, name: str) -> int:
    f = _launchers.get(name)
    if f is None:
        f = _launchers[name] = cast(getattr(load_library(lib), name), c_void_p).value
    return f


class Fp8Matrix:
    """Rows of 8-bit numbers.  ``shape``: (rows, columns) or (experts, rows, columns).  ``gated``: the rows of a gate and of its
    partner alternate, so that a product has half as many results as there are rows.  It is not to be changed once it is in
    use.  ``data`` holds ``values``, uint8 [rows of all experts, columns rounded up to 16], an expert's matrix beginning on a
    multiple of 128 rows, and behind them ``scales``, uint8 [rows / 128, columns / 512, 512]."""
    __slots__ = ("data", "shape", "gated", "rows", "cols", "outputs", "group_rows", "total", "device", "index", "packed", "stream", "fresh")

    def __init__(self, data: torch.Tensor, shape: tuple, gated: bool = False):
        shape = tuple(shape)
        if len(shape) not in (2, 3) or shape[0] < 0 or shape[-2] < 0 or shape[-1] <= 0 or (gated and shape[-2] % 2):
            raise KernelError(f"Fp8Matrix: {shape} is no shape of rows or of experts' matrices" + (" with gate and partner in turn" if gated else ""))
        rows = shape[0] if len(shape) == 2 else shape[0] * _round_up(shape[1], 128)
        need = _bytes(rows, shape[-1], rows)
        if data.dtype != torch.uint8 or data.dim() != 1 or not data.is_contiguous() or data.numel() < need:
            raise KernelError(f"Fp8Matrix: a matrix of shape {shape} is {need} bytes (uint8, one dimension, packed), not {tuple(data.shape)} of {data.dtype}")
        self._lay(data, shape, gated)

    def _lay(self, data: torch.Tensor, shape: tuple, gated: bool) -> "Fp8Matrix":
        self.data, self.shape, self.gated = data, shape, gated
        self.rows, self.cols = rows, cols = shape[-2], shape[-1]
        # how many results a row's product with this matrix has
        self.outputs = rows >> 1 if gated else rows
        # rows that an expert's matrix takes, and all of them
        self.group_rows = rows if len(shape) == 2 else (rows + 127) & -128
        self.total = rows if len(shape) == 2 else shape[0] * self.group_rows
        self.device = data.device
        self.index = index = data.get_device()
        # What makes it ends on this stream without a fence, so a product right behind that, with another stream's product already
        # launched or none, must not read ahead.  Other streams reach the matrix through an event, which is behind its stores.
        self.stream = _raw_stream(index) if index >= 0 else 0
        self.fresh = True
        at, ld = data.data_ptr(), (cols + 15) & -16
        self.packed = (at, at + ((self.total * ld + 511) & -512), ld)
        return self

    def __reduce__(self):
        return Fp8Matrix, (self.data, self.shape, self.gated)      # a copy has addresses of its own

    @property
    def values(self) -> torch.Tensor:
        return self.data[:self.total * self.packed[2]].view(self.total, self.packed[2])

    @property
    def scales(self) -> torch.Tensor:
        return self.data[self.packed[1] - self.packed[0]:].view((self.total + 127) >> 7, (self.cols + 511) >> 9, _TILE)

    @property
    def nbytes(self) -> int:
        return self.data.numel()

    def float(self) -> torch.Tensor:
        """The values that the matrix stands for."""
        y = torch.empty(self.shape, dtype=_F32, device=self.device)
        fp8_read(self, y)
        return y

    def __repr__(self) -> str:
        return f"Fp8Matrix({self.shape}, gated={self.gated}, {self.device})"


def _round_up(n: int, m: int) -> int:
    return (n + m - 1) // m * m


def _bytes(rows: int, cols: int, scale_rows: int) -> int:
    return ((rows * ((cols + 15) & -16) + 511) & -512) + ((scale_rows + 127) >> 7) * ((cols + 511) >> 9) * _TILE


def _empty(shape: tuple, device, gated: bool = False) -> Fp8Matrix:
    rows = shape[0] if len(shape) == 2 else shape[0] * _round_up(shape[1], 128)
    # (what the constructor asks holds here; asking costs the host 0.5 us)
    return _new_matrix(Fp8Matrix)._lay(torch.empty(_bytes(rows, shape[-1], rows), dtype=torch.uint8, device=device), shape, gated)


def _refuse(what: str, t: torch.Tensor, name: str, dim: int = 2) -> None:
    """Names what is wrong with a tensor of rows; returns if nothing is."""
    if t.dtype not in _CODES:
        raise KernelError(f"{what}: {name} has the element type {t.dtype}, not float32 or bfloat16")
    if not t.is_cuda:
        raise KernelError(_NO_CPU)
    if t.get_device() != _device():
        raise KernelError(f"{what}: {name} lives on {t.device}, the current device is cuda:{_device()}")
    if t.dim() != dim:
        raise KernelError(f"{what}: {name} has {t.dim()} dimensions, not {dim}")
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise KernelError(f"{what}: the rows of {name} must be packed (strides {tuple(t.stride())})")


def _quantize(x: torch.Tensor, packed: tuple, group: int, pad: int, early: int) -> None:
    rows, cols = x.shape
    _call("fp8_rows", "brolm_fp8_quantize", _ROWS.pack(x.data_ptr(), packed[0], packed[1], _raw_stream(_device()), x.stride(0), packed[2], rows,
                                                       _CODES[x.dtype], cols, group, pad, early), "fp8_quantize")


def fp8_quantize(x: torch.Tensor) -> Fp8Matrix:
    """x [rows, columns] or [experts, rows, columns], float32 or bfloat16, packed rows (any stride between them; a stack of
    experts contiguous) -> the same in 8 bits."""
    what = "fp8_quantize"
    if not isinstance(x, torch.Tensor) or x.dim() not in (2, 3) or x.shape[-1] == 0:
        raise KernelError(f"{what}: rows or a stack of matrices are wanted, not {tuple(getattr(x, 'shape', ()))}")
    shape = tuple(x.shape)
    if x.dtype not in _CODES or x.get_device() < 0 or x.get_device() != _device() or x.stride(-1) != 1:
        _refuse(what, x, "x", len(shape))
    if len(shape) == 3 and not x.is_contiguous():
        raise KernelError(f"{what}: a stack of matrices must be contiguous")
    m = _empty(shape, x.device)
    if x.numel():
        _quantize(x.view(-1, shape[-1]) if len(shape) == 3 else x, m.packed, m.rows, m.group_rows, 0)
    return m


def fp8_gate_up(gate: torch.Tensor, up: torch.Tensor) -> Fp8Matrix:
    """The two matrices of a gated feed-forward, or of a stack of experts, in 8 bits, their rows one after the other in turn."""
    if gate.dim() not in (2, 3) or gate.shape != up.shape or gate.dtype != up.dtype or gate.device != up.device:
        raise KernelError(f"fp8_gate_up: two matrices of a kind are wanted, not {tuple(gate.shape)} {gate.dtype} and {tuple(up.shape)} {up.dtype}")
    m = fp8_quantize(torch.stack((gate, up), dim=-2).flatten(-3, -2))
    return Fp8Matrix(m.data, m.shape, True)


def fp8_read(m: Fp8Matrix, out: torch.Tensor) -> None:
    """out (the matrix's shape, float32 or bfloat16, packed rows; a stack contiguous) = the values that ``m`` stands for."""
    _refuse("fp8_read", out, "out", len(m.shape))
    if tuple(out.shape) != m.shape or (out.dim() == 3 and not out.is_contiguous()):
        raise KernelError(f"fp8_read: a matrix of shape {m.shape} goes into such a (packed) tensor, not into {tuple(out.shape)}")
    if m.device != out.device:
        raise KernelError("fp8_read: the matrix and the result live on two devices")
    if out.dim() == 2 and out.shape[0] > 1 and out.stride(0) < out.shape[1]:
        raise KernelError(f"fp8_read: the rows of the result lie over one another (strides {tuple(out.stride())})")
    if not out.numel():
        return
    y = out.view(-1, out.shape[-1]) if out.dim() == 3 else out
    _call("fp8_rows", "brolm_fp8_read", _ROWS.pack(y.data_ptr(), m.packed[0], m.packed[1], _raw_stream(_device()), y.stride(0), m.packed[2], y.shape[0],
                                                   _CODES[y.dtype], m.cols, m.rows, m.group_rows, 1), "fp8_read")


def residual_rmsnorm_fp8_ok(hidden: int) -> bool:
    """Whether ``residual_rmsnorm_fp8`` takes rows of as many numbers."""
    return 0 < hidden <= 8192 and hidden % 4 == 0


def residual_rmsnorm_fp8(h: torch.Tensor, y: torch.Tensor, post_weight: Optional[torch.Tensor], post_eps: float, post_offset: float,
                         next_weight: torch.Tensor, next_eps: float, next_offset: float) -> Fp8Matrix:
    """h += rmsnorm(y; post) (or y when ``post_weight`` is None); -> rmsnorm(h; next) as rows of 8 bits, rounded once from its float
    result.  h and y float32 [rows, hidden], contiguous, ``hidden`` a multiple of 4 and 8,192 at most; both and the gains begin on
    borders of 16 bytes."""
    what = "residual_rmsnorm_fp8"
    device = h.get_device()
    fine = h.dtype == y.dtype == _F32 and h.dim() == 2 and h.shape == y.shape and h.is_contiguous() and y.is_contiguous() \
        and device >= 0 and device == _device() == y.get_device() and residual_rmsnorm_fp8_ok(h.shape[1])
    for w in (next_weight, post_weight):
        if fine and w is not None:
            fine = w.dtype == next_weight.dtype and w.dtype in _CODES and w.numel() == h.shape[1] and w.is_contiguous() and w.get_device() == device
    if not fine:
        for t, name in ((h, "h"), (y, "y")):
            _refuse(what, t, name)
            if t.dtype != _F32 or not t.is_contiguous() or t.shape != h.shape:
                raise KernelError(f"{what}: {name} is a packed float32 [rows, hidden], not {tuple(t.shape)} {t.dtype}")
        if not residual_rmsnorm_fp8_ok(h.shape[1]):
            raise KernelError(f"{what}: rows of {h.shape[1]} numbers (a multiple of 4, 8,192 at most, is wanted)")
        raise KernelError(f"{what}: the gains are packed rows of {h.shape[1]} numbers of one element type (float32 or bfloat16) on {h.device}")
    m = _empty(tuple(h.shape), h.device)
    if m.rows:
        _call("fp8_rows", "brolm_residual_rmsnorm_fp8",
              _NORM.pack(h.data_ptr(), y.data_ptr(), post_weight.data_ptr() if post_weight is not None else 0, next_weight.data_ptr(), m.packed[0], m.packed[1],
                         _raw_stream(device), m.packed[2], m.rows, m.cols, _CODES[next_weight.dtype], post_eps, post_offset, next_eps, next_offset), what)
    return m


# --- products ----------------------------------------------------------------
STREAM_ROWS = 128        # up to as many rows W is streamed; more are tiles of 256 x 256
FUSED_ROWS = 16          # up to as many rows the stream of W can round the rows itself ...
_FUSED_BLOCKS = 16       # ... where a block keeps no more than as many blocks of K of them
_PIECE = 32              # blocks of K that a float32 result is summed over, in tiles and streams, before the sum goes to registers
_ACTS = {(gated, name): code for gated, table in ((True, ACTIVATIONS), (False, EXPERT_ACTS)) for name, code in table.items()}


@functools.lru_cache(maxsize=1024)
def fp8_slices(tiles: int, nkb: int, sms: int) -> int:
    """Into how many slices K is cut for a product of few rows, ``tiles`` tiles of 128 rows of W and ``nkb`` blocks of K: as many
    as find room at a time (two blocks an SM, of which clusters leave an eighth empty), of two blocks of K at least.
    8 rows in 8 bits, 1 / 4 / 8 slices: 2,304 x 9,216 17.8 / 7.9 / 6.7 us; 4,608 x 36,864 in 1 / 4 / 7 / 8: 68 / 31.4 / 28.4 / 37.1."""
    best = 1
    for s in range(2, 9):
        per = (nkb + s - 1) // s
        if per >= 2 and (s - 1) * per < nkb and 8 * tiles * s <= 14 * sms:
            best = s
    return best


def fp8_fused(rows: int, nkb: int, slices: int, words: int) -> bool:
    """Whether the stream of W rounds the rows itself: every block those of its slice, four blocks of K of a row (``words`` words
    of sixteen bytes a lane: 2 for bfloat16, 4 for float32) a warp, eight warps with eight such words each in one round.  A
    launch less, and every block's time, whose ring the rows leave fewer stages.  Fused / apart in a captured loop, bfloat16 rows:
    2,304 x 9,216 (slices of 9 blocks) 1 row 6.9 / 8.5 us, 8 rows 8.4 / 8.7; 5,000 x 11,000 (15) 4 rows 12.3 / 13.0; 18,432 x 2,048
    (16) 1 row 10.1 / 10.5, 4 rows 10.7 / 10.6; x 2,304 (18) 11.1 / 10.8 and 11.9 / 10.8; x 2,944 (23) 13.9 / 12.6 and 14.8 / 12.7.
    From Python, 1 row: 7.3 / 11.8 with 9 blocks, 11.1 / 11.8 with 18, 14.0 / 13.0 with 23."""
    per = (nkb + slices - 1) // slices
    return rows <= FUSED_ROWS and per <= _FUSED_BLOCKS and rows * ((per + 6) // 4) * words <= 64


def _act_code(what: str, w: Fp8Matrix, activation: str) -> int:
    code = _ACTS.get((w.gated, activation))
    if code is None:
        table = ACTIVATIONS if w.gated else EXPERT_ACTS
        raise KernelError(f"{what}: unknown activation '{activation}' for {'gated' if w.gated else 'plain'} rows (known: {sorted(table)})")
    return code


def _checked(what: str, x, w: Fp8Matrix, out: torch.Tensor, outputs: int) -> None:
    """Refuses rows, a matrix and a result that do not go together."""
    if type(x) is Fp8Matrix:
        if len(x.shape) != 2 or x.cols != w.cols:
            raise KernelError(f"{what}: rows of {w.cols} numbers are wanted, not {x.shape}")
        fine = x.index == w.index
    else:
        fine = x.dtype in _CODES and x.dim() == 2 and x.shape[1] == w.cols and x.get_device() == w.index and (x.stride(1) == 1 or w.cols == 1)
    if fine and len(w.shape) == 2 and w.index >= 0 and w.index == _device() and out.dtype in _CODES and out.get_device() == w.index and out.dim() == 2 \
            and out.shape[0] == x.shape[0] and out.shape[1] == outputs and (out.stride(1) == 1 or outputs == 1) \
            and (out.stride(0) >= outputs or out.shape[0] <= 1):
        return
    if len(w.shape) != 2:
        raise KernelError(f"{what}: a stack of experts' matrices goes to experts_fp8")
    if type(x) is not Fp8Matrix:
        _refuse(what, x, "x")
        if x.shape[1] != w.cols:
            raise KernelError(f"{what}: rows of {w.cols} numbers are wanted, not {tuple(x.shape)}")
    _refuse(what, out, "out")
    if tuple(out.shape) != (x.shape[0], outputs):
        raise KernelError(f"{what}: the result has the shape {(x.shape[0], outputs)}, not {tuple(out.shape)}")
    if out.shape[0] > 1 and out.stride(0) < out.shape[1]:
        raise KernelError(f"{what}: the rows of the result lie over one another (strides {tuple(out.stride())})")
    raise KernelError(f"{what}: the rows, the matrix and the result live on {x.device}, {w.device} and {out.device}; the current device is cuda:{_device()}")


_NO_EXPERTS = (0,) * 13
_THERE = (0, 0, 0, 0)        # rows in 8 bits already


@functools.lru_cache(maxsize=1024)
def fp8_streamed(rows: int, w_rows: int, nkb: int, sms: int) -> bool:
    """Whether a product streams W (128 rows of it at a time) or goes in tiles of 256 x 256.  Up to 64 rows it does; up to 128
    but where the tiles come out as one round of the pairs of SMs that is nearly full, or K is short: 128 rows 18,432 x 2,304
    (72 tiles) 17.7 us streamed and 14.0 in tiles, 1,000 x 640 6.9 and 5.3, but 2,304 x 9,216 (9 tiles) 12.5 and 23.1, 28,672 x
    3,584 (112 tiles) 28.8 and 29.2; 64 rows 13.7 and 14.0, 5.1 and 5.1."""
    if rows <= 64 or rows > STREAM_ROWS:
        return rows <= 64
    tiles, pairs = (w_rows + 255) // 256, sms // 2
    return not (nkb <= 6 or (4 * tiles >= 3 * pairs and tiles <= pairs and nkb <= 32))


def _rounded(M: int, K: int, w_rows: int, out: int, words: int, sms: int) -> tuple:
    """How a product goes: (streamed, the cut of K, whether the stream rounds the rows itself); ``words`` as ``fp8_fused`` has
    them, 0 for rows in 8 bits."""
    nkb = (K + 127) >> 7
    if out != 2 and fp8_streamed(M, w_rows, nkb, sms):
        cut = fp8_slices((w_rows + 127) >> 7, nkb, sms)
        return True, cut, words > 0 and fp8_fused(M, nkb, cut, words)
    return False, _PIECE, False


_rounded = functools.lru_cache(maxsize=4096)(_rounded)


def _pack(how: tuple, x, at: int, M: int, w: Fp8Matrix, y: tuple, out: int, act: int, limit: float, stream: int, piece: int) -> bytes:
    """A product's struct.  ``x``: (values, scales, stride) of rows in 8 bits, or (numbers, 0, stride, type) of rows that are
    rounded on the way, into the scratch at ``at`` if not by the product itself.  ``piece``: of a float result that stays one."""
    K = w.cols
    fused, raw = 0, _THERE
    if len(x) == 4:
        if how[2]:
            fused = _FUSED[x[3]]
        else:
            ld = (K + 15) & -16
            raw = (_launcher("fp8_rows", "brolm_fp8_quantize"), x[0], x[2], _CODES[x[3]])
            x = (at, at + ((M * ld + 511) & -512), ld)
    wv, ws, ldw = w.packed
    return _PRODUCT.pack(x[0], x[1], wv, ws, y[0], y[1], stream, x[2], ldw, y[2], M, w.outputs, K, 1 if w.gated else 0, act, out, fused, how[1], limit,
                         *_NO_EXPERTS, *raw, piece, 1 if w.fresh else 0)


def _launched(stream: int, *matrices: Fp8Matrix) -> None:
    """Products with these matrices have been launched on ``stream``: there the matrices are complete for what comes next."""
    for w in matrices:
        if w.fresh and stream == w.stream and not torch.cuda.is_current_stream_capturing():
            w.fresh = False


def linear_fp8(x, w: Fp8Matrix, out: torch.Tensor, activation: str = "none", limit: float = 0.0) -> None:
    """out [rows, w.outputs] (float32 or bfloat16) = act(x w^T).  x [rows, columns]: float32 or bfloat16, which is rounded to 8
    bits first, or such rows.  With a plain matrix ``activation`` is "none" or "relu2" (the square of relu), with a gated one one
    of ``ACTIVATIONS``: act(gate) * partner.  ``out`` does not lie over x or the matrix."""
    act = _act_code("linear_fp8", w, activation)
    _checked("linear_fp8", x, w, out, w.outputs)
    M, K, device = x.shape[0], w.cols, w.index
    if not M or not w.outputs:
        return
    held, at = None, 0
    if type(x) is Fp8Matrix:
        x = x.packed
        how = _rounded(M, K, w.rows, 0, 0, device_sms(w.device))
    else:
        how = _rounded(M, K, w.rows, 0, x.element_size(), device_sms(w.device))
        if not how[2]:
            held = torch.empty(_bytes(M, K, M), dtype=torch.uint8, device=w.device)
            at = held.data_ptr()
            add_launches(1)
        x = (x.data_ptr(), 0, x.stride(0), x.dtype)
    stream = _raw_stream(device)
    packed = _pack(how, x, at, M, w, (out.data_ptr(), 0, out.stride(0)), _OUT[out.dtype], act, limit, stream, _PIECE)
    if how[0]:
        _call("fp8_stream", "brolm_fp8_stream", packed, "linear_fp8")
    else:
        _call("fp8_gemm", "brolm_fp8_gemm", packed, "linear_fp8")
    if w.fresh:
        _launched(stream, w)


def feedforward_fp8(x, gate_up: Fp8Matrix, down: Fp8Matrix, out: torch.Tensor, activation: str = "gelu_tanh", limit: float = 0.0) -> None:
    """out [rows, down.rows] = (act(x Wg^T) * (x Wu^T)) Wd^T; what goes into the second product is rounded to 8 bits, too.
    ``gate_up`` may be a plain matrix with "relu2" or "none" for an ``activation``: out = act(x W^T) Wd^T."""
    if len(gate_up.shape) != 2 or len(down.shape) != 2 or down.gated or gate_up.outputs != down.cols or gate_up.index != down.index:
        raise KernelError(f"feedforward_fp8: matrices of shapes {gate_up.shape} and {down.shape} do not follow one another")
    act = _act_code("feedforward_fp8", gate_up, activation)
    _checked("feedforward_fp8", x, gate_up, out, down.rows)
    M, inter, device = x.shape[0], down.cols, down.index
    if not M or not down.rows:
        return
    sms = device_sms(down.device)
    # what lies between is rounded by the first product's own end, but where K is cut or a stream has more than 64 rows, whose
    # accumulator is one and waits: then it leaves floats (2,304 and 9,216: 8 rows 21.0 us for 24.0, 64 22.5 for 23.8, 100 26.9 for 25.4)
    words = 0 if type(x) is Fp8Matrix else x.element_size()
    first = _rounded(M, gate_up.cols, gate_up.rows, 0, words, sms)
    floats = first[0] and (first[1] > 1 or M > 64)
    second = _rounded(M, inter, down.rows, 0, 4 if floats else 0, sms)
    # one room: x in 8 bits, what lies between in 8 bits, as floats
    x8 = _bytes(M, gate_up.cols, M) if words and not first[2] else 0
    h8 = 0 if second[2] else _bytes(M, inter, M)
    held = torch.empty(x8 + h8 + (4 * M * inter if floats else 0), dtype=torch.uint8, device=down.device)
    at = held.data_ptr()
    x = x.packed if not words else (x.data_ptr(), 0, x.stride(0), x.dtype)
    ld = (inter + 15) & -16
    between = (at + x8, at + x8 + ((M * ld + 511) & -512), ld)
    stream = _raw_stream(device)
    a = _pack(first, x, at, M, gate_up, (at + x8 + h8, 0, inter) if floats else between, 1 if floats else 2, act, limit, stream, 0)
    b = _pack(second, (at + x8 + h8, 0, inter, _F32) if floats else between, at + x8, M, down, (out.data_ptr(), 0, out.stride(0)), _OUT[out.dtype], 0, 0.0, stream, _PIECE)
    f = _functions.get("brolm_fp8_two")
    if f is None:
        f = _functions["brolm_fp8_two"] = _fn("fp8_rows", "brolm_fp8_two", [c_char_p, c_void_p, c_char_p, c_void_p])
    launch = lambda streamed: _launcher("fp8_stream", "brolm_fp8_stream") if streamed else _launcher("fp8_gemm", "brolm_fp8_gemm")
    _check(f(a, launch(first[0]), b, launch(second[0])), "feedforward_fp8")
    add_launches(1 + (1 if x8 else 0) + (1 if floats and h8 else 0))
    if gate_up.fresh or down.fresh:
        _launched(stream, gate_up, down)


# --- routed experts -----------------------------------------------------------
def experts_fp8_rows(pairs: int, experts: int) -> int:
    """How many rows a tile of an expert's pairs has: 16 or 32 with the experts' matrices streamed, 256 on pairs of SMs.  32 experts
    of 2,048 x 1,024, 4 a token, with 16 / 32 / 256: 128 tokens (16 pairs an expert) 58 / 58 / 72 us, 256 73 / 70 / 77, 384 (48) 83 /
    77 / 78, 512 98 / 89 / 79; 8 experts, 2 a token: 128 (32) 30 / 28 / 31, 192 (48) 36 / 33 / 34."""
    mean = pairs / max(experts, 1)
    return 16 if mean <= 16 else 32 if mean <= 48 else 256


def _experts_checked(what: str, x, ids, up: Fp8Matrix, down: Fp8Matrix, scale) -> None:
    device = x.get_device()
    if x.dtype in _CODES and device >= 0 and device == _device() and x.dim() == 2 and ids.dim() == 2 and x.stride(1) == 1 \
            and len(up.shape) == 3 and len(down.shape) == 3 and not down.gated and up.shape[0] == down.shape[0] <= 4096 and up.outputs == down.cols \
            and x.shape[1] == up.cols and ids.shape[0] == x.shape[0] and ids.dtype == torch.int32 and ids.is_contiguous() \
            and device == ids.get_device() == up.index == down.index \
            and (scale is None or (scale.dtype == _F32 and scale.shape == ids.shape and scale.is_contiguous() and scale.get_device() == device)):
        return
    _refuse(what, x, "x")
    if len(up.shape) != 3 or len(down.shape) != 3 or down.gated or up.shape[0] != down.shape[0] or up.outputs != down.cols:
        raise KernelError(f"{what}: stacks of shapes {up.shape} and {down.shape} do not follow one another")
    if up.shape[0] > 4096:
        raise KernelError(f"{what}: {up.shape[0]} experts are more than 4,096")
    if x.shape[1] != up.cols:
        raise KernelError(f"{what}: rows of {up.cols} numbers are wanted, not {tuple(x.shape)}")
    if ids.dim() != 2 or ids.shape[0] != x.shape[0] or ids.dtype != torch.int32 or not ids.is_contiguous():
        raise KernelError(f"{what}: ids are a packed int32 [tokens, top]")
    if scale is not None and (scale.dtype != _F32 or scale.shape != ids.shape or not scale.is_contiguous()):
        raise KernelError(f"{what}: the pairs' numbers are a packed float32 [tokens, top]")
    for t in (ids, up, down, scale):
        if t is not None and t.device != x.device:
            raise KernelError(f"{what}: tensors on {x.device} and {t.device}")


def _experts(what: str, x, ids, up: Fp8Matrix, down: Fp8Matrix, pairs, out, activation: str, limit: float, scale, weights) -> None:
    act = _act_code(what, up, activation)
    E, (T, top), K, inter, N = up.shape[0], ids.shape, up.cols, down.cols, down.rows
    P = T * top
    if not P or not E or not N:
        return
    rows = experts_fp8_rows(P, E)
    most = (P + rows - 1) // rows + min(E, P)
    up512 = lambda n: (n + 511) & -512
    # the order and the list; the rows of both products in 8 bits with a tile of scales for every tile of the list
    need = 3 * up512(4 * P) + up512(4 * E + 8) + 2 * up512(4 * most)
    for cols in (K, inter):
        need += up512(P * ((cols + 15) & -16)) + ((rows + 127) >> 7) * most * ((cols + 511) >> 9) * _TILE
    held = None
    if pairs is None:
        held = torch.empty(need + 4 * P * N, dtype=torch.uint8, device=x.device)
        y = held.data_ptr() + need
    else:
        held, y = torch.empty(need, dtype=torch.uint8, device=x.device), pairs.data_ptr()
    product = _launcher("fp8_gemm", "brolm_fp8_gemm") if rows == 256 else _launcher("fp8_stream", "brolm_fp8_stream")
    pack = _EXPERTS.pack(x.data_ptr(), ids.data_ptr(), scale.data_ptr() if scale is not None else 0, weights.data_ptr() if weights is not None else 0,
                         up.packed[0], up.packed[1], down.packed[0], down.packed[1], y, out.data_ptr() if out is not None else 0, held.data_ptr(),
                         _raw_stream(x.get_device()), product, x.stride(0), up.packed[2], down.packed[2], out.stride(0) if out is not None else 0, need,
                         _CODES[x.dtype], T, top, E, K, inter, N, up.group_rows, down.group_rows, 1 if up.gated else 0, act, rows, _PIECE,
                         1 if out is not None and out.dtype == _F32 else 0, limit)
    _call("fp8_experts", "brolm_fp8_experts", pack, what)
    # (a call counts as one launch: the others of this pass)
    add_launches((1 if P > 256 or E > 256 else 0) + 2 + (1 if out is not None else 0))


def experts_fp8_pairs(x: torch.Tensor, ids: torch.Tensor, up: Fp8Matrix, down: Fp8Matrix, out: torch.Tensor, activation: str = "silu",
                      limit: float = 0.0, scale: Optional[torch.Tensor] = None) -> None:
    """Every (token, choice) pair through its expert: out float32 [top, tokens, down.rows], a pair's result at [its choice, its
    token].  ``ids`` int32 [tokens, top]: a number that is no expert's has no result (its place stays as it was).  ``up`` a stack
    [experts, ...], gated or not, ``down`` the stack of the second matrices; ``scale`` float32 [tokens, top] multiplies a pair's
    sums before the activation."""
    what = "experts_fp8"
    _experts_checked(what, x, ids, up, down, scale)
    if tuple(out.shape) != (ids.shape[1], x.shape[0], down.rows) or out.dtype != _F32 or not out.is_contiguous() or out.device != x.device:
        raise KernelError(f"{what}: the pairs' results are a packed float32 {(ids.shape[1], x.shape[0], down.rows)} on {x.device}")
    _experts(what, x, ids, up, down, out, None, activation, limit, scale, None)


def experts_fp8(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, up: Fp8Matrix, down: Fp8Matrix, out: torch.Tensor, activation: str = "silu",
                limit: float = 0.0, scale_input: bool = False) -> None:
    """out [tokens, down.rows] (float32 or bfloat16) = the sum over a token's choices of ``weights`` times its expert's result, in
    the order of the choices; a number in ``ids`` that is no expert's adds nothing.  With ``scale_input`` the weight multiplies
    the sums before the activation and not the result."""
    what = "experts_fp8"
    _experts_checked(what, x, ids, up, down, weights)
    if out.dtype not in _CODES or out.dim() != 2 or out.get_device() != x.get_device() or (out.stride(1) != 1 and down.rows > 1):
        _refuse(what, out, "out")
    if out.shape[0] != x.shape[0] or out.shape[1] != down.rows or (out.shape[0] > 1 and out.stride(0) < down.rows):
        raise KernelError(f"{what}: the result has the shape {(x.shape[0], down.rows)}, not {tuple(out.shape)} (strides {tuple(out.stride())})")
    if ids.shape[1] == 0 or up.shape[0] == 0:
        out.zero_()
        return
    _experts(what, x, ids, up, down, None, out, activation, limit, weights if scale_input else None, None if scale_input else weights)


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
