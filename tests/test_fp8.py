"""Products in 8-bit floating point: the oracle itself, the rules and the refusals, on the CPU."""
import math

import pytest
import torch

from brolm_b200 import kernels
from brolm_b200.kernels import fp8
from tests.plain import fp8_plain as plain


def test_numbers_of_the_format():
    assert len(plain.E4M3) == 127 and plain.E4M3[-1] == 448.0 and plain.E4M3[1] == 2.0 ** -9
    every = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    assert sorted(every.tolist()) == plain.E4M3


def test_oracle_rounds_like_a_cast():
    g = torch.Generator().manual_seed(3)
    u = torch.randn(20000, generator=g).double() * torch.exp2(torch.randint(-12, 8, (20000,), generator=g).double())
    u = torch.cat([u.clamp(-448, 448), torch.tensor(plain.E4M3), (torch.tensor(plain.E4M3)[1:] + torch.tensor(plain.E4M3)[:-1]) / 2])
    u = u.float().double()
    assert torch.equal(plain.nearest(u), u.float().to(torch.float8_e4m3fn).double())


@pytest.mark.parametrize("most, scale", [(448.0, 1.0), (448.1, 2.0), (447.9, 1.0), (224.0, 0.5), (224.1, 1.0), (0.0, 2.0 ** -127), (1e-45, 2.0 ** -127),
                                         (2.0 ** -126, 2.0 ** -127), (3.4e38, 2.0 ** 120)])
def test_scale(most, scale):
    assert plain.scale_of(most) == scale


@pytest.mark.parametrize("tiles, nkb", [(18, 72), (18, 18), (32, 18), (36, 288), (144, 18), (7, 8), (1, 1), (1, 2), (3, 5), (400, 9), (18, 7)])
def test_slices_hold_all_blocks_and_none_is_empty(tiles, nkb):
    s = fp8.fp8_slices(tiles, nkb, 148)
    per = (nkb + s - 1) // s
    assert 1 <= s <= 8 and (s - 1) * per < nkb <= s * per and (s == 1 or tiles * s <= 259)


def _matrix(rows, cols, gated=False):
    m = fp8._empty((rows, cols), "cpu", gated)
    return m


def test_layout():
    m = _matrix(300, 1000)
    assert m.values.shape == (300, 1008) and m.scales.shape == (3, 2, 512) and (m.rows, m.cols, m.outputs) == (300, 1000, 300)
    e = fp8._empty((5, 200, 130), "cpu")
    assert e.values.shape == (5 * 256, 144) and e.scales.shape == (10, 1, 512) and e.group_rows == 256


def test_refusals():
    w = _matrix(64, 256)
    with pytest.raises(kernels.KernelError, match="CUDA"):
        kernels.fp8_quantize(torch.zeros(2, 128))
    with pytest.raises(kernels.KernelError, match="float64"):
        kernels.fp8_quantize(torch.zeros(2, 128, dtype=torch.float64))
    with pytest.raises(kernels.KernelError, match="relu2"):
        kernels.linear_fp8(_matrix(3, 256), w, torch.zeros(3, 64), "silu")
    with pytest.raises(kernels.KernelError, match="256 numbers"):
        kernels.linear_fp8(_matrix(3, 128), w, torch.zeros(3, 64))
    with pytest.raises(kernels.KernelError, match="follow"):
        kernels.feedforward_fp8(_matrix(3, 256), _matrix(500, 256, True), w, torch.zeros(3, 64))
    with pytest.raises(kernels.KernelError, match="experts"):
        kernels.linear_fp8(_matrix(3, 256), fp8._empty((2, 64, 256), "cpu"), torch.zeros(3, 64))
    with pytest.raises(kernels.KernelError, match="two matrices"):
        kernels.fp8_gate_up(torch.zeros(4, 8), torch.zeros(4, 9))


def test_model_refuses_other_types():
    import brolm_b200 as bb
    from tests.helpers import TINY_A
    with pytest.raises(ValueError, match="weight_dtype"):
        bb.Model(bb.Gemma2Config(**TINY_A), device="cpu", weight_dtype="int4")
    with pytest.raises(kernels.KernelError, match="CUDA"):
        bb.Model(bb.Gemma2Config(**TINY_A), device="cpu", weight_dtype="fp8").init_random(0)


@pytest.mark.parametrize("rows, w_rows, nkb, streamed", [(1, 100, 1, True), (64, 18432, 18, True), (65, 18432, 18, False), (128, 18432, 18, False), (128, 2304, 72, True),
                                                         (128, 28672, 28, True), (128, 1000, 5, False), (129, 2304, 72, False)])
def test_which_products_stream_their_matrix(rows, w_rows, nkb, streamed):
    assert fp8.fp8_streamed(rows, w_rows, nkb, 148) is streamed


@pytest.mark.parametrize("pairs, experts, rows", [(1, 32, 16), (512, 32, 16), (513, 32, 32), (1536, 32, 32), (1537, 32, 256), (5, 1, 16), (100000, 8, 256), (3, 0, 16)])
def test_rows_of_an_experts_tile(pairs, experts, rows):
    assert fp8.experts_fp8_rows(pairs, experts) == rows


def test_which_rows_a_norm_can_leave_in_8_bits():
    assert [n for n in (0, 2, 4, 6, 100, 2304, 4608, 8190, 8192, 8196) if kernels.residual_rmsnorm_fp8_ok(n)] == [4, 100, 2304, 4608, 8192]


def test_a_norm_in_8_bits_refuses_tensors_of_the_host():
    h = torch.zeros(2, 64)
    with pytest.raises(kernels.KernelError, match="CUDA"):
        kernels.residual_rmsnorm_fp8(h, h.clone(), None, 1e-6, 0.0, torch.ones(64), 1e-6, 0.0)
