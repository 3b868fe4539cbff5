"""When a product may read its matrix ahead of what runs before it, and what a matrix keeps, on the CPU: the launchers are replaced."""
import copy
import os
import pickle

import pytest
import torch

from brolm_b200 import kernels
from brolm_b200.kernels import fp8
from brolm_b200.kernels.build import CSRC

MAKER, OTHER = 11, 22          # two streams


class Launches:
    """Stands for the device: which stream is current, whether it is capturing, and the products' structs as they were launched."""

    def __init__(self, monkeypatch):
        self.stream, self.capturing, self.fails, self.products = MAKER, False, False, []
        monkeypatch.setattr(fp8, "_raw_stream", lambda device: self.stream)
        monkeypatch.setattr(fp8, "_device", lambda: 0)
        monkeypatch.setattr(fp8, "device_sms", lambda device: 148)
        monkeypatch.setattr(fp8, "_checked", lambda *args: None)
        monkeypatch.setattr(fp8, "add_launches", lambda n: None)
        monkeypatch.setattr(fp8, "_launcher", lambda lib, name: 1)
        monkeypatch.setattr(fp8, "_call", lambda lib, name, packed, what: self.launch(packed))
        monkeypatch.setitem(fp8._functions, "brolm_fp8_two", lambda a, first, b, second: self.launch(a, b))
        monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: self.capturing)

    def launch(self, *products):
        if self.fails:
            raise kernels.KernelError("refused")
        self.products += products
        return 0

    def waits(self):
        """Of the products launched since the last look: whether each waits before it reads its matrix."""
        said = [bool(fp8._PRODUCT.unpack(p)[-1]) for p in self.products]
        self.products = []
        return said


@pytest.fixture
def device(monkeypatch):
    return Launches(monkeypatch)


def matrix(rows, cols, gated=False):
    m = fp8._empty((rows, cols), "cpu", gated)
    m.index, m.stream = 0, MAKER
    return m


def product(w):
    kernels.linear_fp8(matrix(3, w.cols), w, torch.zeros(3, w.outputs))


def test_the_first_product_waits_and_later_ones_do_not(device):
    w = matrix(64, 256)
    product(w)
    product(w)
    assert device.waits() == [True, False]


def test_a_product_on_another_stream_leaves_the_matrix_new_for_the_one_that_made_it(device):
    w = matrix(64, 256)
    device.stream = OTHER
    product(w)
    device.stream = MAKER
    product(w)
    device.stream = OTHER
    product(w)
    assert device.waits() == [True, True, False]


def test_a_captured_product_leaves_the_matrix_new(device):
    w = matrix(64, 256)
    device.capturing = True
    product(w)
    product(w)
    device.capturing = False
    product(w)
    product(w)
    assert device.waits() == [True, True, True, False]


def test_a_refused_launch_leaves_the_matrix_new(device):
    w, up, down = matrix(64, 256), matrix(2 * 128, 256, True), matrix(64, 128)
    device.fails = True
    with pytest.raises(kernels.KernelError):
        product(w)
    with pytest.raises(kernels.KernelError):
        kernels.feedforward_fp8(matrix(3, 256), up, down, torch.zeros(3, 64), "silu")
    device.fails = False
    product(w)
    kernels.feedforward_fp8(matrix(3, 256), up, down, torch.zeros(3, 64), "silu")
    kernels.feedforward_fp8(matrix(3, 256), up, down, torch.zeros(3, 64), "silu")
    assert device.waits() == [True, True, True, False, False]


def test_what_a_product_says_of_its_matrix_is_what_it_found(device):
    """Two threads with a new matrix: the second packs before the first has launched."""
    w = matrix(64, 256)
    seen = []
    launch = device.launch

    def between(*products):
        if not seen:
            seen.append(w.fresh)
            product(w)                                   # (the other thread's whole call)
        return launch(*products)
    device.launch = between
    product(w)
    assert seen == [True] and device.waits() == [True, True]


@pytest.mark.parametrize("source", ["fp8_stream.cu", "fp8_gemm.cu"])
def test_the_thread_that_lets_the_next_kernel_begin_has_waited(source):
    """One thread's trigger stands for its block.  The products have the loader's, and the loader waits on every way to it (in the
    stream on one of two: ahead of its first loads, or behind those of the matrix); the stream also has that of the warps that round
    rows, all of whose threads wait before they read one."""
    with open(os.path.join(CSRC, source)) as f:
        kernel = f.read().split("__global__", 1)[1].split("\n}\n", 1)[0]
    loader, rest = kernel[kernel.index("if (warp == 0) {"):].split("} else if (warp == 1) {", 1)
    ahead = loader[:loader.rindex("pdl_trigger()")]
    if source == "fp8_gemm.cu":
        assert kernel.count("pdl_trigger()") == 1 and "\n            pdl_wait();\n" in ahead        # (at the loader's own level: on every way)
        return
    assert kernel.count("pdl_trigger()") == 3
    wait = "auto wait = [&]() {\n                pdl_wait();\n                if (AT_ONCE) pdl_trigger();\n            };\n"
    ways = ahead.split(wait)
    assert len(ways) == 2 and "pdl_trigger()" not in ways[0] + ways[1]
    assert ways[1].startswith("            if (!ahead) wait();\n") and ways[1][ways[1].index("if (ahead) {"):].count("\n                wait();\n") == 1
    rounding = rest[rest.index("const int quarter = warp & 3;"):rest.index("pdl_trigger()")]
    assert "\n        if (EXPERTS || FUSED) pdl_wait();\n        if (FUSED) {\n" in rounding
    assert "\n        }\n" not in rounding[rounding.index("if (FUSED) {"):]        # the trigger is in that branch


@pytest.mark.parametrize("how", [copy.deepcopy, copy.copy, lambda m: pickle.loads(pickle.dumps(m))])
def test_a_copy_of_a_matrix_lies_where_its_own_data_does(how):
    """A copied model's products read the copy's memory, not that of a matrix which may be gone."""
    for m in (fp8._empty((300, 1000), "cpu"), fp8._empty((5, 200, 130), "cpu"), fp8._empty((64, 40), "cpu", True)):
        m.data.copy_(torch.arange(m.data.numel()) % 251)
        c = how(m)
        assert (c.shape, c.gated, c.rows, c.cols, c.outputs, c.total) == (m.shape, m.gated, m.rows, m.cols, m.outputs, m.total)
        assert torch.equal(c.data, m.data) and c.fresh
        assert c.packed[0] == c.data.data_ptr() == c.values.data_ptr() and c.packed[1] == c.scales.data_ptr() and c.packed[2] == m.packed[2]


def test_a_matrix_copied_with_what_holds_it():
    class Part:
        pass
    p = Part()
    p.w = fp8._empty((300, 1000), "cpu")
    q = copy.deepcopy(p)
    assert q.w is not p.w and q.w.packed[0] == q.w.data.data_ptr() != p.w.packed[0]


@pytest.mark.parametrize("data", [torch.zeros(63 * 256 + 512, dtype=torch.uint8), torch.zeros(64 * 256 + 511, dtype=torch.uint8), torch.zeros(64 * 256 + 512),
                                  torch.zeros(2 * (64 * 256 + 512), dtype=torch.uint8)[::2], torch.zeros(2, 64 * 256 + 512, dtype=torch.uint8)])
def test_a_matrix_of_too_little_or_other_data_is_refused(data):
    """64 rows of 256 columns: 64 * 256 bytes of values and 512 of scales."""
    with pytest.raises(kernels.KernelError, match="Fp8Matrix"):
        kernels.Fp8Matrix(data, (64, 256))


@pytest.mark.parametrize("shape, gated", [((64,), False), ((2, 2, 2, 2), False), ((64, 0), False), ((63, 256), True), ((-1, 256), False)])
def test_a_matrix_of_no_such_shape_is_refused(shape, gated):
    with pytest.raises(kernels.KernelError, match="Fp8Matrix"):
        kernels.Fp8Matrix(torch.zeros(1 << 16, dtype=torch.uint8), shape, gated)


def test_gate_and_partner_are_matrices():
    with pytest.raises(kernels.KernelError, match="fp8_gate_up"):
        kernels.fp8_gate_up(torch.zeros(64), torch.zeros(64))
