"""The 8-bit cache without a GPU: the plain restatement's own properties, and what the entry points refuse."""
import math
import random

import pytest
import torch

from brolm_b200 import kernels
from tests.plain import kv8_plain as plain

I32 = torch.int32


def test_scale_is_the_least_power_of_two_that_holds_the_block():
    for amax in (127.0, 126.99, 127.01, 254.0, 1.0, 3.4e38, 1e-37, 1e-45, 0.0):
        s = plain.scale_of(amax)
        assert math.frexp(s)[0] == 0.5 and amax <= 127 * s
        assert s == 2.0 ** -126 or amax > 127 * s / 2
    assert math.isnan(plain.scale_of(math.inf)) and math.isnan(plain.scale_of(math.nan))


def test_a_block_that_grows_token_by_token_is_off_by_less_than_one_step():
    g = torch.Generator().manual_seed(0)
    for trial in range(20):
        x = torch.randn((32, 1, 16), generator=g) * torch.exp2(torch.arange(32) * (trial / 8.0))[:, None, None]
        pages, scales = torch.zeros((1, 1, 32, 16), dtype=torch.float64), torch.zeros((1, 1), dtype=torch.float64)
        for t in range(32):
            plain.write(x[t:t + 1], [t], pages, scales)
        off = (pages[0, 0] * scales[0, 0] - x[:, 0].double()).abs().max()
        assert off < scales[0, 0], trial


def test_extend_hands_out_every_block_once():
    rng = random.Random(5)
    block, ring, S, N = 32, 128, 9, 40
    free, count = list(range(N)), N
    tables, held, lengths = [[0] * 12 for _ in range(S)], [0] * S, [0] * S
    for _ in range(30):
        rows = rng.sample(range(S), rng.randint(1, S))
        new = [rng.randint(0, 60) for _ in rows]
        r = 0 if rng.random() < 0.5 else ring
        if not r and any(plain.need(lengths[s] + n, block) > 12 for s, n in zip(rows, new)):
            continue
        status, *_, tables, held, count = plain.extend(rows, [lengths[s] for s in rows], new, tables, held, free, count, block, r, 1000)
        if status == 0:
            for s, n in zip(rows, new):
                lengths[s] += n
        out = [b for t, h in zip(tables, held) for b in t[:h]]
        assert sorted(out + free[:count]) == list(range(N))


def _cache(n=4, G=2, P=32, D=32):
    pages = lambda: torch.zeros((n, G, P, D), dtype=torch.int8)
    return [pages(), pages(), torch.zeros((n, G)), torch.zeros((n, G))]


def _i(*v):
    return torch.tensor(v, dtype=I32)


@pytest.mark.parametrize("change", ["dtype", "shape", "scales", "strides", "pages", "k", "tokens", "rows", "cpu"])
def test_write_refusals(change):
    cache = _cache()
    k, v = torch.zeros((3, 2, 32)), torch.zeros((3, 2, 32))
    args = dict(cu_q=_i(0, 3), positions=_i(0, 1, 2), cache_rows=_i(0, 1, 2))
    if change == "dtype":
        k = k.half()
    elif change == "shape":
        cache[1] = cache[1][:, :, :, :16].contiguous()
    elif change == "scales":
        cache[2] = cache[2].double()
    elif change == "strides":
        k = torch.zeros((3, 32, 2)).transpose(1, 2)
    elif change == "pages":
        cache[0] = cache[0].float()
    elif change == "k":
        k = torch.zeros((3, 4, 32))
    elif change == "tokens":
        args["positions"] = _i(0, 1)
    elif change == "rows":
        args["cache_rows"] = args["cache_rows"].long()
    with pytest.raises(kernels.KernelError):
        kernels.kv8_write(k, v, *args.values(), *cache, max_q_len=3)


@pytest.mark.parametrize("change", ["heads", "ring", "ring_all", "out", "lens", "tables", "stride", "cpu"])
def test_attention_refusals(change):
    cache = _cache()
    q = torch.zeros((3, 4 * 32))
    kw = dict(n_kv=2, group=2, head_dim=32, scale=1.0, cap=0.0, window=0, ring=0, batch=1, max_q_len=3, max_kv_len=3)
    pos = dict(out=torch.zeros_like(q), cu_q=_i(0, 3), kv_len=_i(3), slots=_i(0), tables=torch.zeros((1, 4), dtype=I32))
    if change == "heads":
        kw["n_kv"], kw["group"] = 4, 1
    elif change == "ring":                       # one key short of what three tokens under a window of 32 need
        kw.update(window=32 + 1, ring=64)
    elif change == "ring_all":
        kw.update(window=0, ring=64)
    elif change == "out":
        pos["out"] = torch.zeros((3, 4 * 32), dtype=torch.bfloat16)
    elif change == "lens":
        pos["kv_len"] = _i(3, 3)
    elif change == "tables":
        pos["tables"] = torch.zeros(4, dtype=I32)
    elif change == "stride":
        q = torch.zeros((4 * 32, 3)).t()
    with pytest.raises(kernels.KernelError, match="ring" if change.startswith("ring") else None):
        kernels.attention_kv8(q, *pos.values(), *cache, **kw)


@pytest.mark.parametrize("change", ["lengths", "cu_q", "tables", "free", "status", "cpu"])
def test_extend_and_release_refusals(change):
    pos = dict(slots=_i(0), lengths=_i(0), new=_i(2), tables=torch.zeros((2, 3), dtype=I32), held=_i(0, 0), free=_i(0, 1, 2),
               free_count=_i(3))
    out = dict(cu_q=_i(0, 0), kv_len=_i(0), positions=_i(0, 0), tok_seq=_i(0, 0), cache_rows=_i(0, 0), status=_i(0))
    if change == "lengths":
        pos["lengths"] = _i(0, 0)
    elif change == "cu_q":
        out["cu_q"] = _i(0)
    elif change == "tables":
        pos["tables"] = pos["tables"][:, :2]
    elif change == "free":
        pos["free"] = pos["free"].long()
    elif change == "status":
        out["status"] = _i(0, 0)
    with pytest.raises(kernels.KernelError):
        kernels.blocks_extend(*pos.values(), block=32, **out)
    if change in ("tables", "free", "status", "cpu"):
        with pytest.raises(kernels.KernelError):
            kernels.blocks_release(pos["slots"], pos["tables"], pos["held"], pos["free"], pos["free_count"], status=out["status"])


def test_calls_are_counted_as_launches(monkeypatch):
    """What the engine looks at to know whether anything ran since its last check, and what a captured step adds a replay."""
    from brolm_b200.kernels import kv8
    results = {"good": 0, "bad": 10002}
    for name, status in results.items():
        monkeypatch.setitem(kv8._functions, name, lambda packed, status=status: status)
    before = kernels.launch_count()
    kv8._call("kv8", "good", b"", "a call")
    assert kernels.launch_count() == before + 1
    with pytest.raises(kernels.KernelError, match="a call"):
        kv8._call("kv8", "bad", b"", "a call")
    assert kernels.launch_count() == before + 1


def test_what_an_earlier_launch_may_still_be_writing_is_not_read_as_constant():
    """The kernels are let in before the launch ahead of them has ended, so what that one writes is not constant for as long
    as they are resident: no load of theirs may go past the ordinary caches' order, by intrinsic, by PTX or by __restrict__."""
    import os
    import re
    folder = os.path.join(os.path.dirname(__file__), "..", "brolm_b200", "csrc")
    for name in ("blocks.cu", "kv8.cu", "attn_kv8.cu", "attn_kv8_tc.cu", "attn_kv8_join.cuh"):
        with open(os.path.join(folder, name)) as fh:
            assert not re.search(r"__ldg\b|ld\.global\S*\.nc|__restrict__", fh.read()), name
