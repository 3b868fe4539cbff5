"""Engines whose cache is in 8 bits: page tables made on the device, prompts at once and in pieces, decoding."""
import numpy as np
import pytest
import torch

import brolm_b200 as bb
from brolm_b200 import kernels
from tests.helpers import TINY, make_folder, oracle_inputs, random_prompts
from tests.plain import kv8_plain
from tests.plain.gemma2_stepwise import StepwiseGemma2

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
# a head of 256 entries and two layer kinds, the sizes of which the tensor-core kernels take
WIDE = dict(vocab_size=300, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
            head_dim=256, rope_theta=10000.0, sliding_window=100, attn_logit_softcapping=50.0, final_logit_softcapping=30.0,
            query_pre_attn_scalar=256, rms_norm_eps=1e-6, max_position_embeddings=1024)
# A number is off by at most a step of its block, under 2/127 of the block's largest, and mostly by far less than half of one;
# over two or three layers the logits stay within a tenth of their norm.
NEAR = 0.1


def build(name="B", dtype="float32"):
    cfg, seed, std = (WIDE, 5, 0.05) if name == "wide" else TINY[name]
    return bb.Model(bb.Gemma2Config(**cfg), dtype=dtype, device=DEV).init_random(seed=seed, weight_std=std, norm_std=0.1)


def both(model, max_tokens, **kw):
    plain = {k: v for k, v in kw.items() if k != "max_piece"}
    return bb.Engine(model, max_tokens, **plain), bb.Engine(model, max_tokens, cache_dtype="int8", **kw)


def near(a, b):
    off = float((a.double() - b.double()).norm() / b.double().norm())
    assert off <= NEAR, off
    return off


def check_tables(engine):
    """The device's tables hold as many pages a slot as the host has counted, nothing twice, and the rest is free."""
    for g in engine.cache.kv_groups:
        t = g.tables
        held, tables, free = t.held.tolist(), t.tables.tolist(), t.free.tolist()
        count = int(t.free_count)
        live = {s: len(p) for s, p in g.pages.items()}
        assert all(held[s] == live.get(s, 0) for s in range(len(held))), (held, live)
        out = [p for row, n in zip(tables, held) for p in row[:n]]
        assert sorted(out + free[:count]) == list(range(g.pool.num_pages)) and count == g.pool.free_pages
        assert int(t.status) == 0


@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("B", "bfloat16"), ("wide", "bfloat16"), ("wide", "float32")])
def test_prompts_and_decoding_beside_a_cache_of_the_models_type(name, dtype):
    model = build(name, dtype)
    vocab = model.config.vocab_size
    plain, int8 = both(model, 64 * 40, max_slots=6)
    prompts = random_prompts(vocab, [5, 130, 64, 1], seed=1)
    more = torch.randint(0, vocab, (4, 90), generator=torch.Generator().manual_seed(2)).tolist()
    slots = [e.open(4) for e in (plain, int8)]
    a, b = (e.step(s, prompts) for e, s in zip((plain, int8), slots))
    assert torch.equal(a, b)                               # a prompt attends to its own keys, whatever is kept of them
    check_tables(int8)
    for t in range(90):
        tokens = [[row[t]] for row in more]
        a, b = (e.step(s, tokens) for e, s in zip((plain, int8), slots))
        near(b, a)
    check_tables(int8)
    # half the bytes a place, but for the scales and the page more that a window's ring has
    places = lambda e: sum(g.k.shape[0] * g.pool.num_pages for g in e.cache.kv_groups) * 64
    per_place = model.config.num_key_value_heads * model.config.head_dim * 2
    scales = sum(2 * g.k_scale.numel() * 4 for g in int8.cache.kv_groups)
    assert int8.cache.bytes() == places(int8) * per_place + scales
    assert plain.cache.bytes() == places(plain) * per_place * (2 if dtype == "bfloat16" else 4)
    int8.close(slots[1][1:3])
    check_tables(int8)
    again = int8.open(2)
    x = int8.step(again, prompts[1:3])
    plain.close(slots[0])
    y = plain.step(plain.open(2), prompts[1:3])
    assert torch.equal(x, y)
    int8.close([slots[1][0], slots[1][3]] + again)
    check_tables(int8)


def test_the_first_layers_keys_and_values_are_the_projected_ones():
    """Layer 0 sees the embedding alone, so its keys and values do not depend on the cache: what the 8-bit one holds is
    theirs to half a step."""
    model = build("B", "float32")
    plain, int8 = both(model, 1024)
    prompt = random_prompts(model.config.vocab_size, [150], seed=3)
    sp, si = plain.open(1), int8.open(1)
    plain.step(sp, prompt)
    int8.step(si, prompt)
    ep, ei = plain.cache.entry(1), int8.cache.entry(1)    # entry 1 keeps all keys; both layers before it saw no cache
    ep = plain.cache.entry(0) if ep.group.ring else ep
    ei = int8.cache.entry(0) if ei.group.ring else ei
    page = plain.cache.page_size
    ids = plain.cache.kv_groups[ep.group_id].pages[sp[0]]
    G, D = ep.group.spec.n_kv, ep.group.spec.head_dim
    k, v = torch.empty((2, 150, G, D), device=DEV)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)
    t = ei.group.tables
    kernels.kv8_read(i32(0, 150), i32(150), i32(*si), t.tables, ei.k, ei.v, *ei.scales, k, v, max_q_len=150)
    for got, pages, scale in ((k, ep.k, ei.scales[0]), (v, ep.v, ei.scales[1])):
        want = torch.cat([pages[p] for p in ids], dim=1)[:, :150].transpose(0, 1)
        step = torch.cat([scale[t.tables[si[0], j]][None].expand(page, -1) for j in range(len(ids))])[:150]
        assert bool(((got - want).abs() <= 0.5 * step[:, :, None]).all()) and float(want.abs().max()) > 0


@pytest.mark.parametrize("name,dtype", [("B", "float32"), ("wide", "bfloat16")])
def test_captured_steps_give_the_bits_of_uncaptured_ones(name, dtype, monkeypatch):
    # (a captured step's bound on the lengths is a power of two, so it may share the keys out otherwise: here neither does)
    monkeypatch.setattr(kernels.kv8, "kv8_shares", lambda *a: (1, 1))
    model = build(name, dtype)
    prompts = random_prompts(model.config.vocab_size, [70, 3, 129], seed=4)
    results = []
    for graphs in (True, False):
        e = bb.Engine(model, 64 * 20, max_slots=3, cache_dtype="int8", use_graphs=graphs)
        s = e.open(3)
        logits, out = e.step(s, prompts), []
        for _ in range(70):
            ids = logits.argmax(dim=1).to(torch.int32)
            out.append(logits.clone())
            logits = e.step_from(s, ids, [0, 1, 2])
        results.append(torch.stack(out))
        check_tables(e)
    assert torch.equal(*results)


@pytest.mark.parametrize("name,dtype", [("B", "float32"), ("wide", "bfloat16")])
def test_captured_steps_whose_clusters_are_dealt_out(name, dtype, monkeypatch):
    """Who gets how many hangs on the lengths alone, which a captured step reads anew: the same bits as uncaptured ones."""
    monkeypatch.setattr(kernels.kv8, "kv8_shares", lambda *a: (1, -20))
    model = build(name, dtype)
    prompts = random_prompts(model.config.vocab_size, [250, 3, 120], seed=14)
    results = []
    for graphs in (True, False):
        e = bb.Engine(model, 64 * 20, max_slots=3, cache_dtype="int8", use_graphs=graphs)
        s = e.open(3)
        logits, out = e.step(s, prompts), []
        for _ in range(40):
            ids = logits.argmax(dim=1).to(torch.int32)
            out.append(logits.clone())
            logits = e.step_from(s, ids, [0, 1, 2])
        results.append(torch.stack(out))
        check_tables(e)
    assert torch.equal(*results) and bool(torch.isfinite(results[0]).all())


@pytest.mark.parametrize("name,dtype,most", [("A", "float32", 50), ("B", "bfloat16", 7), ("wide", "bfloat16", 200), ("wide", "float32", 64)])
def test_prompts_in_pieces(name, dtype, most):
    """A prompt brought a piece at a time, beside sequences that go on by one token and that begin."""
    model = build(name, dtype)
    vocab = model.config.vocab_size
    plain, int8 = both(model, 64 * 40, max_slots=4, max_piece=most)
    tokens = random_prompts(vocab, [400, 90, 30], seed=6)
    sp, si = plain.open(3), int8.open(3)
    whole = plain.step(sp, tokens)
    at = [0, 0, 0]
    int8.step(si[:1], [tokens[0][:most]])
    at[0] = most
    last = {}
    while any(at[i] < len(tokens[i]) for i in range(3)):
        now = [i for i in range(3) if at[i] < len(tokens[i])]
        sizes = [min(len(tokens[i]) - at[i], (most, max(1, most // 3), 1)[i]) for i in now]
        logits = int8.step([si[i] for i in now], [tokens[i][at[i]:at[i] + n] for i, n in zip(now, sizes)])
        for r, (i, n) in enumerate(zip(now, sizes)):
            at[i] += n
            last[i] = logits[r].clone()
    check_tables(int8)
    near(torch.stack([last[i] for i in range(3)]), whole)
    with pytest.raises(bb.StepError, match="max_piece"):
        int8.step(si[:2], [[1] * (most + 1), [2]])
    check_tables(int8)


def test_steps_and_closing_on_streams_that_change():
    model = build("wide", "bfloat16")
    prompts = random_prompts(model.config.vocab_size, [300, 65], seed=8)

    def run(streams):
        e = bb.Engine(model, 64 * 9, max_slots=2, cache_dtype="int8")
        out, turn = [], 0
        for _ in range(3):
            for what in ("prompt", "decode", "decode", "close"):
                st = streams[turn % len(streams)]
                turn += 1
                with torch.cuda.stream(st):
                    if what == "prompt":
                        s = e.open(2)
                        logits = e.step(s, prompts)
                    elif what == "decode":
                        logits = e.step(s, [[7], [9]])
                    else:
                        e.close(s)
                        continue
                    out.append(logits.clone())
        torch.cuda.synchronize()
        check_tables(e)
        return out

    alone = run([torch.cuda.default_stream()])
    mixed = run([torch.cuda.Stream(), torch.cuda.default_stream(), torch.cuda.Stream()])
    assert all(torch.equal(a, b) for a, b in zip(alone, mixed))


def test_generation_and_the_command_line(capsys, tmp_path):
    import json
    from brolm_b200 import cli
    model = build("B", "bfloat16")
    prompts = random_prompts(model.config.vocab_size, [9, 40, 1, 77, 20], seed=9)
    opts = bb.GenerateOptions(max_new_tokens=70, sampling=bb.SamplingParams(temperature=0.0), stop_on_eos=False)
    e = bb.Engine(model, 64 * 12, max_slots=3, cache_dtype="int8")
    outs = bb.generate(e, prompts, eos_id=-1, opts=opts)
    assert [len(o) for o in outs] == [70] * 5 and e.cache.live_slots == 0
    check_tables(e)
    s = e.open(1)
    logits, ids = e.step(s, prompts[3:4]), []
    for _ in range(70):
        ids.append(int(logits.argmax()))
        logits = e.step(s, [[ids[-1]]])
    # (a batch of its own cuts its keys otherwise: now and then another token is as likely)
    assert sum(a == b for a, b in zip(ids, outs[3])) >= 35
    config = tmp_path / "config.json"
    config.write_text(json.dumps(dict(TINY["A"][0], architectures=["Gemma2ForCausalLM"])))
    assert cli.main(["--random", "--config", str(config), "--ids", "5,6,7", "--max-new", "5", "--cache-dtype", "int8", "--no-eos"]) == 0
    assert "generated 5 tokens" in capsys.readouterr().out


class Quantised(StepwiseGemma2):
    """The stepwise restatement whose decode steps see keys and values as pages of 8 bits hold them.  A prompt sees its own
    as they are; then every page is rounded at once, and a page that goes on token by token as it grows."""

    def begin(self, tokens):
        rows = [self.push(t) for t in tokens]
        c = self.c
        G, D = int(c["num_key_value_heads"]), int(c["head_dim"])
        new = lambda: (torch.zeros((16, G, 64, D), dtype=torch.float64), torch.zeros((16, G), dtype=torch.float64))
        self.pages = [[new(), new()] for _ in range(self.n_layers)]
        self.lists = (self.keys, self.values)
        for layer in range(self.n_layers):
            for which, held in enumerate(self.lists):
                self.keep(layer, which, held[layer], 0)
        self.decoding = True
        return rows[-1]

    def keep(self, layer, which, new, first):
        pages, scales = self.pages[layer][which]
        x = torch.from_numpy(np.stack(new))
        kv8_plain.write(x, list(range(first, first + len(new))), pages, scales)
        held = self.lists[which][layer]
        for p in range(first // 64 * 64, len(held)):
            held[p] = (pages[p // 64, :, p % 64] * scales[p // 64][:, None]).numpy()

    def attend(self, layer, q):
        if getattr(self, "decoding", False):
            for which, held in enumerate(self.lists):
                self.keep(layer, which, held[layer][-1:], len(held[layer]) - 1)
        return super().attend(layer, q)


@pytest.mark.parametrize("name", ["A", "B"])
def test_decoding_against_the_stepwise_restatement_with_rounded_pages(name, tmp_path):
    """The engine's keys differ from the restatement's by float rounding, which now and then rounds a number to the other
    side, one step of some hundred numbers' largest: a hundredth of the logits' norm is more than all of that."""
    folder = make_folder(tmp_path, name)
    config, weights = oracle_inputs(folder)
    model = bb.load_model(folder, dtype="float32", device=DEV)
    e = bb.Engine(model, 64 * 12, max_slots=2, cache_dtype="int8", max_piece=3)
    prompts = random_prompts(config["vocab_size"], [70, 5], seed=11)
    more = torch.randint(0, config["vocab_size"], (2, 80), generator=torch.Generator().manual_seed(12)).tolist()
    oracles = [Quantised(config, weights) for _ in prompts]
    want = [o.begin(p) for o, p in zip(oracles, prompts)]
    s = e.open(2)
    got = e.step(s, prompts)
    for t in range(80):
        for i in range(2):
            ref = torch.from_numpy(want[i])
            off = float((got[i].cpu().double() - ref).norm() / ref.norm())
            assert off <= 0.01, (t, i, off)
        want = [o.push(row[t]) for o, row in zip(oracles, more)]
        got = e.step(s, [[row[t]] for row in more])


@pytest.mark.parametrize("graphs", [True, False])
def test_a_decode_step_that_the_tables_refuse_is_reported(graphs):
    """The device has fewer free pages than the host counts: the step that needs one is refused, the next is fine again; who
    closes the sequences (or begins another) learns of it, once, and the engine goes on."""
    model = build("B", "float32")
    e = bb.Engine(model, 64 * 12, max_slots=3, cache_dtype="int8", use_graphs=graphs)
    prompts = random_prompts(model.config.vocab_size, [64, 64], seed=4)
    for end in ("close", "step"):
        s = e.open(2)
        e.step(s, prompts)
        counts = [g.tables.free_count.clone() for g in e.cache.kv_groups]
        for g in e.cache.kv_groups:
            g.tables.free_count.zero_()
        e.step(s, [[1], [2]])                                    # the 65th token wants a page
        for g, n in zip(e.cache.kv_groups, counts):
            g.tables.free_count.copy_(n)
        for t in range(3):
            e.step(s, [[3], [4]])
        if end == "step":
            other = e.open(1)
            with pytest.raises(bb.StepError, match="refused a step.*too few free blocks"):
                e.step(other, [[5]])
            e.step(other, [[5]])
            e.close(other)
            e.close(s)
        else:
            with pytest.raises(bb.StepError, match="refused a step.*too few free blocks"):
                e.close(s)
        check_tables(e)


def test_more_slots_than_a_step_has_rows_are_closed_at_once():
    model = build("A", "float32")
    e = bb.Engine(model, 64 * 4300, max_slots=4300, max_seq_len=64, cache_dtype="int8")
    s = e.open(4200)
    for at, n in ((0, 3000), (3000, 1100)):
        e.step(s[at:at + n], [[1 + i % 7] for i in range(n)])
    e.step(s[10:4100], [[2]] * 4090)
    check_tables(e)
    e.close(s)
    check_tables(e)
    assert e.cache.live_slots == 0


@pytest.mark.parametrize("graphs", [True, False])
def test_steps_pass_the_debug_checks_and_tables_that_differ_do_not(graphs, monkeypatch):
    from brolm_b200.engine import debug
    monkeypatch.setattr(debug, "ENABLED", True)
    model = build("B", "float32")
    e = bb.Engine(model, 64 * 20, max_slots=3, cache_dtype="int8", max_piece=60, use_graphs=graphs)
    s = e.open(3)
    prompts = random_prompts(model.config.vocab_size, [60, 130, 7], seed=4)
    e.step(s, prompts)
    e.step(s[:2], [[1] * 30, [2] * 11])
    for t in range(70):
        e.step(s, [[3], [4], [5]])
    at = [g.ring for g in e.cache.kv_groups].index(None)            # (a ring's pages are all held by now)
    tables = e.cache.kv_groups[at].tables
    before = tables.free_count.clone()
    tables.free_count -= 1                     # (a page that nobody has any more)
    for tokens in ([[1], [2], [3]], [[1, 2], [3], [4]]):
        with pytest.raises(bb.StepError, match=f"debug: group {at}.*each once"):
            e.step(s, tokens)
    tables.free_count.zero_()
    with pytest.raises(bb.StepError, match=f"debug: group {at}: too few free blocks"):
        e.step(s, [[1] * 60, [2] * 50, [3]])
    tables.free_count.copy_(before)
    with pytest.raises(bb.StepError, match="refused a step"):       # (that step, told once more where the waits are looked at)
        e.step(s, [[1] * 3, [2], [3]])
    e.step(s, [[1], [2], [3]])
    e.close(s)
    check_tables(e)
