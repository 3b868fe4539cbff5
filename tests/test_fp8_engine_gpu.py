"""Models whose matrices are in 8-bit floating point: against the same model with the products done by the oracle in 64 bits,
against the oracle's model, prompts against decoding, captured steps against steps that are not."""
import os
import subprocess
import sys

import pytest
import torch

import brolm_b200 as bb
from brolm_b200 import kernels
from tests import banevik_helpers, kedasun_helpers, neburax_helpers, papusun_helpers, relulix_helpers, ritirax_helpers
from tests.helpers import TINY, make_folder, oracle_inputs, random_prompts
from tests.plain import fp8_plain, gemma2_plain

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
ROOT = os.path.normpath(os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))
WIDE = dict(vocab_size=300, hidden_size=384, intermediate_size=640, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
            head_dim=128, rope_theta=10000.0, sliding_window=100, attn_logit_softcapping=50.0, final_logit_softcapping=30.0,
            query_pre_attn_scalar=128, rms_norm_eps=1e-6, max_position_embeddings=1024)


def build(name="B", dtype="float32", weight_dtype="fp8"):
    cfg, seed, std = (WIDE, 5, 0.05) if name == "wide" else TINY[name]
    return bb.Model(bb.Gemma2Config(**cfg), dtype=dtype, device=DEV, weight_dtype=weight_dtype).init_random(seed=seed, weight_std=std, norm_std=0.1)


def off(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def held(m):
    y = torch.empty(m.shape, dtype=torch.float32, device=DEV)
    kernels.fp8_read(m, y)
    return y.double()


def act_of(w, z, activation, limit):
    return fp8_plain.gated(z[..., 0::2], z[..., 1::2], activation, limit) if w.gated else fp8_plain.act(z, activation)


def plain_linear(x, w, out, activation="none", limit=0.0):
    out.copy_(act_of(w, fp8_plain.values(x.float()) @ held(w).T, activation, limit))


def plain_feedforward(x, gate_up, down, out, activation="gelu_tanh", limit=0.0):
    h = act_of(gate_up, fp8_plain.values(x.float()) @ held(gate_up).T, activation, limit)
    out.copy_(fp8_plain.values(h.float()) @ held(down).T)


def plain_pairs(x, ids, up, down, out, activation="silu", limit=0.0, scale=None):
    xe, ue, de = fp8_plain.values(x.float()), held(up), held(down)
    for t in range(ids.shape[0]):
        for c in range(ids.shape[1]):
            e = int(ids[t, c])
            if 0 <= e < up.shape[0]:
                z = (xe[t] @ ue[e].T) * (float(scale[t, c]) if scale is not None else 1.0)
                h = act_of(up, z, activation, limit)
                out[c, t] = (fp8_plain.values(h.float()[None])[0] @ de[e].T).float()


def by_the_oracle(monkeypatch):
    monkeypatch.setattr(kernels, "linear_fp8", plain_linear)
    monkeypatch.setattr(kernels, "feedforward_fp8", plain_feedforward)
    monkeypatch.setattr(kernels, "experts_fp8_pairs", plain_pairs)


# A float sum that lands on the other side of a border of 8 bits moves a number by 2^-3 of itself at most, about one number in
# ten thousand: a few products of a row of some hundred numbers change by 2^-3 / sqrt(some hundred), one in a hundred rows.
SAME = 5e-3


@pytest.mark.parametrize("name", ["A", "B", "C", "wide"])
def test_gemma_beside_the_products_in_64_bits(name, monkeypatch):
    model = build(name)
    prompts = random_prompts(model.config.vocab_size, [5, 40, 1, 17], seed=1)
    engine = bb.Engine(model, max_tokens=64 * 8, max_slots=4)
    got = engine.step(engine.open(4), prompts).clone()
    by_the_oracle(monkeypatch)
    other = bb.Engine(model, max_tokens=64 * 8, max_slots=4, use_graphs=False)
    assert off(got, other.step(other.open(4), prompts)) <= SAME


@pytest.mark.parametrize("helpers, cls, names", [
    (banevik_helpers, bb.BanevikConfig, ["P", "Q", "R"]), (neburax_helpers, bb.NeburaxConfig, ["S", "T"]), (ritirax_helpers, bb.RitiraxConfig, ["S", "T"]),
    (relulix_helpers, bb.RelulixConfig, ["S", "T"]), (kedasun_helpers, bb.KedasunConfig, ["S", "T"]), (papusun_helpers, bb.PapusunConfig, ["S", "T"])])
def test_other_designs_beside_the_products_in_64_bits(helpers, cls, names, monkeypatch):
    for name in names:
        cfg, seed, std = helpers.CONFIGS[name]
        model = bb.Model(cls.from_dict(cfg), dtype="float32", device=DEV, weight_dtype="fp8").init_random(seed=seed, weight_std=std)
        kept = [p for p, _ in model._tensor_names if any(isinstance(v, kernels.Fp8Matrix) for v in vars(p).values())]
        assert kept
        prompts = random_prompts(model.layout.embedding.vocab, [3, 21], seed=2)
        more = random_prompts(model.layout.embedding.vocab, [4, 4], seed=3)
        runs = []
        for plain in (False, True):
            with monkeypatch.context() as m:
                if plain:
                    by_the_oracle(m)
                engine = bb.Engine(model, max_tokens=64 * 4, max_slots=2, use_graphs=not plain)
                slots = engine.open(2)
                out = [engine.step(slots, prompts).clone()]
                out += [engine.step(slots, [[row[t]] for row in more]).clone() for t in range(4)]
                runs.append(torch.stack(out))
        assert off(runs[0], runs[1]) <= SAME, (cls.__name__, name)


@pytest.mark.parametrize("name,dtype", [("A", "float32"), ("B", "bfloat16"), ("C", "float32"), ("A", "bfloat16")])
def test_near_the_oracles_model_with_the_same_matrices(name, dtype, tmp_path):
    """The matrices are the rounded ones on both sides, so what is left is the rows' rounding, 2^-4 of a number at most and a
    fortieth of it on average, eight or twelve products one after the other: a tenth of the logits."""
    folder = make_folder(tmp_path, name)
    config, weights = oracle_inputs(folder)
    rounded = {k: fp8_plain.values(v) if v.dim() == 2 and "layers" in k else v for k, v in weights.items()}
    model = bb.load_model(folder, dtype=dtype, weight_dtype="fp8")
    engine = bb.Engine(model, max_tokens=256)
    ids = random_prompts(config["vocab_size"], [23], seed=4)[0]
    got = engine.step(engine.open(1), [ids])[0]
    want = gemma2_plain.forward(config, rounded, ids)[-1].to(DEV)
    assert off(got, want) <= 0.15
    assert float(torch.nn.functional.cosine_similarity(got.double(), want, dim=0)) > 0.99


@pytest.mark.parametrize("name,dtype,bound", [("wide", "float32", SAME), ("B", "float32", SAME), ("wide", "bfloat16", 4e-2)])
def test_decoding_gives_what_the_whole_prompt_gives(name, dtype, bound):
    """In float the same numbers are rounded; in bfloat16 the attention of prompts and of decoding round their results at other
    places, 2^-8 of them, which goes through the layers as such and moves numbers across borders."""
    model = build(name, dtype)
    vocab = model.config.vocab_size
    whole = random_prompts(vocab, [30, 150, 9], seed=7)
    engine = bb.Engine(model, max_tokens=64 * 12, max_slots=6)
    slots = engine.open(3)
    engine.step(slots, [p[:-6] for p in whole])
    for t in range(6, 0, -1):
        last = engine.step(slots, [[p[-t]] for p in whole]).clone()
    fresh = bb.Engine(model, max_tokens=64 * 12, max_slots=6)
    assert off(last, fresh.step(fresh.open(3), whole)) <= bound
    engine.close(slots)
    fresh.close([0, 1, 2])


@pytest.mark.parametrize("batch", [1, 5, 20, 40])
def test_captured_steps_give_the_same_bits(batch):
    model = build("wide", "bfloat16")
    prompts = random_prompts(model.config.vocab_size, [3 + i % 5 for i in range(batch)], seed=8)
    outs = []
    for graphs in (True, False):
        engine = bb.Engine(model, max_tokens=64 * batch, max_slots=batch, use_graphs=graphs)
        slots = engine.open(batch)
        engine.step(slots, prompts)
        outs.append([engine.step(slots, [[7 + t]] * batch).clone() for t in range(4)])
        engine.close(slots)
    for a, b in zip(*outs):
        assert torch.equal(a, b)


def test_two_engines_on_one_model_and_generation():
    model = build("wide", "bfloat16")
    prompts = random_prompts(model.config.vocab_size, [12, 3, 33], seed=9)
    opts = bb.GenerateOptions(max_new_tokens=12, sampling=bb.SamplingParams(temperature=0.0), stop_on_eos=False)
    a, b = bb.Engine(model, max_tokens=512), bb.Engine(model, max_tokens=1024, cache_dtype="int8")
    first = bb.generate(a, prompts, eos_id=-1, opts=opts)
    bb.generate(b, prompts, eos_id=-1, opts=opts)
    assert bb.generate(a, prompts, eos_id=-1, opts=opts) == first and all(len(o) == 12 for o in first)


def test_matrices_take_about_half_the_bytes():
    a, b = build("wide", "bfloat16", None), build("wide", "bfloat16", "fp8")
    full = lambda p: sum(t.numel() * 2 for t in (p.mixer.w_qkv, p.mixer.w_o, p.feedforward.w_gate_up, p.feedforward.w_down))
    part = lambda p: sum(t.nbytes for t in (p.mixer.w_qkv, p.mixer.w_o, p.feedforward.w_gate_up, p.feedforward.w_down))
    assert sum(map(part, b.blocks)) <= 0.51 * sum(map(full, a.blocks))
    assert b.head.dtype == torch.bfloat16 and b.embedding.dtype == torch.bfloat16


def test_from_the_command_line(tmp_path):
    folder = make_folder(tmp_path, "A", torch.bfloat16)
    r = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "run_model"), "--model", folder, "--weight-dtype", "fp8", "--ids", "5,17,3", "--max-new", "5",
                        "--no-eos"], capture_output=True, text=True, timeout=600)
    assert r.returncode == 0, r.stderr
    assert "generated 5 tokens" in r.stdout


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("name", ["B", "wide"])
def test_norms_that_leave_8_bits_beside_norms_and_roundings(name, dtype, monkeypatch):
    model = build(name, dtype)
    assert all(b.pre_mixer_norm.eight_bits and b.pre_ffn_norm.eight_bits and not b.post_ffn_norm.eight_bits for b in model.blocks) and not model.final_norm.eight_bits
    prompts = random_prompts(model.config.vocab_size, [5, 40, 1, 17], seed=2)

    def steps():
        engine = bb.Engine(model, max_tokens=64 * 8, max_slots=4, use_graphs=False)
        slots = engine.open(4)
        out = [engine.step(slots, prompts).clone()]
        for t in range(3):
            out.append(engine.step(slots, [[7 + t]] * 4).clone())
        return out
    got = steps()
    calls = []

    def apart(h, y, post_weight, post_eps, post_offset, next_weight, next_eps, next_offset):
        calls.append(len(h))
        out = torch.empty_like(h)
        residual_rmsnorm(h, y, post_weight, post_eps, post_offset, next_weight, next_eps, next_offset, out)
        return kernels.fp8_quantize(out)
    residual_rmsnorm = kernels.residual_rmsnorm
    monkeypatch.setattr(kernels, "residual_rmsnorm_fp8", apart)
    want = steps()
    assert len(calls) == 4 * (2 * len(model.blocks) - 1)
    for a, b in zip(got, want):
        assert off(a, b) < SAME


def test_matrices_and_the_cache_in_8_bits_together():
    """Whole prompts and the same in pieces on top of a cache in 8 bits, with rows in 8 bits from norm to product.  A piece reads keys
    and values off by a 254th of a page's largest, some 1 % of their size; a row that is 1 % off has one number in nine on the other
    side of a border of 8 bits, a step of 9 %: 3 % of a product, and six products follow one another: 7 %, doubled."""
    model = build("wide", "bfloat16")
    prompts = random_prompts(model.config.vocab_size, [70, 9], seed=4)
    whole = bb.Engine(model, max_tokens=64 * 8, max_slots=2, cache_dtype="int8")
    slots = whole.open(2)
    a = [whole.step(slots, prompts).clone()] + [whole.step(slots, [[t], [t + 1]]).clone() for t in (3, 8)]
    pieces = bb.Engine(model, max_tokens=64 * 8, max_slots=2, cache_dtype="int8", max_piece=128)
    slots = pieces.open(2)
    pieces.step(slots, [p[:4] for p in prompts])
    b = [pieces.step(slots, [p[4:] for p in prompts]).clone()] + [pieces.step(slots, [[t], [t + 1]]).clone() for t in (3, 8)]
    for x, y in zip(a, b):
        assert x.isfinite().all() and y.isfinite().all() and off(x, y) < 0.15
