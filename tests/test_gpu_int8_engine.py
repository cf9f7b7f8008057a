"""Weights in 8 bits through the engine: every layer against the definitions in plain arithmetic, requests that do not see each other, drafts, the
command line."""
import functools
import math
import os
import subprocess
import sys

import pytest
import torch

import gpu_fixtures as gf
import plain_model as pm
import tiny_configs as tc

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def _rows(v):
    """The values that rows of 8-bit integers stand for (64-bit)."""
    v = v.double()
    m = v.abs().amax(1, keepdim=True)
    return torch.round(v * (127 / m.clamp(min=1e-300))) * (m / 127)


def _engine(case, dtype, **options):
    from geneinfer_b200.engine.loading import load_model
    from geneinfer_b200.engine.step import StepEngine
    model = load_model(gf.model_dir(case), dtype=dtype, weights="int8")
    return StepEngine(model, n_pages=64, max_requests=4, max_step_tokens=512, debug_checks=True, **options)


def _off(got, want):
    return float((got.double() - want).norm() / want.norm())


@functools.lru_cache(maxsize=None)
def _plain(case):
    w, cfg = pm.load_plain(gf.model_dir(case))
    return w, cfg


# How far a half of a layer may be from the definitions: the engine's values ahead of a rounding differ from the formula's by up to 2^-16 of themselves
# (32-bit sums and exponentials). A value falls to the other of two neighbours where it lies that near to their border: of 127 steps at most 2 * 127 * 2^-16
# = 0.4 % of the values, and through the 2^-9 steps of bfloat16 2^-7 = 0.8 %. Each is then a step, 1/127 of the row's largest value, off, and that is at
# most 6 times the row's root mean square here: sqrt(0.012) * 6 / 127 = 0.005 of a row. What 8 bits cost themselves is several times that.
NEAR = 0.005


@pytest.mark.parametrize("length", [1, 7, 33, 64])
@pytest.mark.parametrize("case", ["a", "b", "c", "d"])
def test_layers(case, length):
    """Everything but the projections in 32-bit: both halves of every layer from the stream that the engine itself had ahead of them."""
    w, cfg = _plain(case)
    engine = _engine(case, "float32")
    seen = {}
    engine.tap = lambda tag, layer, tensor, ctx: seen.__setitem__((tag, layer), tensor.detach().clone())
    from geneinfer_b200.engine.step import StepEntry
    tokens = tc.random_tokens(length, cfg["vocab"], 7)
    engine.open("r")
    engine.step([StepEntry("r", tokens, [length - 1])])
    torch.cuda.synchronize()
    H, Hkv, hd = cfg["heads"], cfg["kv_heads"], cfg["head_dim"]
    cos, sin = pm.plain_rope_table(range(length), hd, cfg["theta"], cfg["scaling"])
    cost = []
    x = seen["embedding", -1].cpu()
    for layer in range(cfg["layers"]):
        p = f"model.layers.{layer}."
        for exact in (True, False):
            rows = _rows if exact else (lambda v: v.double())
            weight = (lambda name: _rows(w[p + name]).T) if exact else (lambda name: w[p + name].double().T)      # a channel is a row
            xn = rows(pm.plain_rmsnorm(x.double(), w[p + "input_layernorm.weight"].double(), cfg["eps"]))
            q, k, v = ((xn @ weight(f"self_attn.{n}_proj.weight")).float().reshape(length, heads, hd) for n, heads in (("q", H), ("k", Hkv), ("v", Hkv)))
            att = pm.plain_attention(pm.plain_rope(q, cos, sin), pm.plain_rope(k, cos, sin), v, 1.0 / math.sqrt(hd))
            mixed = rows(att.reshape(length, H * hd)) @ weight("self_attn.o_proj.weight")
            after = seen["attn_out", layer].cpu()
            xn = rows(pm.plain_rmsnorm(after.double(), w[p + "post_attention_layernorm.weight"].double(), cfg["eps"]))
            h = pm.plain_swiglu(xn @ weight("mlp.gate_proj.weight"), xn @ weight("mlp.up_proj.weight"))
            fed = rows(h.to(torch.bfloat16) if exact else h) @ weight("mlp.down_proj.weight")
            last = seen["ffn_out", layer].cpu()
            off = _off(after.double() - x.double(), mixed), _off(last.double() - after.double(), fed)
            if exact:
                assert max(off) < NEAR, (layer, off)
            else:
                cost.append(off)
        x = last
    assert max(max(c) for c in cost) > NEAR, "the projections do not look like 8 bits"


@pytest.mark.parametrize("case", ["a", "b", "c", "d"])
def test_requests_do_not_see_each_other(case):
    """In 32-bit besides the projections a request's tokens are those it gets alone, whatever runs beside it: the sums are whole numbers."""
    from geneinfer_b200 import Engine
    vocab = gf.CASES[case][0]["vocab_size"]
    prompts = [tc.random_tokens(n, vocab, 40 + n) for n in (5, 90, 33, 1)]
    together = Engine(gf.model_dir(case), dtype="float32", weights="int8", max_running=4, step_tokens=48, prefill_chunk=32, debug_checks=True)
    alone = Engine(gf.model_dir(case), dtype="float32", weights="int8", max_running=1)
    got = together.generate(prompts, max_new_tokens=20, temperature=0.0)
    assert got == [alone.generate([p], max_new_tokens=20, temperature=0.0)[0] for p in prompts]
    assert all(len(g) == 20 for g in got)


@pytest.mark.parametrize("case", ["c", "d", "w", "w3"])
def test_generation_in_bfloat16(case):
    """The serving path: prompts in portions, decoded steps from graphs; twice the same, no wait gave up, and half the projections' bytes."""
    from geneinfer_b200 import Engine
    from geneinfer_b200.ops import kernels
    vocab = gf.CASES[case][0]["vocab_size"]
    prompts = [tc.random_tokens(n, vocab, 50 + n) for n in (130, 12, 60)]
    engine = Engine(gf.model_dir(case), weights="int8", max_running=3, max_seq_len=256, step_tokens=128, prefix_cache=False, decode_weight_copy=False)
    first = engine.generate(prompts, max_new_tokens=24, temperature=0.0)
    assert first == engine.generate(prompts, max_new_tokens=24, temperature=0.0)
    assert kernels.gemm_tc_status(engine.steps.device) == 0, "a bounded wait gave up"
    assert engine.steps.graph_replays > 0
    native = Engine(gf.model_dir(case), max_running=1, max_seq_len=64, decode_weight_copy=False)
    embedding = 2 * native.model.embedding.numel()
    outside = embedding if gf.CASES[case][0]["tie_word_embeddings"] else 2 * embedding
    if case == "w":      # (sizes that are whole tiles)
        assert engine.model.weight_bytes() - outside < 0.51 * (native.model.weight_bytes() - outside)


def test_drafts_of_a_served_model_in_8_bits():
    """Greedy generation with drafts gives what the served model alone gives (32-bit besides the projections)."""
    from geneinfer_b200 import Engine, SpeculativeEngine
    prompts = [tc.random_tokens(n, 256, 90 + n) for n in (4, 21)]
    drafted = SpeculativeEngine(gf.model_dir("a"), gf.model_dir("a"), drafts=3, dtype="float32", max_running=2, max_seq_len=96, weights="int8")
    alone = Engine(gf.model_dir("a"), dtype="float32", weights="int8", max_running=2, max_seq_len=96)
    assert drafted.generate(prompts, max_new_tokens=24, temperature=[0.0, 0.0]) == alone.generate(prompts, max_new_tokens=24, temperature=0.0)


def test_adapters_are_refused_beside_it():
    engine = _engine("a", "bfloat16")
    with pytest.raises(ValueError, match="takes none"):
        engine.enable_adapters(2, 4)


def test_command_line():
    from geneinfer_b200 import Engine
    prompt = tc.random_tokens(9, 500, 3)
    run = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "gi_generate"), "--model", gf.model_dir("c"), "--weights", "int8", "--temperature", "0",
                          "--steps", "20", "--no-echo", "--profile", "--prompt-ids", " ".join(map(str, prompt))], stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
    assert run.returncode == 0, run.stderr
    engine = Engine(gf.model_dir("c"), weights="int8", max_running=1, prefix_cache=False)
    want = engine.generate([prompt], max_new_tokens=20 - len(prompt) + 1, temperature=0.0)[0]
    assert [int(t) for t in run.stdout.split()] == want
    assert "8-bit integers" in run.stderr
    drafted = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "gi_generate"), "--model", gf.model_dir("c"), "--weights", "int8", "--draft-model",
                              gf.model_dir("c"), "--temperature", "0", "--steps", "20", "--no-echo", "--prompt-ids", " ".join(map(str, prompt))],
                             stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
    assert drafted.returncode == 0 and len(drafted.stdout.split()) == len(want), drafted.stderr


@pytest.mark.parametrize("flags", [["--weights", "int8", "--dtype", "fp32"], ["--dtype", "fp32", "--weights", "int8"]])
def test_command_line_in_32_bit_besides_the_projections(flags):
    from geneinfer_b200 import Engine
    prompt = tc.random_tokens(7, 256, 5)
    run = subprocess.run([sys.executable, os.path.join(ROOT, "bin", "gi_generate"), "--model", gf.model_dir("a"), *flags, "--temperature", "0", "--steps", "20", "--no-echo",
                          "--prompt-ids", " ".join(map(str, prompt))], stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True)
    assert run.returncode == 0, run.stderr
    engine = Engine(gf.model_dir("a"), dtype="float32", weights="int8", max_running=1, prefix_cache=False)
    assert [int(t) for t in run.stdout.split()] == engine.generate([prompt], max_new_tokens=20 - len(prompt) + 1, temperature=0.0)[0]
    assert engine.model.layers[0].int8 and engine.model.dtype is torch.float32


def _logits(engine, name, tokens, portion, wanted):
    """32-bit logits of the wanted positions of a prompt fed in portions; the request is closed again."""
    from geneinfer_b200.engine.step import StepEntry
    engine.open(name)
    rows = []
    for at in range(0, len(tokens), portion):
        here = tokens[at:at + portion]
        out = engine.step([StepEntry(name, here, [p - at for p in wanted if at <= p < at + len(here)])])
        if out is not None:
            rows.append(out.clone())
    engine.close(name)
    return torch.cat(rows)


@pytest.mark.parametrize("length", [700, 1300])
def test_long_prompts_in_one_step_and_in_portions(length):
    """A step of more rows than any projection takes as few (1,300 at these widths; at 700 some of each) gives what portions of 64 and of 7 tokens give, to the bit, the
    first time and from the recorded launches."""
    from geneinfer_b200.engine.loading import load_model
    from geneinfer_b200.engine.step import StepEngine
    from geneinfer_b200.ops import kernels
    model = load_model(gf.model_dir("w"), dtype="float32", weights="int8", max_position=2048)
    engine = StepEngine(model, n_pages=256, max_requests=2, max_step_tokens=1400, debug_checks=True)
    layer = model.layers[0]
    forms = {kernels._int8_plan(length, linear.weight)[0] for linear in (layer.mixer.w_qkv, layer.mixer.w_o, layer.feed_forward.w_gate_up, layer.feed_forward.w_down)}
    assert forms == ({"many"} if length == 1300 else {"few", "many"})
    tokens = tc.random_tokens(length, 128256, length)
    wanted = [0, 5, 63, 64, 300, length - 1]
    whole = _logits(engine, "whole", tokens, length, wanted)
    assert bool(whole.isfinite().all())
    before = engine.program_runs
    assert torch.equal(_logits(engine, "again", tokens, length, wanted), whole) and engine.program_runs > before
    assert torch.equal(_logits(engine, "portions", tokens, 64, wanted), whole)
    assert torch.equal(_logits(engine, "small", tokens[:301], 7, wanted[:5]), whole[:5])
    assert kernels.gemm_tc_status(engine.device) == 0


def test_long_prompts_of_the_serving_path():
    """bfloat16, steps of 1,400 tokens: products of many rows, the gated epilogue, the addition with the norm; twice the same, and near the 32-bit path."""
    from geneinfer_b200.engine.loading import load_model
    from geneinfer_b200.engine.step import StepEngine
    from geneinfer_b200.ops import kernels
    tokens, wanted = tc.random_tokens(1300, 128256, 3), [0, 300, 1299]
    rows = {}
    for dtype in ("bfloat16", "float32"):
        engine = StepEngine(load_model(gf.model_dir("w"), dtype=dtype, weights="int8", max_position=2048), n_pages=256, max_requests=2, max_step_tokens=1400, debug_checks=True)
        rows[dtype] = _logits(engine, "first", tokens, 1300, wanted)
        assert torch.equal(_logits(engine, "again", tokens, 1300, wanted), rows[dtype])
        assert kernels.gemm_tc_status(engine.device) == 0
    # The cache, the attention and the head's input round to bfloat16, 2^-9 of a value: half a step of 127 and more, so that the rows of a projection round apart. Two
    # roundings of one value that know nothing of each other differ by sqrt(1/6) of a step, a step is 1/127 of a row's largest value, that at most 6 times its root mean
    # square: 6 / 127 / sqrt(6) = 0.019 of a row. Eight projections (four in each of two layers), in squares: 0.055; the bfloat16 roundings themselves are a tenth of it.
    assert _off(rows["bfloat16"], rows["float32"].double()) < 0.0625
