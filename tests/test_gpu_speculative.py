"""Adapters and drafted tokens through the engine: a request's adapter does what its matrices added to the weights would do, and generation with
drafts gives what the target model alone gives."""
import json
import os

import numpy as np
import pytest
import torch

import gpu_fixtures as gf
import tiny_configs as tc

pytestmark = pytest.mark.gpu

PUBLISHED = {"self_attn.q_proj": "self_attn.q_proj.weight", "self_attn.k_proj": "self_attn.k_proj.weight", "self_attn.v_proj": "self_attn.v_proj.weight",
             "self_attn.o_proj": "self_attn.o_proj.weight", "mlp.gate_proj": "mlp.gate_proj.weight", "mlp.up_proj": "mlp.up_proj.weight",
             "mlp.down_proj": "mlp.down_proj.weight"}


def adapter_and_merged(case, seed, tmp_path, rank=6, only=None, std=0.1):
    """(adapter folder, model folder in 32-bit with the adapter added to its weights)."""
    from geneinfer_b200.weights import SafetensorsFile, read_config, write_safetensors
    from geneinfer_b200.weights.adapters import read_adapter, write_random_adapter, PLACES
    source = gf.model_dir(case)
    _, config, _ = read_config(source)
    folder = str(tmp_path / f"adapter_{case}_{seed}")
    write_random_adapter(config, seed, folder, rank=rank, alpha=9.0, std=std)
    if only is not None:
        path = os.path.join(folder, "adapter_model.safetensors")
        with SafetensorsFile(path) as f:
            kept = [(n, f.tensor(n).clone()) for n in f.names() if any(o in n for o in only)]
        write_safetensors(path, kept)
    pairs, scale = read_adapter(folder)
    merged = str(tmp_path / f"merged_{case}_{seed}")
    os.makedirs(merged)
    with open(os.path.join(source, "config.json")) as f, open(os.path.join(merged, "config.json"), "w") as g:
        g.write(f.read())
    by_name = {}
    for (layer, name), parts in pairs.items():
        for published, (projection, place, _) in PLACES.items():
            if projection == name and parts[place] is not None:
                by_name[f"model.layers.{layer}.{PUBLISHED[published]}"] = parts[place]
    with SafetensorsFile(os.path.join(source, "model.safetensors")) as f:
        tensors = []
        for n in f.names():
            w = f.tensor(n).float()
            if n in by_name:
                down, up = by_name[n]
                w = w + scale * (up.double() @ down.double()).float()
            tensors.append((n, w))
    assert by_name and all(any(n == m for m, _ in tensors) for n in by_name)
    write_safetensors(os.path.join(merged, "model.safetensors"), tensors)
    return folder, merged


def engine_of(folder, dtype, slots=0, **options):
    from geneinfer_b200.engine.loading import load_model
    from geneinfer_b200.engine.step import StepEngine
    steps = StepEngine(load_model(folder, dtype=dtype), n_pages=96, max_requests=4, max_step_tokens=512, debug_checks=True, **options)
    if slots:
        steps.enable_adapters(slots, 8)
    return steps


@pytest.mark.parametrize("case", ["a", "b", "c"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_an_adapter_does_what_added_to_the_weights_it_would_do(case, dtype, tmp_path):
    """Two requests with adapters and one without in the same steps: a prompt, a portion beside single tokens, then single tokens (captured and replayed).
    32-bit: both sides differ in the order of sums. bfloat16: the merged side keeps its weights unrounded in 32 bits, so the distance is the
    model's own rounding noise, of which the fixture's comparisons allow three quarters beside the plain form; here both the weights and the
    adapters' sums round, twice the noise."""
    from geneinfer_b200.engine.step import StepEntry
    from geneinfer_b200.weights.adapters import read_adapter
    folders = [adapter_and_merged(case, s, tmp_path, std=0.1 if dtype == "float32" else 0.03) for s in (1, 2)]
    steps = engine_of(gf.model_dir(case), dtype, slots=3)
    for slot, (folder, _) in zip((2, 0), folders):
        steps.put_adapter(slot, *read_adapter(folder))
    plain = [engine_of(m, "float32") for m in (folders[0][1], folders[1][1], gf.model_dir(case))]
    vocab = steps.model.vocab_size
    texts = [tc.random_tokens(n, vocab, 9 + n) for n in (40, 21, 33)]
    slots = (2, 0, -1)
    for r in range(3):
        steps.open(r)
        plain[r].open(r)
    bound = 2e-4 if dtype == "float32" else 2 * max(gf.bf16_noise(case), 1e-2)
    at = [0, 0, 0]
    for counts in ((40 - 6, 21 - 6, 33 - 6), (2, 1, 1), (1, 1, 1), (1, 1, 1), (1, 1, 1), (0, 2, 0)):
        entries = [StepEntry(r, texts[r][at[r]:at[r] + n], [n - 1], adapter=slots[r]) for r, n in enumerate(counts) if n]
        got = steps.step(entries).float().cpu().numpy().copy()
        for row, e in zip(got, entries):
            want = plain[e.key].step([StepEntry(e.key, e.tokens, e.want)]).cpu().numpy()[0]
            assert np.abs(row - want).max() <= bound * max(1.0, np.abs(want).max()), (counts, e.key)
        at = [a + n for a, n in zip(at, counts)]
    assert steps.graph_replays > 0


def test_adapters_of_some_projections_only_and_steps_without_any(tmp_path):
    from geneinfer_b200.engine.step import StepEntry
    from geneinfer_b200.weights.adapters import read_adapter
    folder, merged = adapter_and_merged("a", 3, tmp_path, only=("layers.0.self_attn.v_proj", "layers.1.mlp.up_proj"))
    steps, plain, base = engine_of(gf.model_dir("a"), "float32", slots=1), engine_of(merged, "float32"), engine_of(gf.model_dir("a"), "float32")
    steps.put_adapter(0, *read_adapter(folder))
    text = tc.random_tokens(30, 256, 5)
    for engine in (steps, plain, base):
        for r in range(2):
            engine.open(r)
    a = steps.step([StepEntry(0, text, [29], adapter=0), StepEntry(1, text, [29])]).cpu().numpy().copy()
    b = plain.step([StepEntry(0, text, [29])]).cpu().numpy()[0].copy()
    c = base.step([StepEntry(0, text, [29]), StepEntry(1, text, [29])]).cpu().numpy()[0].copy()
    assert np.abs(a[0] - b).max() <= 2e-4 * np.abs(b).max() and np.abs(a[1] - c).max() <= 2e-5 * np.abs(c).max() and np.abs(a[0] - c).max() > 1e-2
    # a step in which no request has one runs as an engine without adapters runs it, to the bit
    d = steps.step([StepEntry(1, text[:3], [2])]).cpu().numpy().copy()
    e = base.step([StepEntry(1, text[:3], [2])]).cpu().numpy().copy()
    assert np.array_equal(d, e)
    steps.adapter_sets[0]["w_qkv"].clear(0)
    steps.adapter_sets[1]["w_gate_up"].clear(0)
    steps.truncate(0, 0)
    f = steps.step([StepEntry(0, text, [29], adapter=0)]).cpu().numpy()[0]
    assert np.abs(f - c).max() <= 2e-5 * np.abs(c).max()


def test_adapters_through_generate_and_their_refusals(tmp_path):
    from geneinfer_b200 import Engine
    from geneinfer_b200.engine.step import StepEntry
    folder, merged = adapter_and_merged("a", 4, tmp_path)
    engine = Engine(gf.model_dir("a"), dtype="float32", max_running=3, adapter_slots=2, adapter_rank=6)
    engine.load_adapter(1, folder)
    alone, base = Engine(merged, dtype="float32", max_running=3), Engine(gf.model_dir("a"), dtype="float32", max_running=3)
    shared = tc.random_tokens(40, 256, 7)                     # a prefix of whole pages that must not be shared between adapters
    prompts = [shared + [1], shared + [2], shared + [3]]
    got = engine.generate(prompts, max_new_tokens=10, adapters=[1, -1, 1])
    again = engine.generate(prompts, max_new_tokens=10, adapters=[-1, 1, -1])
    want, plain = alone.generate(prompts, max_new_tokens=10), base.generate(prompts, max_new_tokens=10)
    assert got[0] == want[0] and got[1] == plain[1] and got[2] == want[2]
    assert again[0] == plain[0] and again[1] == want[1] and again[2] == plain[2]
    assert want != plain
    with pytest.raises(ValueError):
        engine.submit([1, 2], adapter=2)
    with pytest.raises(ValueError):
        base.submit([1, 2], adapter=0)
    engine.steps.open("x")
    with pytest.raises(ValueError):
        engine.steps.step([StepEntry("x", [1], [], adapter=2)])
    with pytest.raises(RuntimeError):
        engine.steps.enable_adapters(1, 4)
    sets = engine.steps.adapter_sets[0]["w_qkv"]
    for bad in ([None], [(torch.zeros(7, 64), torch.zeros(64, 7)), None, None], [(torch.zeros(4, 63), torch.zeros(64, 4)), None, None],
                [(torch.zeros(4, 64), torch.zeros(64, 5)), None, None]):
        if bad[0] is not None and bad[0][0].shape[0] == 7:
            bad = [(torch.zeros(sets.rank + 1, 64), torch.zeros(64, sets.rank + 1)), None, None]
        with pytest.raises(ValueError):
            sets.put(0, bad, 1.0)
    with pytest.raises(ValueError):
        sets.put(2, [None, None, None], 1.0)
    with pytest.raises(ValueError):
        engine.steps.put_adapter(0, {(0, "w_other"): [None]}, 1.0)
    with open(os.path.join(folder, "adapter_config.json"), "w") as f:
        json.dump({"r": 6, "use_dora": True}, f)
    with pytest.raises(ValueError):
        engine.load_adapter(0, folder)


# ---- drafted tokens
def speculative(case, draft, dtype, **options):
    from geneinfer_b200 import SpeculativeEngine
    options = {"drafts": 4, "max_running": 3, "max_seq_len": 100, "step_tokens": 48, **options}
    return SpeculativeEngine(gf.model_dir(case), gf.model_dir(draft) if draft in gf.CASES else draft, dtype=dtype, **options)


@pytest.mark.parametrize("draft", ["a", "a_named"])
@pytest.mark.parametrize("drafts", [1, 4])
def test_greedy_generation_with_drafts_is_the_targets(draft, drafts):
    """32 bits, where the target's logits do not depend on how positions are cut into steps: token for token what the engine gives alone. The target as its
    own drafter proposes nothing that is refused."""
    from geneinfer_b200 import Engine
    prompts = [tc.random_tokens(n, 256, 40 + n) for n in (7, 1, 33, 60, 2)]
    want = Engine(gf.model_dir("a"), dtype="float32", max_running=3).generate(prompts, max_new_tokens=21)
    engine = speculative("a", draft, "float32", drafts=drafts)
    assert engine.generate(prompts, max_new_tokens=21) == want
    if draft == "a":
        assert engine.kept == engine.proposed > 0
    # again, with a stop token that comes up
    stop = want[0][5]
    cut = [w[:w.index(stop) + 1] if stop in w else w for w in want]
    assert engine.generate(prompts, max_new_tokens=21, stop_ids=[stop]) == cut
    for side in (engine.target, engine.draft):                # pages: none lost, none twice
        held = side.tables[side.tables >= 0].tolist()
        assert sorted(held + side.free[:int(side.n_free)].tolist()) == list(range(side.free.numel()))


def test_sampled_generation_with_the_target_as_drafter_keeps_every_draft():
    """p = q to the bit: u q(x) < p(x) for every u below 1."""
    engine = speculative("a", "a", "float32")
    out = engine.generate([tc.random_tokens(9, 256, 3), tc.random_tokens(20, 256, 4)], max_new_tokens=20, temperature=[0.9, 1.3], seed=5)
    assert engine.kept == engine.proposed and all(len(o) == 20 for o in out)
    assert engine.generate([tc.random_tokens(9, 256, 3), tc.random_tokens(20, 256, 4)], max_new_tokens=20, temperature=[0.9, 1.3], seed=5) == out
    assert engine.generate([tc.random_tokens(9, 256, 3), tc.random_tokens(20, 256, 4)], max_new_tokens=20, temperature=[0.9, 1.3], seed=6) != out


def test_sampled_generation_with_drafts_is_distributed_as_the_target():
    """600 requests of one prompt, the first two tokens: counts of the eight likeliest first tokens and of the likeliest second ones against the target's
    probabilities, within five standard deviations."""
    from geneinfer_b200.engine.loading import load_model
    from geneinfer_b200.engine.step import StepEngine, StepEntry
    prompt, n, T = tc.random_tokens(12, 256, 8), 600, 0.7
    engine = speculative("a", "a_named", "float32", max_running=100, max_seq_len=40, drafts=3)
    out = engine.generate([prompt] * n, max_new_tokens=2, temperature=T, seed=1000)
    steps = StepEngine(load_model(gf.model_dir("a"), dtype="float32"), n_pages=32, max_requests=1)
    steps.open(0)
    p = torch.softmax(steps.step([StepEntry(0, prompt, [11])])[0].double().cpu() / T, 0)
    counts = torch.bincount(torch.tensor([o[0] for o in out]), minlength=256).double()
    top = p.argsort(descending=True)[:8]
    assert bool(((counts[top] - n * p[top]).abs() <= 5 * (n * p[top] * (1 - p[top])).sqrt()).all())
    first = int(counts.argmax())
    second = [o[1] for o in out if o[0] == first]
    p2 = torch.softmax(steps.step([StepEntry(0, [first], [0])])[0].double().cpu() / T, 0)
    best = int(p2.argmax())
    m, share = len(second), float(p2[best])
    assert abs(sum(t == best for t in second) - m * share) <= 5 * (m * share * (1 - share)) ** 0.5 + 1
    assert 0 < engine.kept < engine.proposed


def test_drafts_and_adapters_together(tmp_path):
    """Every operator at once: requests with and without an adapter, drafts of the plain model, block tables on the device."""
    from geneinfer_b200 import Engine
    folder, merged = adapter_and_merged("a", 6, tmp_path)
    prompts = [tc.random_tokens(n, 256, 70 + n) for n in (5, 31, 18)]
    engine = speculative("a", "a", "float32", adapter_slots=1, adapter_rank=8)
    engine.load_adapter(0, folder)
    got = engine.generate(prompts, max_new_tokens=16, adapters=[0, -1, 0])
    want = Engine(merged, dtype="float32").generate(prompts, max_new_tokens=16)
    base = Engine(gf.model_dir("a"), dtype="float32").generate(prompts, max_new_tokens=16)
    assert got == [want[0], base[1], want[2]]
    assert 0 < engine.kept < engine.proposed


@pytest.mark.parametrize("case", ["c", "d"])
def test_drafts_in_bfloat16(case):
    """The tensor-core kernels with rows of several tokens a request: against the engine alone up to the first near-tie."""
    from geneinfer_b200 import Engine
    vocab = gf.CASES[case][0]["vocab_size"]
    prompts = [tc.random_tokens(n, vocab, 90 + n) for n in (17, 40)]
    want = Engine(gf.model_dir(case), dtype="bfloat16", max_running=2).generate(prompts, max_new_tokens=24)
    engine = speculative(case, case, "bfloat16", max_running=2)
    got = engine.generate(prompts, max_new_tokens=24)
    same = [next((i for i, (a, b) in enumerate(zip(g, w)) if a != b), len(w)) for g, w in zip(got, want)]
    assert all(len(g) == 24 for g in got) and sum(same) >= 24 and engine.kept > engine.proposed / 2


def test_speculative_refuses_what_does_not_fit():
    from geneinfer_b200 import SpeculativeEngine
    with pytest.raises(ValueError):
        SpeculativeEngine(gf.model_dir("a"), gf.model_dir("b"), dtype="float32")          # other vocabularies
    with pytest.raises(ValueError):
        speculative("a", "a", "float32", drafts=0)
    engine = speculative("a", "a", "float32")
    for arguments in (dict(prompts=[[]]), dict(prompts=[[256]]), dict(prompts=[[1] * 90], max_new_tokens=30), dict(prompts=[[1]], temperature=-1.0),
                      dict(prompts=[[1], [2]], temperature=[0.5]), dict(prompts=[[1]], adapters=[0])):
        with pytest.raises(ValueError):
            engine.generate(**arguments)
    assert engine.generate([[1, 2]], max_new_tokens=0) == [[]]


def test_the_command_line_with_an_adapter_and_a_draft_model(tmp_path, capsys):
    from geneinfer_b200.cli.generate_main import main
    folder, merged = adapter_and_merged("a", 9, tmp_path)
    prompt = " ".join(map(str, tc.random_tokens(11, 256, 12)))
    common = ["--prompt-ids", prompt, "--steps", "30", "--temperature", "0", "--dtype", "fp32", "--quiet"]

    def run(*more):
        assert main([*common, *more]) == 0
        return capsys.readouterr().out.split()

    want = run("--model", merged)
    assert run("--model", gf.model_dir("a"), "--adapter", folder) == want
    assert run("--model", gf.model_dir("a"), "--adapter", folder, "--draft-model", gf.model_dir("a_named"), "--drafts", "3") == want
    assert main([*common, "--model", merged, "--draft-model", merged, "--top-p", "0.9"]) == 2
    assert main([*common, "--model", merged, "--draft-model", merged, "--drafts", "0"]) == 2


def test_experts_named_by_token_ids_see_the_steps_own_tokens(tmp_path):
    """Recorded launches name the place of a step's tokens: portions of prompts of one size, one after another, and the steps of a drafter. One rank for all layers, so
    that a single group of pages serves the design."""
    import pinorax_configs as pc
    from geneinfer_b200 import Engine, SpeculativeEngine
    layers = [pc.layer(3, 24, 40, 48, 0.2, pc.moe(40, 0.8, 7, 2, shared=(56, 1.7))), pc.layer(5, 8, 16, 48, 0.3, pc.moe(72, 2.5, 5, 1)),
              pc.layer(2, 16, 24, 48, 0.25, pc.dense(64))]
    folders = [pc.make_model_dir(pc.model(96, 190, 256, 1e-5, 0.45, 9.0, layers), seed, str(tmp_path / f"model{seed}"), std=0.2) for seed in (3, 4)]
    prompts = [tc.random_tokens(n, 190, 30 + n) for n in (75, 20, 1, 130)]
    want = Engine(folders[0], dtype="float32", max_running=2).generate(prompts, max_new_tokens=20)
    for draft in folders:
        engine = SpeculativeEngine(folders[0], draft, dtype="float32", max_running=2, max_seq_len=200, step_tokens=16)
        for _ in range(2):
            assert engine.generate(prompts, max_new_tokens=20) == want
        if draft == folders[0]:
            assert engine.kept >= 0.9 * engine.proposed > 0


def test_a_refused_call_of_the_step_tables_ends_the_generation(monkeypatch):
    """One call in the middle of a round, or in a prompt, says that it was refused (its tables are made all the same, so that the model runs on sound ones); the
    calls behind it are met. The next generation starts from nothing."""
    from geneinfer_b200.ops import kernels
    engine = speculative("a", "a_named", "float32", max_running=2, step_tokens=10)
    prompts = [tc.random_tokens(n, 256, n) for n in (25, 3)]
    want = engine.generate(prompts, max_new_tokens=12)
    for name in ("step_tables", "trim_tables"):
        real = getattr(kernels, name)
        for at in (0, 1, 5, 8):
            calls = []

            def some(*args, real=real, at=at, calls=calls):
                real(*args)
                calls.append(None)
                if len(calls) == at + 1:
                    args[-1].fill_(-2)

            monkeypatch.setattr(kernels, name, some)
            with pytest.raises(RuntimeError, match="-2"):
                engine.generate(prompts, max_new_tokens=12)
            monkeypatch.setattr(kernels, name, real)
            assert len(calls) > at + 1
            assert engine.generate(prompts, max_new_tokens=12) == want


def test_a_step_that_the_pool_may_not_hold_is_not_run():
    """Sides whose pool (or whose tables) are smaller than their requests can grow: the step is refused on the host, ahead of any kernel that would run on the tables of another."""
    for side in ("target", "draft"):
        for name in ("free", "tables"):
            engine = speculative("a", "a_named", "float32", max_running=2)
            some = getattr(engine, side)
            if name == "free":
                some.free, some.n_free = some.free[:2].contiguous(), some.n_free.fill_(2)
            else:
                some.tables = some.tables[:, :1].contiguous()
            with pytest.raises(RuntimeError, match="pages"):
                engine.generate([tc.random_tokens(25, 256, 1), [3]], max_new_tokens=12)


def test_a_round_is_launched_without_a_wait_for_what_runs():
    """Half a second of earlier work on the stream: the rounds of three requests return while it still runs."""
    engine = speculative("a", "a_named", "float32", max_running=3)
    prompts = [tc.random_tokens(n, 256, n) for n in (25, 3, 9)]
    want = engine.generate(prompts, max_new_tokens=12)
    real, waited = engine._round, []

    def behind_work(*args):
        if len(waited) == 1:                   # (the second round: the first is still to be collected)
            torch.cuda._sleep(1_000_000_000)
        earlier = torch.cuda.Event()
        earlier.record()
        out = real(*args)
        waited.append(earlier.query())
        return out

    engine._round = behind_work
    assert engine.generate(prompts, max_new_tokens=12) == want
    assert len(waited) > 2 and not waited[1]


@pytest.mark.parametrize("drafts", [1, 4])
@pytest.mark.parametrize("draft", ["a", "a_named"])
def test_generation_up_to_the_end_of_the_context(draft, drafts):
    """128 positions, of which the last token's is the last one fed: rounds near the end propose fewer tokens, down to none. Requests end at different places, one
    long before the others, one at the context's last position with its prompt."""
    from geneinfer_b200 import Engine
    for lengths, new in (((10, 60, 119, 2), 10), ((128, 20), 1), ((126, 125, 30), 3), ((9,), 120)):
        prompts = [tc.random_tokens(n, 256, 60 + n) for n in lengths]
        want = Engine(gf.model_dir("a"), dtype="float32", max_running=4).generate(prompts, max_new_tokens=new)
        engine = speculative("a", draft, "float32", drafts=drafts, max_seq_len=128)
        assert engine.generate(prompts, max_new_tokens=new) == want
        for side in (engine.target, engine.draft):
            held = side.tables[side.tables >= 0].tolist()
            assert sorted(held + side.free[:int(side.n_free)].tolist()) == list(range(side.free.numel()))
    sampled = engine.generate([prompts[0]] * 3, max_new_tokens=120, temperature=0.8, seed=3)
    assert [len(s) for s in sampled] == [120] * 3 and sampled[0] != sampled[1]
    with pytest.raises(ValueError):
        engine.generate([tc.random_tokens(10, 256, 1)], max_new_tokens=120)


def test_the_command_line_with_a_draft_model_fills_the_context(capsys):
    from geneinfer_b200.cli.generate_main import main
    common = ["--model", gf.model_dir("a"), "--prompt-ids", " ".join(map(str, tc.random_tokens(11, 256, 12))), "--temperature", "0", "--dtype", "fp32", "--quiet"]
    for more in ([], ["--steps", "400"], ["--max-seq-len", "70"], ["--steps", "60"]):
        assert main([*common, *more]) == 0
        want = capsys.readouterr().out.split()
        assert main([*common, *more, "--draft-model", gf.model_dir("a_named")]) == 0
        assert capsys.readouterr().out.split() == want


def test_the_command_line_with_drafts_and_a_design_of_its_own(tmp_path, capsys):
    """Pinorax names its context ``max_positions``; what does not go with a draft model is refused by name."""
    import pinorax_configs as pc
    from geneinfer_b200.cli.generate_main import main
    config = pc.model(96, 190, 64, 1e-5, 0.45, 9.0, [pc.layer(3, 24, 40, 48, 0.2, pc.dense(136)), pc.layer(5, 8, 16, 48, 0.3, pc.dense(64))])
    folder = pc.make_model_dir(config, 5, str(tmp_path / "model"), std=0.2)
    common = ["--model", folder, "--prompt-ids", "5 9 2 100", "--temperature", "0", "--dtype", "fp32", "--quiet"]
    for more in ([], ["--max-seq-len", "40"], ["--steps", "20"]):
        assert main([*common, *more]) == 0
        want = capsys.readouterr().out.split()
        assert main([*common, *more, "--draft-model", folder]) == 0, capsys.readouterr().err
        assert capsys.readouterr().out.split() == want
    for flags in (["--profile"], ["--kv-pages", "64"]):
        assert main([*common, "--draft-model", folder, *flags]) == 2
        assert flags[0] in capsys.readouterr().err


def test_an_adapter_that_does_not_fit_leaves_the_slots_as_they_were(tmp_path):
    from geneinfer_b200.weights.adapters import read_adapter
    folder, _ = adapter_and_merged("a", 14, tmp_path)
    steps = engine_of(gf.model_dir("a"), "float32", slots=2)
    pairs, scale = read_adapter(folder)
    steps.put_adapter(1, pairs, scale)
    sets = [s for layer in steps.adapter_sets.values() for s in layer.values()]
    before = [[t.clone() for t in (s.down, s.up, s.scales)] for s in sets]

    def unchanged():
        return all(torch.equal(a, b) for s, old in zip(sets, before) for a, b in zip((s.down, s.up, s.scales), old))

    last = max(pairs)
    for bad in (lambda d, u: (d[:, :-1], u), lambda d, u: (d, u[:-1]), lambda d, u: (d.repeat(3, 1), u.repeat(1, 3)), lambda d, u: (d[0], u)):
        other = {k: [None if p is None else (p[0] + 1, p[1] + 1) for p in v] for k, v in pairs.items()}
        other[last] = [bad(*p) if p is not None else None for p in other[last]]
        with pytest.raises(ValueError):
            steps.put_adapter(1, other, 2 * scale)
        assert unchanged()
    for slot in (-1, 2):
        with pytest.raises(ValueError):
            steps.put_adapter(slot, pairs, 2 * scale)
        assert unchanged()
    with pytest.raises(ValueError):
        steps.put_adapter(1, {**pairs, last: pairs[last] + [None]}, 2 * scale)
    assert unchanged()


def test_ranks_and_slots_beyond_the_kernels_are_refused_before_anything_is_made():
    """[q; k; v] stacks three ranks: 168 each at most (512 in all, in steps of four). What the largest gives is what the plain model gives: its adapters are none."""
    from geneinfer_b200.engine.step import StepEntry
    for slots, rank in ((1, 169), (1, 172), (1, 512), (8193, 4), (0, 4), (1, 0)):
        steps = engine_of(gf.model_dir("a"), "float32")
        with pytest.raises(ValueError):
            steps.enable_adapters(slots, rank)
        assert steps.adapter_step is None and not steps.adapter_sets
        assert all(l.adapters is None for layer in steps.model.layers for _, l, _ in layer.mixer.adaptable() + layer.feed_forward.adaptable())
    text = tc.random_tokens(30, 256, 5)
    rows = []
    for dtype in ("float32", "bfloat16"):
        for adapter in (-1, 0):
            steps = engine_of(gf.model_dir("a"), dtype)
            steps.enable_adapters(1, 168)
            steps.open(0)
            rows.append(steps.step([StepEntry(0, text, [29], adapter=adapter)]).cpu().numpy().copy())
        bound = 2e-5 if dtype == "float32" else 2 * max(gf.bf16_noise("a"), 1e-2)
        assert np.abs(rows[-1] - rows[-2]).max() <= bound * np.abs(rows[-1]).max()


def test_generate_looks_at_every_adapter_before_it_takes_a_request(tmp_path):
    from geneinfer_b200 import Engine
    folder, _ = adapter_and_merged("a", 15, tmp_path)
    engine = Engine(gf.model_dir("a"), dtype="float32", max_running=2, adapter_slots=1, adapter_rank=6)
    engine.load_adapter(0, folder)
    prompts = [tc.random_tokens(n, 256, n) for n in (5, 9)]
    for adapters in ([0], [0, 1], [0, 0, 0], []):
        with pytest.raises(ValueError):
            engine.generate(prompts, max_new_tokens=4, adapters=adapters)
        assert engine.scheduler.idle()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_steps_of_more_than_a_thousand_rows_with_adapters(dtype, tmp_path):
    """1,500 rows of four requests in one step, whose rows the device puts in their adapters' order first; the launches are recorded by the first such step and repeated by
    the others, with other tokens and other adapters. Against models with the adapters in their weights, one request at a time; bounds as in the test of small steps."""
    from geneinfer_b200.engine.loading import load_model
    from geneinfer_b200.engine.step import StepEngine, StepEntry
    from geneinfer_b200.weights.adapters import read_adapter
    folders = [adapter_and_merged("c", s, tmp_path, std=0.1 if dtype == "float32" else 0.03) for s in (21, 22)]
    steps = StepEngine(load_model(gf.model_dir("c"), dtype=dtype), n_pages=160, max_requests=4, max_step_tokens=2048, debug_checks=True)
    steps.enable_adapters(3, 8)
    for slot, (folder, _) in zip((2, 0), folders):
        steps.put_adapter(slot, *read_adapter(folder))
    plain = {slot: engine_of(m, "float32") for slot, m in ((2, folders[0][1]), (0, folders[1][1]), (-1, gf.model_dir("c")))}
    bound = 2e-4 if dtype == "float32" else 2 * max(gf.bf16_noise("c"), 1e-2)
    for turn, slots in enumerate(((2, 0, -1, 2), (-1, 0, 2, 0), (0, 0, 0, 0))):
        entries = []
        for r, n in enumerate((400, 300, 420, 380)):
            steps.open((turn, r))
            entries.append(StepEntry((turn, r), tc.random_tokens(n, 500, 10 * turn + r), [0, n // 2, n - 1], adapter=slots[r]))
        got = steps.step(entries).float().cpu().numpy().copy().reshape(4, 3, -1)
        for r, e in enumerate(entries):
            engine = plain[slots[r]]
            engine.open(e.key)
            want = engine.step([StepEntry(e.key, e.tokens, e.want)]).cpu().numpy()
            engine.close(e.key)
            assert np.abs(got[r] - want).max() <= bound * max(1.0, np.abs(want).max()), (turn, r)
            steps.close(e.key)
    assert steps.program_runs > 0


@pytest.mark.parametrize("case", ["c", "d"])
def test_drafts_in_bfloat16_follow_the_targets_own_choices(case):
    """Every token of a greedy generation against the logits that the target itself has behind the tokens before it, in one step: it is the largest there, or nearer to it
    than the noise that two cuts of the same positions show (the fixture's bound on bfloat16)."""
    from geneinfer_b200.engine.loading import load_model
    from geneinfer_b200.engine.step import StepEngine, StepEntry
    vocab = gf.CASES[case][0]["vocab_size"]
    prompts = [tc.random_tokens(n, vocab, 190 + n) for n in (17, 40, 3)]
    engine = speculative(case, case, "bfloat16", max_running=3)
    got = engine.generate(prompts, max_new_tokens=40)
    steps = StepEngine(load_model(gf.model_dir(case), dtype="bfloat16"), n_pages=96, max_requests=1, max_step_tokens=512)
    bound = float(gf.tolerance("bfloat16", case))
    ties = 0
    for r, (p, out) in enumerate(zip(prompts, got)):
        assert len(out) == 40
        steps.open(r)
        logits = steps.step([StepEntry(r, p + out[:-1], list(range(len(p) - 1, len(p) + 39)))]).float().cpu().numpy()
        steps.close(r)
        for k, t in enumerate(out):
            row = logits[k]
            ties += t != int(row.argmax())
            assert row.max() - row[t] <= 2 * bound * max(1.0, np.abs(row).max()), (r, k)
    assert ties <= 12


@pytest.mark.parametrize("case,dtype", [("a", "float32"), ("c", "bfloat16"), ("d", "bfloat16"), ("w", "bfloat16")])
def test_a_drafters_steps_are_the_engines_own_to_the_bit(case, dtype):
    """Every single-token step of the drafter, over pages' ends and rewinds, against an engine that is fed the same tokens at the same positions: the tables are written by
    a kernel of the step, ahead of kernels that read them early. And the same generation again gives the same rounds."""
    from geneinfer_b200.engine.loading import load_model
    from geneinfer_b200.engine.step import StepEngine, StepEntry
    vocab = gf.CASES[case][0]["vocab_size"]
    engine = speculative(case, case, dtype, max_running=1, max_seq_len=120, page_size=8)
    prompt, seen, rounds = tc.random_tokens(11, vocab, 77), [], []
    real = engine.draft.forward

    def forward(tokens, counts, counts_dev, lengths, *rest, **more):
        at = (tokens.clone(), lengths.clone())
        logits = real(tokens, counts, counts_dev, lengths, *rest, **more)
        seen.append((*at, None if logits is None else logits.clone()))
        return logits

    engine.draft.forward = forward
    for _ in range(4):
        engine.rounds = engine.kept = 0
        rounds.append((engine.generate([prompt], max_new_tokens=90), engine.rounds, engine.kept))
    assert all(r == rounds[0] for r in rounds)
    steps = StepEngine(load_model(gf.model_dir(case), dtype=dtype, max_position=128), n_pages=32, max_requests=1, page_size=8)
    steps.open(0)
    some = 0
    for tokens, length, logits in seen:
        tokens, length = tokens.tolist(), int(length)
        if length == 0 or steps.cache.requests[0].length > length:
            steps.truncate(0, length)
        got = steps.step([StepEntry(0, tokens, [len(tokens) - 1])])
        if logits is not None:
            assert torch.equal(got, logits), length
            some += 1
    assert some >= 4 * 72


def test_the_profile_of_a_step_has_the_requests_adapter_in_it(tmp_path, capsys):
    from geneinfer_b200.cli.generate_main import main
    folder, _ = adapter_and_merged("a", 16, tmp_path)
    common = ["--model", gf.model_dir("a"), "--prompt-ids", "5 9 2 100", "--steps", "8", "--temperature", "0", "--dtype", "fp32", "--quiet", "--profile"]
    assert main(common) == 0
    assert "low-rank adapters" not in capsys.readouterr().err
    assert main([*common, "--adapter", folder]) == 0
    line = next(l for l in capsys.readouterr().err.splitlines() if "low-rank adapters" in l)
    assert int(line.split("low-rank adapters")[1].split()[0]) == 4 * 2          # four projections of two layers


@pytest.mark.parametrize("drafts", [2, 6])
def test_generation_with_drafts_over_the_ends_of_the_attentions_chunks(drafts):
    """Contexts that grow from below 256 positions to the model's 512, beside a short one: the bounds on the lengths, by which launches are sized, run ahead of the lengths."""
    from geneinfer_b200 import Engine
    prompts = [tc.random_tokens(n, 500, 300 + n) for n in (250, 312, 5)]
    want = Engine(gf.model_dir("c"), dtype="float32", max_running=3).generate(prompts, max_new_tokens=200)
    engine = speculative("c", "c", "float32", drafts=drafts, max_seq_len=512, page_size=8)
    assert engine.generate(prompts, max_new_tokens=200) == want
    assert engine.kept >= 0.95 * engine.proposed > 0
    other = speculative("c", "c", "bfloat16", drafts=drafts, max_seq_len=512)
    first = other.generate(prompts, max_new_tokens=200)
    assert other.generate(prompts, max_new_tokens=200) == first and [len(f) for f in first] == [200] * 3
