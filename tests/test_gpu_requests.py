"""Requests with adapters and sampling rules of their own through the engine, against the plain model:
merged weights for the adapters, the plain edits and draws on the plain logits."""
import math

import numpy as np
import pytest
import torch

import plain_llama
import plain_requests as plain
import tiny

pytestmark = pytest.mark.gpu

TARGETS = {"self_attn": ("q_proj", "k_proj", "v_proj", "o_proj"), "mlp": ("gate_proj", "up_proj", "down_proj")}


def engine_of(folder, dtype="float32", **more):
    from foundry_b200 import Engine
    more = {**dict(max_tokens=4096, max_slots=8), **more}
    return Engine.from_folder(folder, dtype=dtype, **more)


def make_adapter(cfg, weights, seed, rank=4, scale=1.5, targets=TARGETS, size=0.25):
    """(tensors as an adapter's file holds them, the weights with it merged in)."""
    g = torch.Generator().manual_seed(seed)
    tensors, merged = {}, dict(weights)
    for layer in range(cfg["num_hidden_layers"]):
        for part, names in targets.items():
            for name in names:
                p = f"model.layers.{layer}.{part}.{name}"
                w = torch.as_tensor(weights[p + ".weight"]).double()
                a = (torch.randn(rank, w.shape[1], generator=g) / math.sqrt(w.shape[1])).bfloat16()
                b = (size * torch.randn(w.shape[0], rank, generator=g)).bfloat16()
                tensors[f"base_model.model.{p}.lora_A.weight"] = a
                tensors[f"base_model.model.{p}.lora_B.weight"] = b
                merged[p + ".weight"] = w + scale * b.double() @ a.double()
    return tensors, merged


@pytest.fixture(scope="module")
def setting(tiny_folders):
    cfg, weights = plain_llama.read_model(tiny_folders["tiny_b"])
    one, merged_one = make_adapter(cfg, weights, 1)
    two, merged_two = make_adapter(cfg, weights, 2, rank=7, scale=-0.7,
                                   targets={"self_attn": ("k_proj", "o_proj"), "mlp": ("up_proj", "down_proj")})
    return dict(folder=tiny_folders["tiny_b"], cfg=cfg, models={None: weights, "one": merged_one, "two": merged_two},
                tensors={"one": one, "two": two}, scales={"one": 1.5, "two": -0.7})


def adapted_engine(setting, dtype="float32", **more):
    engine = engine_of(setting["folder"], dtype, **more)
    engine.enable_adapters(max_adapters=3, max_rank=8)
    for name in ("one", "two"):
        engine.load_adapter(name, setting["tensors"][name], setting["scales"][name])
    return engine


def logits_of(setting, name, tokens):
    return np.asarray(plain_llama.forward(setting["cfg"], setting["models"][name], list(tokens)), np.float64)


# ------------------------------------------------------------------- adapters
LENS = [(3,), (5, 21, 1, 9), (150, 40, 200)]


def rows_for(setting, lens):
    names = ["one", None, "two", "one"][:len(lens)]
    return names, [tiny.random_tokens(50 + i, n + 4, setting["cfg"]["vocab_size"]) for i, n in enumerate(lens)]


def stepped(engine, names, rows, lens):
    """Logits of a prompt step of all rows and of three single tokens each: [row, step, vocab]."""
    from foundry_b200 import SequenceStep
    slots = [engine.open_sequence(name) if name else engine.open_sequence() for name in names]
    got = [engine.step([SequenceStep(s, r[:n], [n - 1]) for s, r, n in zip(slots, rows, lens)]).cpu().numpy()]
    for k in range(3):
        got.append(engine.step([SequenceStep(s, [r[n + k]], [0]) for s, r, n in zip(slots, rows, lens)]).cpu().numpy())
    for s in slots:
        engine.close_sequence(s)
    return np.stack(got, 1).astype(np.float64)


@pytest.mark.parametrize("lens", LENS)
def test_adapters_are_their_merged_weights(setting, lens):
    """Prompts of several adapters in one step, then single tokens of all."""
    names, rows = rows_for(setting, lens)
    got = stepped(adapted_engine(setting), names, rows, lens)
    for i, n in enumerate(lens):
        want = logits_of(setting, names[i], rows[i])[n - 1:n + 3]
        tiny.assert_logits_close(got[i], want, "float32", f"{names[i]}, prompt of {n}")


@pytest.mark.parametrize("lens", LENS)
def test_adapters_in_16_bits_are_as_near_as_merged_weights_in_16_bits(setting, tmp_path, lens):
    """The yardstick is an engine of the same type that runs the merged weights: it rounds the weights
    where adapters round their rank numbers, and the same activations, so the two are equally far from
    the exact logits (root mean square over all of a row's, half as much again for chance)."""
    import os
    import shutil
    from foundry_b200.weights.safetensors_io import SINGLE_FILE, save_file
    names, rows = rows_for(setting, lens)
    engine = adapted_engine(setting, "bfloat16")
    got = stepped(engine, names, rows, lens)
    for i, n in enumerate(lens):
        if names[i] is None:
            continue
        folder = str(tmp_path / names[i])
        if not os.path.exists(folder):
            os.makedirs(folder)
            shutil.copy(os.path.join(setting["folder"], "config.json"), folder)
            save_file({k: torch.as_tensor(v).to(torch.bfloat16) for k, v in setting["models"][names[i]].items()},
                      os.path.join(folder, SINGLE_FILE), metadata={"format": "pt"})
        merged = stepped(engine_of(folder, "bfloat16"), [None], [rows[i]], [n])[0]
        want = logits_of(setting, names[i], rows[i])[n - 1:n + 3]
        rms = lambda v: float(np.sqrt(np.mean(v * v)))  # noqa: E731
        assert np.isfinite(got[i]).all()
        assert rms(got[i] - want) <= 1.5 * rms(merged - want), (names[i], rms(got[i] - want), rms(merged - want))


def test_a_prompt_in_pieces_and_plain_launches(setting):
    from foundry_b200 import SequenceStep
    engine = adapted_engine(setting)
    engine.use_graphs = False
    row = tiny.random_tokens(9, 60, setting["cfg"]["vocab_size"])
    want = logits_of(setting, "two", row)
    slot = engine.open_sequence("two")
    other = engine.open_sequence()
    engine.step([SequenceStep(slot, row[:25], []), SequenceStep(other, row[:3], [])])
    got = engine.step([SequenceStep(slot, row[25:], [34])])
    tiny.assert_logits_close(got[0].cpu().numpy(), want[59], "float32")


def test_steps_without_an_adapter_are_as_they_were(setting):
    """An engine with room for adapters runs unadapted steps as one without: bit for bit."""
    from foundry_b200 import SequenceStep
    row = tiny.random_tokens(4, 30, setting["cfg"]["vocab_size"])
    results = []
    for engine in (engine_of(setting["folder"], "bfloat16"), adapted_engine(setting, "bfloat16")):
        slot = engine.open_sequence()
        results.append([engine.step([SequenceStep(slot, row[:20], [19])]).clone()] +
                       [engine.step([SequenceStep(slot, [t], [0])]).clone() for t in row[20:]])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_generation_with_adapters(setting):
    engine = adapted_engine(setting)
    names = ["two", None, "one", "two", "one"]
    prompts = [tiny.random_tokens(70 + i, n, setting["cfg"]["vocab_size"]) for i, n in enumerate((4, 11, 1, 30, 7))]
    want = [plain_llama.greedy_generate(setting["cfg"], setting["models"][name], p, 8) for name, p in zip(names, prompts)]
    for max_batch in (None, 2):
        out = engine.generate(prompts, 8, eos_token_id=[], adapters=names, max_batch=max_batch)
        assert out.token_ids == want
    assert engine.generate(prompts[:2], 8, eos_token_id=[]).token_ids == [
        plain_llama.greedy_generate(setting["cfg"], setting["models"][None], p, 8) for p in prompts[:2]]


def test_places_of_adapters(setting):
    from foundry_b200.engine.adapters import AdapterError
    engine = engine_of(setting["folder"])
    with pytest.raises(ValueError, match="enable_adapters"):
        engine.open_sequence("one")
    engine.enable_adapters(1, 8)
    engine.load_adapter("one", setting["tensors"]["one"], 1.5)
    slot = engine.open_sequence("one")
    for refused in (lambda: engine.unload_adapter("one"), lambda: engine.open_sequence("two"),
                    lambda: engine.load_adapter("two", setting["tensors"]["two"])):
        with pytest.raises(AdapterError):
            refused()
    engine.close_sequence(slot)
    engine.unload_adapter("one")
    engine.load_adapter("two", setting["tensors"]["two"], -0.7)
    prompt = tiny.random_tokens(3, 12, setting["cfg"]["vocab_size"])
    out = engine.generate([prompt, prompt], 6, eos_token_id=[], adapters=["two", None])
    assert out.token_ids == [plain_llama.greedy_generate(setting["cfg"], setting["models"][n], prompt, 6)
                             for n in ("two", None)]


def test_adapters_beside_the_feed_forwards_of_another_architecture(tmp_path):
    """Parts are shared: an architecture with dense gated feed-forwards takes adapters beside them, here in
    a group of layers that runs three times, under norms behind the parts. Against an engine with the
    merged weights, in 32 bits (its mixers' projections take none)."""
    import rupotar_tiny
    from foundry_b200 import Engine, SequenceStep
    from foundry_b200.weights.safetensors_io import SINGLE_FILE, save_file
    folder, weights = rupotar_tiny.write_folder(str(tmp_path / "plain"), "looped")
    merged_folder, _ = rupotar_tiny.write_folder(str(tmp_path / "merged"), "looped")
    g = torch.Generator().manual_seed(0)
    tensors, merged = {}, dict(weights)
    for name in ("l0.mlp.gate", "l0.mlp.down", "l3.mlp.up"):
        rows, cols = weights[name].shape
        a, b = torch.randn(8, cols, generator=g) / cols ** 0.5, torch.randn(rows, 8, generator=g) * 0.3
        tensors[f"{name}.lora_A.weight"], tensors[f"{name}.lora_B.weight"] = a, b
        merged[name] = (weights[name].double() + 0.5 * b.double() @ a.double()).float()
    save_file(merged, str(tmp_path / "merged" / SINGLE_FILE), metadata={"format": "pt"})
    tokens = tiny.random_tokens(2, 18, 200)
    results = []
    for where, adapter in ((folder, "x"), (merged_folder, None), (folder, None)):
        engine = Engine.from_folder(where, dtype="float32", max_tokens=1024, max_slots=4)
        if adapter:
            engine.enable_adapters(2, 8)
            engine.load_adapter("x", tensors, 0.5)
        slot = engine.open_sequence(adapter) if adapter else engine.open_sequence()
        rows = [engine.step([SequenceStep(slot, tokens[:14], [13])])[0].cpu()]
        rows += [engine.step([SequenceStep(slot, [t], [0])])[0].cpu() for t in tokens[14:]]
        results.append(torch.stack(rows).double().numpy())
    # (both are within 2e-5 of the logit scale of the exact sums)
    scale = max(1.0, np.abs(results[1]).max())
    assert np.abs(results[0] - results[1]).max() <= 4e-5 * scale
    assert np.abs(results[2] - results[1]).max() > 1e-2 * scale


@pytest.mark.parametrize("family,name,names", [
    ("tokovik", "mixed", ("l0.mlp.gate", "l2.mlp.up", "l2.mlp.down")),
    ("tokovik", "other", ("l0.mlp.down", "l1.mlp.gate", "l1.mlp.up")),
    ("vonulorn", "mixed", ("l0.mlp.up", "l2.mlp.gate", "l3.mlp.down")),
    ("vonulorn", "other", ("l1.mlp.gate", "l2.mlp.down"))])
def test_adapters_under_every_arrangement_of_parts(tmp_path, family, name, names):
    """The same where a constant scales the parts' outputs, norms stand behind them, or the layers' streams
    are summed: what a part with adapters returns is taken like what it returns without."""
    import importlib
    from foundry_b200 import Engine, SequenceStep
    from foundry_b200.weights.safetensors_io import SINGLE_FILE, save_file
    made = importlib.import_module(f"{family}_tiny")
    folder, weights = made.write_folder(str(tmp_path / "plain"), name)
    merged_folder, _ = made.write_folder(str(tmp_path / "merged"), name)
    g = torch.Generator().manual_seed(0)
    tensors, merged = {}, dict(weights)
    for where in names:
        rows, cols = weights[where].shape
        a, b = torch.randn(8, cols, generator=g) / cols ** 0.5, torch.randn(rows, 8, generator=g) * 0.3
        tensors[f"{where}.lora_A.weight"], tensors[f"{where}.lora_B.weight"] = a, b
        merged[where] = (weights[where].double() + 0.5 * b.double() @ a.double()).float()
    save_file(merged, str(tmp_path / "merged" / SINGLE_FILE), metadata={"format": "pt"})
    tokens = tiny.random_tokens(3, 30, made.CONFIGS[name].get("vocab_size", made.CONFIGS[name].get("vocab", 64)))
    results = []
    for where, adapter in ((folder, "x"), (merged_folder, None), (folder, None)):
        engine = Engine.from_folder(where, dtype="float32", max_tokens=1024, max_slots=4)
        if adapter:
            engine.enable_adapters(2, 8)
            engine.load_adapter("x", tensors, 0.5)
        slot = engine.open_sequence(adapter) if adapter else engine.open_sequence()
        rows = [engine.step([SequenceStep(slot, tokens[:26], [25])])[0].cpu()]
        rows += [engine.step([SequenceStep(slot, [t], [0])])[0].cpu() for t in tokens[26:]]
        results.append(torch.stack(rows).double().numpy())
    # (both are within 2e-5 of the logit scale of the exact sums)
    scale = max(1.0, np.abs(results[1]).max())
    assert np.abs(results[0] - results[1]).max() <= 4e-5 * scale
    assert np.abs(results[2] - results[1]).max() > 1e-2 * scale


# ------------------------------------------------------------- rules and edits
def simulate(setting, prompt, params, key, steps, name=None, stops=()):
    """The plain model's tokens under a request's rules, their log-probabilities, and how far 32-bit ones
    may be off: each logit by 2e-5 of the largest (`tiny.assert_logits_close`), which a penalty may
    multiply and the temperature divides; a log-probability is the difference of two such numbers."""
    from foundry_b200.sampling import stream_key
    V = setting["cfg"]["vocab_size"]
    said, logprobs, bounds = [], [], []
    for count in range(steps):
        logits = logits_of(setting, name, list(prompt) + said)[-1]
        allowed = None
        if params.allowed_tokens is not None:
            ids = params.allowed_tokens(list(said))
            if ids is not None:
                allowed = np.zeros(V, bool)
                allowed[list(ids)] = True
        counts = plain.counts_of(prompt, said, V) if params.needs_history else None
        v = plain.edited(logits, counts, params.repetition_penalty, params.frequency_penalty, params.presence_penalty,
                         params.logit_bias, allowed, dtype=np.float64)
        token, logprob = plain.sampled(v, params.temperature, params.top_k, params.top_p, params.min_p,
                                       stream_key(params.seed, key), count)
        said.append(token)
        logprobs.append(logprob)
        off = 2e-5 * max(1.0, np.abs(logits).max()) * max(params.repetition_penalty, 1 / params.repetition_penalty)
        bounds.append(2 * off / (params.temperature or 1.0) + 1e-6)
        if token in stops:
            break
    return said, logprobs, bounds


def near(got, want, bounds):
    return len(got) == len(want) and all(abs(g - w) <= b for g, w, b in zip(got, want, bounds))


def rows_of_rules(V):
    from foundry_b200 import SamplingParams
    odd = lambda said: [t for t in range(V) if t % 2 == (1 + len(said)) % 2]  # noqa: E731
    return [SamplingParams(), SamplingParams(repetition_penalty=1.7, logprobs=True),
            SamplingParams(0.9, 4, top_k=5, frequency_penalty=0.8, presence_penalty=0.3, logprobs=True),
            SamplingParams(1.2, 5, top_p=0.8, min_p=0.02, logit_bias={7: -math.inf, 11: 2.0}, logprobs=True),
            SamplingParams(0.0, allowed_tokens=odd, logprobs=True),
            SamplingParams(0.8, 9, allowed_tokens=lambda said: None if len(said) % 2 else range(0, V, 3))]


@pytest.mark.parametrize("graphs", [True, False])
def test_rows_with_rules_of_their_own(setting, graphs):
    """All in one batch, some with adapters too: each row's tokens are the plain model's under its rules."""
    V = setting["cfg"]["vocab_size"]
    engine = adapted_engine(setting)
    engine.use_graphs = graphs
    rules = rows_of_rules(V)
    names = [None, "one", None, "two", "one", None]
    prompts = [tiny.random_tokens(20 + i, n, V) for i, n in enumerate((5, 1, 33, 8, 12, 2))]
    prompts[2][:10] = prompts[2][10:20]  # tokens that come twice
    out = engine.generate(prompts, 10, eos_token_id=[], sampling=rules, adapters=names)
    for r, (prompt, p, name) in enumerate(zip(prompts, rules, names)):
        tokens, logprobs, bounds = simulate(setting, prompt, p, r, 10, name)
        assert out.token_ids[r] == tokens, (r, p)
        if p.logprobs:
            assert near(out.logprobs[r], logprobs, bounds), r
        else:
            assert out.logprobs[r] == []


@pytest.mark.parametrize("which", [1, 2, 3])
def test_one_rule_for_all_and_steps_started_ahead(setting, which):
    """Rows end at different times on stop tokens, so steps that were started on a guess are taken back,
    and the histories with them; the same engine serves the next batch."""
    V = setting["cfg"]["vocab_size"]
    p = rows_of_rules(V)[which]
    engine = engine_of(setting["folder"])
    for batch in range(2):
        prompts = [tiny.random_tokens(30 + 7 * i + batch, 3 + 4 * i, V) for i in range(6)]
        free = [simulate(setting, prompt, p, r, 12) for r, prompt in enumerate(prompts)]
        stops = {free[0][0][2], free[1][0][4], free[4][0][3]}
        out = engine.generate(prompts, 12, eos_token_id=sorted(stops), sampling=p)
        for r, prompt in enumerate(prompts):
            tokens, logprobs, bounds = simulate(setting, prompt, p, r, 12, stops=stops)
            assert out.token_ids[r] == tokens, r
            assert near(out.logprobs[r], logprobs, bounds) if p.logprobs else out.logprobs[r] == []


def test_a_session_that_keeps_tokens_on_the_device(setting):
    """Device-resident steps with penalties count their own tokens."""
    from foundry_b200 import SamplingParams, SequenceStep
    V = setting["cfg"]["vocab_size"]
    p = SamplingParams(repetition_penalty=1.5, frequency_penalty=0.6)
    prompt = tiny.random_tokens(77, 9, V)
    want = simulate(setting, prompt, p, 0, 9)[0]
    engine = engine_of(setting["folder"])
    slot = engine.open_sequence()
    first = engine.step_select([SequenceStep(slot, prompt, [8])], p, [0], [0])
    session = engine.decode_session([slot], p, [0], [1])
    session.set_tokens(first)
    got = list(first)
    for _ in range(8):
        session.step()
        torch.cuda.synchronize()
        got += session.runner.next_tokens[:1].tolist()
    assert got == want


def test_masks_that_leave_nothing_and_masks_on_the_device(setting):
    from foundry_b200 import SamplingParams
    from foundry_b200.engine.generate import NoTokenLeft
    engine = engine_of(setting["folder"])
    prompt = [5, 6, 7]
    for stuck in (0, 2):
        p = SamplingParams(allowed_tokens=lambda said: [] if len(said) >= stuck else [9, 10])
        with pytest.raises(NoTokenLeft):
            engine.generate([prompt, [3]], 6, eos_token_id=[], sampling=[p, SamplingParams()])
        assert engine.free_slots() == 8
    p = SamplingParams(logit_bias={t: -math.inf for t in range(setting["cfg"]["vocab_size"])})
    with pytest.raises(NoTokenLeft):
        engine.generate([prompt], 3, eos_token_id=[], sampling=p)
    with pytest.raises(ValueError, match="vocabulary"):
        engine.generate([prompt], 3, sampling=SamplingParams(logit_bias={10 ** 6: 1.0}))
    slot = engine.open_sequence()
    session = engine.decode_session([slot], SamplingParams(allowed_tokens=lambda said: [1]), [0], [1])
    with pytest.raises(ValueError, match="step_host"):
        session.step()
    engine.close_sequence(slot)
    # and the engine goes on
    want = simulate(setting, prompt, SamplingParams(), 0, 5)[0]
    assert engine.generate([prompt], 5, eos_token_id=[]).token_ids == [want]


def test_a_slot_forgets_the_sequence_before(setting):
    from foundry_b200 import SamplingParams
    p = SamplingParams(repetition_penalty=3.0, presence_penalty=2.0)
    V = setting["cfg"]["vocab_size"]
    engine = engine_of(setting["folder"], max_slots=1)
    for seed in range(4):
        prompt = tiny.random_tokens(90 + seed, 6 + seed, V)
        assert engine.generate([prompt], 6, eos_token_id=[], sampling=p).token_ids == [
            simulate(setting, prompt, p, 0, 6)[0]]


def test_the_command_line_with_an_adapter_and_rules(setting, tmp_path, capsys):
    import json
    from foundry_b200 import SamplingParams
    from foundry_b200.cli import main
    from foundry_b200.weights.safetensors_io import save_file
    save_file(setting["tensors"]["one"], str(tmp_path / "adapter_model.safetensors"))
    (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 4, "lora_alpha": 6}))
    prompt = tiny.random_tokens(8, 10, setting["cfg"]["vocab_size"])
    assert main(["run", "--model", setting["folder"], "--dtype", "float32", "--prompt-ids", ",".join(map(str, prompt)),
                 "--max-new-tokens", "7", "--ignore-eos", "--temperature", "0.7", "--seed", "3", "--top-k", "6",
                 "--frequency-penalty", "0.5", "--adapter", str(tmp_path)]) == 0
    p = SamplingParams(0.7, 3, top_k=6, frequency_penalty=0.5)
    assert json.loads(capsys.readouterr().out) == simulate(setting, prompt, p, 0, 7, "one")[0]
