"""What a request brings of its own, on the host: sampling parameters, the loop that hands them on, the
masks' bits, adapters' names and their place beside a fused projection."""
import math

import numpy as np
import pytest
import torch

import plain_requests as plain
from foundry_b200.engine import adapters
from foundry_b200.engine.generate import GenerateError, generate
from foundry_b200.parts.adapters import AdapterSite
from foundry_b200.sampling import SamplingParams, is_ruled, params_of_rows
from foundry_b200.sampling.rules import bias_room, check_vocabulary, mask_bits
from test_generate_loop import ScriptedBackend


@pytest.mark.parametrize("wrong", [
    dict(temperature=-1.0), dict(temperature=math.nan), dict(top_k=-1), dict(top_k=2.5), dict(top_p=0.0),
    dict(top_p=1.5), dict(top_p=math.nan), dict(min_p=-0.1), dict(min_p=1.1), dict(repetition_penalty=0.0),
    dict(repetition_penalty=math.inf), dict(frequency_penalty=math.nan), dict(presence_penalty=math.inf),
    dict(logit_bias={3: math.nan}), dict(logit_bias={3: math.inf}), dict(logit_bias={-3: 1.0}),
    dict(logit_bias=((3, 1.0), (3, 2.0)))])
def test_parameters_that_are_refused(wrong):
    with pytest.raises(ValueError):
        SamplingParams(**wrong)


def test_parameters_say_what_they_need():
    assert SamplingParams(0.7, 5).plain and not SamplingParams(0.7, 5).needs_history
    for more in (dict(top_k=3), dict(top_p=0.9), dict(min_p=0.1), dict(logit_bias={1: -math.inf}), dict(logprobs=True),
                 dict(allowed_tokens=lambda said: None)):
        p = SamplingParams(**more)
        assert not p.plain and not p.needs_history and is_ruled(p)
    for more in (dict(repetition_penalty=1.2), dict(frequency_penalty=0.1), dict(presence_penalty=-0.1)):
        assert SamplingParams(**more).needs_history
    a, b = SamplingParams(logit_bias={5: 1, 2: -3}), SamplingParams(logit_bias=((2, -3.0), (5, 1.0)))
    assert a == b and hash(a) == hash(b) and a.logit_bias == ((2, -3.0), (5, 1.0))


def test_rows_of_one_or_of_many():
    p, q = SamplingParams(0.5), SamplingParams(0.6)
    assert params_of_rows(p, 3) == [p, p, p] and params_of_rows((p, q), 2) == [p, q]
    assert not is_ruled(p) and not is_ruled([p, p]) and is_ruled([p, q])
    with pytest.raises(ValueError):
        params_of_rows([p], 2)


def test_room_for_biases_and_the_vocabulary():
    rows = [SamplingParams(logit_bias={i: 1.0 for i in range(n)}) for n in (0, 40, 30)]
    assert bias_room(rows) == 128 and bias_room(rows[:1]) == 0 and bias_room(rows[:2]) == 64
    check_vocabulary(rows, 40)
    with pytest.raises(ValueError, match="39"):
        check_vocabulary(rows, 39)


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 500])
def test_mask_bits(vocab):
    rng = np.random.RandomState(vocab)
    flags = rng.rand(vocab) < 0.4
    got = mask_bits(np.nonzero(flags)[0].tolist() * 2, vocab)  # a token twice is a token
    assert np.array_equal(got, plain.pack_bits(flags[None])[0])
    assert not mask_bits([], vocab).any()
    for token in (-1, vocab):
        with pytest.raises(ValueError, match="vocabulary"):
            mask_bits([token], vocab)


class RequestBackend(ScriptedBackend):
    def __init__(self, *args, **more):
        super().__init__(*args, **more)
        self.adapters, self.params = {}, []

    def open_sequence(self, adapter=None):
        slot = super().open_sequence()
        self.adapters[slot] = adapter
        return slot

    def step_select(self, steps, params, keys, counts, more=False):
        self.params.append((list(keys), params, [self.adapters[s.slot] for s in steps]))
        return super().step_select(steps, params, keys, counts, more)

    def last_logprobs(self):
        return [-float(k) - 0.5 for k in self.params[-1][0]]


def test_the_loop_hands_on_each_rows_own():
    script = {0: [10, 99, 12], 1: [20, 21, 22], 2: [30, 31, 32]}
    backend = RequestBackend(script)
    own = [SamplingParams(), SamplingParams(top_k=2, logprobs=True), SamplingParams(0.5)]
    out = generate(backend, [[1], [2, 3], [4]], 3, [99], own, adapters=["a", None, "b"])
    assert out.token_ids == [[10, 99], [20, 21, 22], [30, 31, 32]]
    assert out.logprobs == [[], [-1.5, -1.5, -1.5], []]
    assert backend.params == [([0, 1, 2], own, ["a", None, "b"]), ([0, 1, 2], own, ["a", None, "b"]),
                              ([1, 2], own[1:], [None, "b"])]
    for wrong in (dict(adapters=["a"]), dict(sampling=[SamplingParams()] * 2)):
        with pytest.raises(ValueError):
            generate(backend, [[1], [2], [3]], 2, **wrong)
    assert issubclass(GenerateError, ValueError)


# ------------------------------------------------------------------- adapters
def test_names_of_adapters_tensors():
    a, b = torch.zeros(4, 8), torch.zeros(6, 4)
    for style in ("base_model.model.m.0.q.{}.weight", "m.0.q.{}.weight", "base_model.model.m.0.q.{}.default.weight"):
        pairs = adapters.pairs_of({style.format("lora_A"): a, style.format("lora_B"): b})
        assert list(pairs) == ["m.0.q"] and pairs["m.0.q"] == (a, b)
    for wrong in ({"m.0.q.lora_A.weight": a}, {"m.0.q.weight": a},
                  {"m.0.q.lora_A.bias": a, "m.0.q.lora_B.weight": b}):
        with pytest.raises(adapters.AdapterError):
            adapters.pairs_of(wrong)


@pytest.mark.parametrize("given", [("q", "k", "v"), ("q",), ("k", "v"), ()])
def test_a_site_is_the_sum_of_its_projections(given):
    """The bank beside a fused and reordered matrix adds what each projection's adapter adds."""
    g = torch.Generator().manual_seed(3)
    rows, K, rank = {"q": 12, "k": 6, "v": 5}, 16, 8
    order = torch.randperm(23, generator=g)
    site = AdapterSite([(n, r) for n, r in rows.items()], K, order)
    site.make(3, rank, torch.float32, "cpu")
    pairs = {n: (torch.randn(5, K, generator=g), torch.randn(rows[n], 5, generator=g)) for n in given}
    site.write(1, pairs, 0.5)
    x = torch.randn(7, K, generator=g)
    got = site.bank.scales[1] * (x @ site.bank.a[1].T) @ site.bank.b[1].T
    parts = [0.5 * (x @ pairs[n][0].T) @ pairs[n][1].T if n in pairs else torch.zeros(7, r) for n, r in rows.items()]
    assert torch.allclose(got, torch.cat(parts, 1)[:, order], atol=1e-5)
    assert not site.bank.a[0].any() and not site.bank.b[2].any()
    site.clear(1)
    assert not site.bank.a.any() and not site.bank.b.any() and not site.bank.scales.any()


class FakeModel:
    class spec:
        architecture = "Fake"

    def __init__(self, with_sites=True):
        self._sites = [AdapterSite([("m.q", 6), ("m.k", 4)], 8)] if with_sites else []

    def parts(self):
        model = self

        class Takes:
            def adapter_sites(self):
                return model._sites
        return [object(), Takes()] if self._sites else [object()]


def pair(rows, rank=4, cols=8):
    return {"lora_A": torch.ones(rank, cols), "lora_B": torch.ones(rows, rank)}


def tensors(**projections):
    return {f"m.{p}.{half}.weight": t for p, halves in projections.items() for half, t in halves.items()}


def test_a_store_of_adapters():
    store = adapters.AdapterStore(FakeModel(), 2, 5, torch.float32, "cpu")
    assert store.max_rank == 8
    store.load("one", tensors(q=pair(6)))
    store.load("two", tensors(q=pair(6), k=pair(4, rank=8)), scale=2.0)
    assert store.place_of("one") != store.place_of("two")
    with pytest.raises(adapters.AdapterError, match="taken"):
        store.load("three", tensors(q=pair(6)))
    with pytest.raises(adapters.AdapterError, match="unload"):
        store.load("one", tensors(q=pair(6)))
    place = store.place_of("one")
    store.hold(place)
    store.hold(place)
    store.release(place)
    with pytest.raises(adapters.AdapterError, match="in use"):
        store.unload("one")
    store.release(place)
    store.unload("one")
    with pytest.raises(adapters.AdapterError, match="no adapter"):
        store.place_of("one")
    store.load("three", tensors(k=pair(4)))
    assert store.place_of("three") == place and not store.sites[0].bank.a[place][:8].any()


def test_adapters_that_do_not_fit():
    store = adapters.AdapterStore(FakeModel(), 2, 8, torch.float32, "cpu")
    endless = pair(6)
    endless["lora_B"][2, 1] = math.inf
    for wrong, word in ((tensors(v=pair(6)), "m.v"), (tensors(q=pair(5)), "m.q"), (tensors(q=pair(6, rank=9)), "rank 9"),
                        (tensors(q=pair(6, cols=9)), "m.q"), (tensors(q=endless), "finite"), ({}, "no tensors")):
        with pytest.raises(adapters.AdapterError, match=word):
            store.load("a", wrong)
    with pytest.raises(adapters.AdapterError, match="scale"):
        store.load("a", tensors(q=pair(6)), scale=math.nan)
    store.load("a", tensors(q=pair(6)))  # nothing was taken by what was refused
    store.load("b", tensors(q=pair(6)))
    with pytest.raises(adapters.AdapterError, match="takes adapters"):
        adapters.AdapterStore(FakeModel(False), 2, 8, torch.float32, "cpu")
    with pytest.raises(adapters.AdapterError, match="room"):
        adapters.AdapterStore(FakeModel(), 0, 8, torch.float32, "cpu")


def test_an_adapters_folder(tmp_path):
    import json
    from foundry_b200.weights.safetensors_io import save_file
    save_file({f"base_model.model.{k}": v for k, v in tensors(q=pair(6)).items()},
              str(tmp_path / "adapter_model.safetensors"))

    def config(**more):
        (tmp_path / "adapter_config.json").write_text(json.dumps({"r": 4, "lora_alpha": 8, **more}))
    config()
    got, scale = adapters.read_folder(str(tmp_path))
    assert scale == 2.0 and sorted(adapters.pairs_of(got)) == ["m.q"]
    config(use_rslora=True)
    assert adapters.read_folder(str(tmp_path))[1] == 4.0
    for more in (dict(use_dora=True), dict(bias="all"), dict(r=0), dict(r=None), dict(rank_pattern={"q": 3})):
        config(**more)
        with pytest.raises(adapters.AdapterError):
            adapters.read_folder(str(tmp_path))


def test_the_command_lines_options():
    from foundry_b200.cli import build_parser, sampling_of
    base = ["run", "--model", "m", "--prompt-ids", "1,2", "--max-new-tokens", "3"]
    assert sampling_of(build_parser().parse_args(base)) == SamplingParams()
    args = build_parser().parse_args(base + [
        "--temperature", "0.8", "--seed", "4", "--top-k", "40", "--top-p", "0.9", "--min-p", "0.05",
        "--repetition-penalty", "1.1", "--frequency-penalty", "0.2", "--presence-penalty", "0.3", "--adapter", "d"])
    assert sampling_of(args) == SamplingParams(0.8, 4, 40, 0.9, 0.05, 1.1, 0.2, 0.3) and args.adapter == "d"
