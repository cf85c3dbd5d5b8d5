"""Edits of logits and the draw under a row's own rules, against the plain forms."""
import numpy as np
import pytest
import torch

import plain_requests as plain

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    from foundry_b200.kernels import ops
    return ops


def dev(a, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(a), dtype=dtype).to(DEV)


class Rows:
    """Rows of logits and their requests' edits, on the host and on the device."""

    def __init__(self, ops, n, V, seed, history=True, biased=True, masked=True, pad=0, empty_row=None,
                 wild=False):
        rng = np.random.RandomState(seed)
        wide = (rng.randn(n, V + pad) * 3).astype(np.float32)
        wide[:, :V][rng.rand(n, V) < 0.02] += 8
        if wild:  # values that only a model gone wrong has
            for value in (np.inf, -np.inf, np.nan, -0.0):
                wide[:, :V][rng.rand(n, V) < 0.02] = value
        self.logits = wide[:, :V]
        self.device_logits = dev(wide)[:, :V]
        self.n, self.V = n, V
        self.each = [dict() for _ in range(n)]
        given = {}
        if history:
            table = np.zeros((n + 3, V), np.int32)
            places = rng.permutation(n + 3)[:n].astype(np.int32)
            rep, freq, pres = (rng.uniform(1, 1.5, n).astype(np.float32),
                               rng.uniform(-0.5, 1, n).astype(np.float32),
                               rng.uniform(-0.5, 1, n).astype(np.float32))
            for r in range(n):
                length = int(rng.randint(0, 2 * V + 2))
                ids = (V * rng.rand(length) ** 2).astype(int)
                table[places[r]] = plain.counts_of(ids[:length // 3], ids[length // 3:], V)
            if n > 2:  # rows without a history
                places[1], places[2] = -1, n + 3
            for r in range(n):
                if 0 <= places[r] < n + 3:
                    self.each[r].update(counts=table[places[r]], repetition=rep[r], frequency=freq[r],
                                        presence=pres[r])
            self.history = ops.TokenHistory(dev(table), dev(plain.pack_bits(table != 0)))
            given.update(history=self.history, history_rows=dev(places), repetition=dev(rep),
                         frequency=dev(freq), presence=dev(pres))
        if biased:
            maps = []
            for r in range(n):
                some = rng.choice(V, size=min(V, int(rng.randint(0, 40))), replace=False)
                maps.append({int(t): float(np.float32(rng.choice([-np.inf, rng.uniform(-5, 5)])))
                             for t in some})
            given["bias"] = ops.TokenBiases.from_rows(maps, DEV)
            for r in range(n):
                self.each[r]["bias"] = sorted(maps[r].items())
        if masked:
            masks = rng.rand(3, V) < np.array([[0.05], [0.5], [0.9]])
            masks[:, V // 2] = True
            if empty_row is not None:
                masks[2] = False
            which = rng.randint(-1, 3, n).astype(np.int32)
            which[n // 2] = 1
            if empty_row is not None:
                which[which == 2] = 0
                which[empty_row] = 2
            given.update(allowed=dev(plain.pack_bits(masks)), allowed_rows=dev(which))
            for r in range(n):
                if which[r] >= 0:
                    self.each[r]["allowed"] = masks[which[r]]
        self.edits = ops.LogitEdits(**given)

    def edited(self, dtype=np.float32):
        return np.stack([plain.edited(self.logits[r], dtype=dtype, **self.each[r]) for r in range(self.n)])


def same(got, want):
    got, want = got.cpu().numpy(), np.asarray(want)
    assert got.shape == want.shape and got.dtype == want.dtype
    assert np.array_equal(got, want, equal_nan=True), np.argwhere(~((got == want) | (got != got)))[:5]


# ------------------------------------------------------------------------ edits
@pytest.mark.parametrize("V", [1, 2, 31, 32, 33, 1000, 4096, 4097, 32003])
@pytest.mark.parametrize("n,pad", [(1, 0), (3, 5), (7, 64)])
def test_edits_are_the_32_bit_formulas(ops, V, n, pad):
    rows = Rows(ops, n, V, seed=V + n, pad=pad)
    got = ops.edit_logits(rows.device_logits, rows.edits)
    same(got, rows.edited())
    # and the formulas of 64 bits, as near as four 32-bit operations come (5 with a bias): each is off
    # by 2^-24 of its result at most, and no result here is larger than the sum of the parts' sizes
    exact = rows.edited(np.float64)
    size = np.abs(rows.logits) * 1.5 + np.abs(exact)
    for r, row in enumerate(rows.each):
        if "counts" in row:
            said = row["counts"] & (plain.IN_PROMPT - 1)
            size[r] += abs(row["frequency"]) * said + abs(row["presence"])
        for t, value in row.get("bias", ()):
            size[r, t] += abs(value)
    fine = np.isfinite(exact)
    assert np.array_equal(fine, np.isfinite(got.cpu().numpy()))
    off = np.abs(got.cpu().numpy()[fine].astype(np.float64) - exact[fine])
    assert (off <= 6 * 2.0 ** -24 * size[fine]).all()


@pytest.mark.parametrize("kind", ["history", "biased", "masked"])
def test_each_kind_of_edit_alone(ops, kind):
    only = {k: k == kind for k in ("history", "biased", "masked")}
    rows = Rows(ops, 4, 777, seed=5, **only)
    same(ops.edit_logits(rows.device_logits, rows.edits), rows.edited())


def test_no_edits_copy_the_rows(ops):
    rows = Rows(ops, 3, 100, 1, history=False, biased=False, masked=False, pad=3)
    same(ops.edit_logits(rows.device_logits, rows.edits), rows.logits)


def test_edits_of_infinities_and_nan(ops):
    rows = Rows(ops, 6, 2000, seed=3, wild=True, empty_row=4)
    got = ops.edit_logits(rows.device_logits, rows.edits)
    same(got, rows.edited())
    assert (got[4] == -np.inf).all()  # masked places are -inf whatever they held


def test_edits_in_place_and_into_a_wider_buffer(ops):
    rows = Rows(ops, 5, 4500, seed=8, pad=7)
    want = rows.edited()
    wide = torch.full((5, 4600), 7.0, device=DEV)
    out = ops.edit_logits(rows.device_logits, rows.edits, out=wide[:, 50:4550])
    same(out, want)
    assert (wide[:, :50] == 7).all() and (wide[:, 4550:] == 7).all()
    assert ops.edit_logits(rows.device_logits, rows.edits, out=rows.device_logits) is rows.device_logits
    same(rows.device_logits, want)


def test_equal_ids_add_up_and_foreign_ids_do_nothing(ops):
    V = 5000
    logits = torch.zeros(2, V, device=DEV)
    ids = torch.tensor([-3, 4, 4, 4, 4095, 4096, V, V + 9, 7], dtype=torch.int32, device=DEV)
    values = torch.tensor([9, 0.25, 0.5, 1, 3, -2, 9, 9, 5], dtype=torch.float32, device=DEV)
    starts = torch.tensor([0, 8, 9], dtype=torch.int32, device=DEV)
    got = ops.edit_logits(logits, ops.LogitEdits(bias=ops.TokenBiases(starts, ids, values))).cpu()
    want = torch.zeros(2, V)
    want[0, 4], want[0, 4095], want[0, 4096], want[1, 7] = 1.75, 3, -2, 5
    assert torch.equal(got, want)


# -------------------------------------------------------------------- histories
def test_recorded_tokens(ops):
    V, rng = 333, np.random.RandomState(0)
    history = ops.TokenHistory.empty(4, V, DEV)
    prompt, said = rng.randint(0, V, (4, 500)), rng.randint(0, 40, (4, 300))
    rows = np.repeat(np.arange(4), 500)
    ops.record_tokens(history, dev(rows, torch.int32), dev(prompt.reshape(-1), torch.int32), "prompt")
    rows = np.repeat(np.arange(4), 300)
    ops.record_tokens(history, dev(rows, torch.int32), dev(said.reshape(-1), torch.int32))
    want = np.stack([plain.counts_of(prompt[r], said[r], V) for r in range(4)])
    same(history.counts, want)
    same(history.seen, plain.pack_bits(want != 0))
    # the last hundred of each row are taken back, and more of token 5 than there are
    back = [(r, t) for r in range(4) for t in said[r, 200:]] + [(2, 5)] * 400
    ops.record_tokens(history, dev([r for r, _ in back], torch.int32), dev([t for _, t in back], torch.int32),
                      "taken back")
    want = np.stack([plain.counts_of(prompt[r], said[r, :200], V) for r in range(4)])
    want[2, 5] &= plain.IN_PROMPT
    same(history.counts, want)
    same(history.seen, plain.pack_bits(want != 0))
    # rows and tokens outside of the table change nothing
    ops.record_tokens(history, dev([-1, 4, 0, 0], torch.int32), dev([1, 1, -1, V], torch.int32))
    same(history.counts, want)
    history.clear([1, 3])
    want[[1, 3]] = 0
    same(history.counts, want)
    same(history.seen, plain.pack_bits(want != 0))


# ------------------------------------------------------------------------ draws
def check(ops, logits, edited, rules, edits=None, **more):
    """Draws the rows on the device and compares tokens and log-probabilities."""
    n = len(edited)
    f32 = lambda k: None if k not in rules else dev(rules[k], torch.float32)  # noqa: E731
    i64 = lambda k: None if k not in rules else dev(rules[k], torch.int64)  # noqa: E731
    given = ops.SampleRules(f32("temperature"), None if "top_k" not in rules else dev(rules["top_k"], torch.int32),
                            f32("top_p"), f32("min_p"), i64("streams"), i64("steps"))
    tokens, logprobs = ops.sample_tokens(logits, given, edits, **more)
    tokens, logprobs = tokens.cpu().numpy(), logprobs.cpu().numpy()
    for r in range(n):
        one = {a: rules[b][r] for a, b in (("temperature", "temperature"), ("top_k", "top_k"), ("top_p", "top_p"),
                                           ("min_p", "min_p"), ("stream", "streams"), ("step", "steps"))
               if b in rules}
        T = float(np.float32(one.get("temperature", 0.0)))
        one["temperature"] = T
        token, logprob = plain.sampled(edited[r], **one)
        assert tokens[r] == token, (r, one, tokens[r], token)
        if token < 0:
            assert logprobs[r] == -np.inf
        else:
            assert abs(float(logprobs[r]) - logprob) <= plain.logprob_bound(edited[r], token, T), (r, logprobs[r], logprob)
    return tokens


def rules_of(n, seed, temperature=(0.0, 0.7, 1.0, 1.4), top_k=(0, 1, 3, 40), top_p=(1.0, 0.3, 0.9, 0.99),
             min_p=(0.0, 0.05, 0.5, 1.0)):
    rng = np.random.RandomState(seed)
    pick = lambda some: [some[i] for i in rng.randint(0, len(some), n)]  # noqa: E731
    return dict(temperature=pick(temperature), top_k=pick(top_k), top_p=pick(top_p), min_p=pick(min_p),
                streams=[int(s) for s in rng.randint(-2 ** 62, 2 ** 62, n)],
                steps=[int(s) for s in rng.randint(0, 3000, n)])


@pytest.mark.parametrize("V", [1, 2, 31, 32, 33, 257, 4096, 4097, 8193, 32003])
@pytest.mark.parametrize("n,pad", [(1, 0), (40, 5)])
def test_draws_under_every_rule(ops, V, n, pad):
    rows = Rows(ops, n, V, seed=V + 7, pad=pad)
    check(ops, rows.device_logits, rows.edited(), rules_of(n, V), rows.edits)


@pytest.mark.parametrize("spread", [0.0005, 0.02, 0.3, 1.0])
@pytest.mark.parametrize("V", [3000, 32003, 100000])
def test_borders_among_many_nearly_equal_logits(ops, V, spread):
    """A flat row's border lies in a bin of more tokens than the sorted list holds; 32-bit logits close to
    ten then have few values, and thousands of tokens share one."""
    n = 12
    rng = np.random.RandomState(V)
    logits = (10 + spread * rng.randn(n, V)).astype(np.float32)
    rules = dict(temperature=[0.5, 1.0, 2.0] * 4, top_k=[0, V // 2, 700, V - 1] * 3,
                 top_p=[0.6, 0.1, 0.999] * 4, streams=list(range(n)), steps=[4] * n)
    check(ops, dev(logits), logits, rules)


def test_rows_and_histories_past_32_bits(ops):
    """Rows 1.2 billion logits apart, and a history whose last rows lie behind 2^31 counts."""
    rows = Rows(ops, 3, 128256, seed=6)
    wide = torch.zeros(3 * 1200000000, device=DEV)
    logits = wide.view(3, -1)[:, 700:700 + 128256]
    logits.copy_(rows.device_logits)
    e = rows.edits
    many = 17000
    h = ops.TokenHistory.empty(many, 128256, DEV)
    assert h.counts.numel() > 1 << 31
    places = torch.where(e.history_rows >= 0, e.history_rows + many - e.history.rows, -1).to(torch.int32)
    h.counts[-e.history.rows:] = e.history.counts
    h.seen[-e.history.rows:] = e.history.seen
    edits = ops.LogitEdits(h, places, e.repetition, e.frequency, e.presence, e.bias, e.allowed, e.allowed_rows)
    same(ops.edit_logits(logits, edits), rows.edited())
    check(ops, logits, rows.edited(), rules_of(3, 1), edits)
    last = torch.tensor([many - 1] * 3, dtype=torch.int32, device=DEV)
    before = h.counts[-1, [9, 128255]].clone()
    ops.record_tokens(h, last, torch.tensor([9, 128255, 9], dtype=torch.int32, device=DEV), "generated")
    assert torch.equal(h.counts[-1, [9, 128255]] - before, torch.tensor([2, 1], dtype=torch.int32, device=DEV))


@pytest.mark.parametrize("rule", [{}, dict(top_k=[20] * 8), dict(top_p=[0.5] * 8)])
def test_an_infinite_temperature_gives_equal_shares(ops, rule):
    n, V = 8, 3000
    logits = np.random.RandomState(0).randn(n, V).astype(np.float32)
    logits[:, 5] = -np.inf
    draw = lambda heat: ops.sample_tokens(dev(logits), ops.SampleRules(  # noqa: E731
        dev([heat] * n, torch.float32), dev(rule.get("top_k"), torch.int32) if "top_k" in rule else None,
        dev(rule["top_p"], torch.float32) if "top_p" in rule else None, None,
        torch.arange(n, device=DEV), torch.arange(n, device=DEV)))
    tokens, logprobs = draw(np.inf)
    same_tokens, _ = draw(3e38)
    assert torch.equal(tokens, same_tokens) and (tokens != 5).all()
    assert torch.allclose(logprobs, torch.full_like(logprobs, -float(np.log(V - 1))), rtol=1e-6)


@pytest.mark.parametrize("m", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 257, 600, 3000])
@pytest.mark.parametrize("V,n", [(7000, 6), (70000, 6), (7000, 200)])
def test_borders_in_a_bin_of_so_many_tokens(ops, V, n, m):
    """`m` tokens within a thirtieth of each other, a few in front of them, nothing to speak of behind:
    both rules' borders among them, in the bin's first, a middle and its last token."""
    rng = np.random.RandomState(m)
    logits = np.full((n, V), -40.0, np.float32)
    for r in range(n):
        at = rng.permutation(V)[:m + 3]
        logits[r, at[:3]] = (3.0, 2.5, 2.0)
        logits[r, at[3:]] = (1.0 + 0.029 * rng.rand(m)).astype(np.float32)
    first = np.exp(np.array([0.0, -0.5, -1.0])).sum()
    inside = m * np.exp(-2.0 + 0.0145)
    share = lambda x: float(np.float32((first + x * inside) / (first + inside)))  # noqa: E731
    k = [0, 3 + (m + 1) // 2, 4, 0, 3 + m, 3 + (m + 1) // 2]
    p = [share(0.5), 1.0, 1.0, share(0.02), share(0.99), 0.8]
    rules = dict(temperature=[1.0] * n, top_k=(k * n)[:n], top_p=(p * n)[:n], streams=list(range(n)), steps=[m] * n)
    check(ops, dev(logits), logits, rules)


@pytest.mark.parametrize("size,heat", [(1e6, 0.01), (3e7, 2.0), (1e-30, 1e-31), (200.0, 0.003), (1.0, 1e5)])
def test_logits_and_temperatures_of_any_size(ops, size, heat):
    """Steps between neighbouring 32-bit logits wider than a bin of the histogram, logits near the
    smallest numbers, temperatures that make all tokens or one of them likely."""
    n, V = 12, 6000
    rng = np.random.RandomState(3)
    logits = (size * (1 + 1e-6 * rng.randn(n, V))).astype(np.float32)
    logits[::2] = (size * rng.randn(6, V)).astype(np.float32)
    rules = dict(temperature=[heat] * n, top_k=[0, 0, 700, 50] * 3, top_p=[0.9, 0.5, 0.7] * 4,
                 streams=list(range(n)), steps=[4] * n)
    check(ops, dev(logits), logits, rules)


def test_a_history_of_nearly_all_tokens(ops):
    """More of the history's tokens in a block's share of a row than its list has room for."""
    n, V = 10, 150016
    rng = np.random.RandomState(8)
    logits = (rng.randn(n, V) * 3).astype(np.float32)
    table = rng.randint(0, 4, (n, V)).astype(np.int32)
    table[rng.rand(n, V) < 0.3] |= plain.IN_PROMPT
    table[0] = 1
    rep, freq, pres = (np.full(n, v, np.float32) for v in (1.3, 0.2, 0.1))
    edits = ops.LogitEdits(ops.TokenHistory(dev(table), dev(plain.pack_bits(table != 0))), torch.arange(n, dtype=torch.int32, device=DEV),
                           dev(rep), dev(freq), dev(pres))
    edited = np.stack([plain.edited(logits[r], table[r], rep[r], freq[r], pres[r]) for r in range(n)])
    same(ops.edit_logits(dev(logits), edits), edited)
    check(ops, dev(logits), edited, rules_of(n, 8), edits)


def test_draws_of_a_large_vocabulary(ops):
    rows = Rows(ops, 12, 128256, seed=2)
    check(ops, rows.device_logits, rows.edited(), rules_of(12, 2, top_k=(0, 50, 1000, 100000)), rows.edits)


@pytest.mark.parametrize("V", [131072, 131073, 264192, 264193, 368640, 528384])
def test_draws_of_the_largest_vocabularies(ops, V):
    rows = Rows(ops, 3, V, seed=4, history=False, biased=False, masked=False)
    check(ops, rows.device_logits, rows.logits, rules_of(3, 4, temperature=(0.9,)), None)


@pytest.mark.parametrize("what", ["top_k", "top_p", "min_p"])
def test_one_rule_and_many_streams(ops, what):
    """A thousand draws from one row of few tokens: every border is met."""
    n, V = 1000, 60
    row = (np.random.RandomState(1).randn(V) * 2).astype(np.float32)
    value = {"top_k": 7, "top_p": 0.8, "min_p": 0.1}[what]
    rules = dict(temperature=[0.8] * n, streams=list(range(n)), steps=[3] * n, **{what: [value] * n})
    tokens = check(ops, dev(np.tile(row, (n, 1))), np.tile(row, (n, 1)), rules)
    allowed, _ = plain.kept(row, 0.8, **{what: value})
    assert set(tokens) <= set(allowed.tolist()) and len(set(tokens)) == len(allowed)


@pytest.mark.parametrize("V", [64, 5000, 40000])
@pytest.mark.parametrize("k", [1, 5, 63, 4000])
def test_equal_logits_are_cut_by_their_index(ops, V, k):
    """A handful of values for all tokens: the border runs through thousands of equal ones."""
    rng = np.random.RandomState(V + k)
    logits = rng.randint(-2, 3, (9, V)).astype(np.float32)
    logits[8] = 0.0
    logits[7] = np.where(rng.rand(V) < 0.5, 0.0, -0.0)
    rules = dict(temperature=[1.0] * 9, top_k=[k] * 9, streams=list(range(9)), steps=[0] * 9)
    check(ops, dev(logits), logits, rules)
    rules = dict(temperature=[2.0] * 9, top_p=[0.4] * 9, streams=list(range(9)), steps=[0] * 9)
    check(ops, dev(logits), logits, rules)


@pytest.mark.parametrize("V,p,left", [(8, 0.5, 4), (8, 0.51, 5), (8, 0.125, 1), (8, 0.0, 0), (4096, 0.25, 1024),
                                      (65536, 0.75, 49152)])
def test_a_share_that_is_reached_exactly(ops, V, p, left):
    """Equal weights of one: the sums are whole numbers, and the prefix that reaches the share ends
    where it is reached. A share of nothing keeps the first token."""
    n = 300
    logits = np.zeros((n, V), np.float32)
    rules = dict(temperature=[1.0] * n, top_p=[p] * n, streams=list(range(n)), steps=[1] * n)
    if p > 0:
        assert len(plain.kept(logits[0], 1.0, top_p=p)[0]) == left
        tokens = check(ops, dev(logits), logits, rules)
        assert tokens.max() < left
    else:
        got, _ = ops.sample_tokens(dev(logits), ops.SampleRules(
            dev(rules["temperature"], torch.float32), None, dev(rules["top_p"], torch.float32), None,
            dev(rules["streams"], torch.int64), dev(rules["steps"], torch.int64)))
        assert (got == 0).all()


def test_rows_without_a_token_and_rows_gone_wrong(ops):
    n, V = 9, 6000
    logits = np.random.RandomState(6).randn(n, V).astype(np.float32)
    logits[0] = -np.inf
    logits[1] = np.nan
    logits[2, 5:] = -np.inf                     # five left
    logits[3, [70, 5000]] = np.inf              # only these have a chance
    logits[4] = np.finfo(np.float32).min        # all at the type's lowest value
    logits[5, ::2] = np.nan
    logits[6] = -np.inf
    logits[6, 4321] = 3.0
    for heat in (0.0, 0.9):
        rules = dict(temperature=[heat] * n, top_k=[0, 0, 20, 20, 20, 20, 20, 20, 0],
                     top_p=[0.9, 0.9, 0.99, 0.9, 1.0, 0.9, 0.9, 1.0, 0.9], streams=list(range(n)), steps=[2] * n)
        also = torch.full((n,), 77, dtype=torch.int32, device=DEV)
        tokens = check(ops, dev(logits), logits, rules, also=also)
        assert tokens[0] == tokens[1] == -1 and tokens[6] == 4321
        assert also.cpu().tolist() == [max(0, t) for t in tokens]


def test_a_mask_that_leaves_nothing(ops):
    rows = Rows(ops, 6, 3000, seed=3, empty_row=2)
    tokens = check(ops, rows.device_logits, rows.edited(), rules_of(6, 3), rows.edits)
    assert tokens[2] == -1


def test_without_rules_it_is_the_plain_selection(ops):
    n, V = 30, 20000
    logits = torch.randn(n, V, generator=torch.Generator().manual_seed(0)).to(DEV)
    heat = torch.tensor([0.8 * (i % 2) for i in range(n)], device=DEV)
    streams, steps = torch.arange(n, device=DEV) * 999, torch.arange(n, device=DEV)
    want = ops.select_tokens(logits, torch.empty(n, dtype=torch.int32, device=DEV), heat, streams, steps)
    got, _ = ops.sample_tokens(logits, ops.SampleRules(heat, streams=streams, steps=steps))
    assert torch.equal(got, want)


def test_the_largest_uniform_number_wins_nothing_by_itself(ops):
    """Token 11's uniform number rounds to one in 32 bits: its noise is large, not infinite."""
    V, step = 64, 0
    # by inverting the mix: u of (stream, step, token 11) has all 24 bits set
    stream = _stream_with_full_bits(step, 11)
    assert _bits24(stream, step, 11) == (1 << 24) - 1
    logits = np.zeros((1, V), np.float32)
    logits[0, 5] = 40.0
    check(ops, dev(logits), logits, dict(temperature=[1.0], streams=[stream], steps=[step]))


_M = (1 << 64) - 1
_G, _A, _B = 0x9e3779b97f4a7c15, 0xbf58476d1ce4e5b9, 0x94d049bb133111eb


def _mix(z):
    z = ((z ^ (z >> 30)) * _A) & _M
    z = ((z ^ (z >> 27)) * _B) & _M
    return z ^ (z >> 31)


def _unmix(z):
    def unshift(y, s):
        x = y
        for _ in range(64 // s + 1):
            x = y ^ (x >> s)
        return x
    z = unshift(z, 31)
    z = unshift((z * pow(_B, -1, 1 << 64)) & _M, 27)
    return unshift((z * pow(_A, -1, 1 << 64)) & _M, 30)


def _bits24(stream, step, token):
    z = _mix((stream + _G * (step + 1)) & _M)
    return _mix((z + _G * (token + 1)) & _M) >> 40


def _stream_with_full_bits(step, token):
    z = (_unmix(_M) - _G * (token + 1)) & _M
    stream = (_unmix(z) - _G * (step + 1)) & _M
    return stream - (1 << 64) if stream >> 63 else stream


def test_a_step_records_its_inputs_first(ops):
    rows = Rows(ops, 8, 9000, seed=12)
    inputs = np.random.RandomState(5).randint(0, 9000, 8)
    places = rows.edits.history_rows.cpu().numpy()
    counts = rows.history.counts.cpu().numpy()
    for r in range(8):
        if 0 <= places[r] < counts.shape[0]:
            rows.each[r]["counts"] = rows.each[r]["counts"].copy()
            rows.each[r]["counts"][inputs[r]] += 1
            counts[places[r], inputs[r]] += 1
    check(ops, rows.device_logits, rows.edited(), rules_of(8, 9), rows.edits, record=dev(inputs, torch.int32))
    same(rows.history.counts, counts)
    same(rows.history.seen, plain.pack_bits(counts != 0))


def test_draws_on_another_stream_and_replayed(ops):
    rows = Rows(ops, 5, 40000, seed=21, history=True)
    rules = rules_of(5, 21)
    given = ops.SampleRules(dev(rules["temperature"], torch.float32), dev(rules["top_k"], torch.int32),
                            dev(rules["top_p"], torch.float32), dev(rules["min_p"], torch.float32),
                            dev(rules["streams"], torch.int64), dev(rules["steps"], torch.int64))
    want = ops.sample_tokens(rows.device_logits, given, rows.edits)
    edited = ops.edit_logits(rows.device_logits, rows.edits)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.sample_tokens(rows.device_logits, given, rows.edits)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.sample_tokens(rows.device_logits, given, rows.edits)
        captured_edits = ops.edit_logits(rows.device_logits, rows.edits)
    with torch.cuda.graph(other):
        again = ops.sample_tokens(rows.device_logits, given, rows.edits)
    for _ in range(3):
        with torch.cuda.stream(side):
            graph.replay()
        other.replay()
    torch.cuda.synchronize()
    for got in (captured, again):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert torch.equal(captured_edits, edited)


def test_the_same_call_gives_the_same_bits(ops):
    rows = Rows(ops, 16, 50021, seed=30)
    rules = ops.SampleRules(torch.full((16,), 1.1, device=DEV), None, torch.full((16,), 0.95, device=DEV),
                            streams=torch.arange(16, device=DEV), steps=torch.arange(16, device=DEV))
    first = ops.sample_tokens(rows.device_logits, rules, rows.edits)
    for _ in range(5):
        again = ops.sample_tokens(rows.device_logits, rules, rows.edits)
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_no_rows(ops):
    logits = torch.empty(0, 50, device=DEV)
    tokens, logprobs = ops.sample_tokens(logits, ops.SampleRules())
    assert tokens.shape == logprobs.shape == (0,)
    assert ops.edit_logits(logits, ops.LogitEdits()).shape == (0, 50)
