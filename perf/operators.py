"""What a request brings of its own to a step that many requests share, measured case by case:

  edit     its history's penalties, its biases and its grammar mask, on its row of the logits
           (`ops.edit_logits`)
  sample   the same, and the draw of its next token under its own temperature, top-k, top-p and
           min-p, with the token's log-probability (`ops.sample_tokens`)
  adapted  a shared projection with its own low-rank adapter beside it (`ops.adapted_product`)

Layouts: logits are float32 rows. A history is a row of a table: `counts` (bits 0..29 how often the
token was generated, bit 30 whether the prompt holds it) and `seen` (a bit a token, set where the
count is not zero). A mask is a row of bits, set where a token is allowed. Biases are lists of
ascending token ids. Adapters are `a` [slots, rank, in], `b` [slots, out, rank] and a scale each.
"""
import math
import random

import numpy as np
import torch

own = False

IN_PROMPT = 1 << 30
GOLDEN, M1, M2 = 0x9e3779b97f4a7c15, 0xbf58476d1ce4e5b9, 0x94d049bb133111eb
LARGEST_U = 1.0 - 2.0 ** -24  # the largest 32-bit number below one


# ------------------------------------------------------------------- the cases
def listed():
    def logits(name, kind, rows, vocab, rule="", history=0, biased=0, masked=0.0, pad=0):
        return dict(name=name, kind=kind, rows=rows, vocab=vocab, rule=rule, history=history,
                    biased=biased, masked=masked, pad=pad)

    def adapted(name, tokens, size_in, size_out, rank, adapters, sequences, dtype="bfloat16"):
        return dict(name=name, kind="adapted", tokens=tokens, size_in=size_in, size_out=size_out,
                    rank=rank, adapters=adapters, sequences=sequences, dtype=dtype, pad=0)
    return [
        # a short chat of one user with a penalty for what it said before: latency alone
        logits("edit x1 32000", "edit", 1, 32000, history=300),
        # a busy server of a large vocabulary: long histories, biases, half the replies in a grammar
        logits("edit x64 128256", "edit", 64, 128256, history=4000, biased=300, masked=0.5),
        # rows of a wider buffer, an odd vocabulary
        logits("edit x7 50021 strided", "edit", 7, 50021, history=1000, biased=40, masked=0.3, pad=11),
        # one user, the usual nucleus
        logits("sample x1 128256 top-p", "sample", 1, 128256, "top_p"),
        # a handful of users with rules of their own, penalties and biases
        logits("sample x8 32000 mixed", "sample", 8, 32000, "mixed", history=800, biased=20),
        # many replies drawn among the k best
        logits("sample x33 50021 top-k", "sample", 33, 50021, "top_k", pad=11),
        # a busy server: every kind of rule beside every kind of edit
        logits("sample x64 128256 mixed", "sample", 64, 128256, "mixed", history=4000, biased=300,
               masked=0.25),
        # one user's adapter beside an output projection of the 1B layer size
        adapted("adapted 1b x1", 1, 2048, 2048, 16, 1, 1),
        # gate and up of the 8B layer size, eight replies with five adapters
        adapted("adapted 8b x8", 8, 4096, 28672, 32, 5, 8),
        # an output projection for a full batch of replies, a dozen adapters
        adapted("adapted 8b x48", 48, 4096, 4096, 64, 12, 48),
        # q, k and v of three prompts prefilled together, two of which have an adapter
        adapted("adapted 8b prompt 2048", 2048, 4096, 6144, 48, 2, 3),
        # the 32-bit path
        adapted("adapted 1b f32 333", 333, 2048, 2048, 8, 2, 3, "float32"),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    """One more case of the same ranges; no larger than the largest listed one."""
    kind = rng.choice(["edit", "sample", "sample", "adapted", "adapted"])
    if kind != "adapted":
        vocab = rng.choice([32000, 128256, _spread(rng, 1000, 150000)])
        return dict(kind=kind, rows=_spread(rng, 1, 64), vocab=vocab,
                    rule=rng.choice(["greedy", "plain", "top_k", "top_p", "min_p", "mixed"])
                    if kind == "sample" else "",
                    history=_spread(rng, 1, 4000) if kind == "edit" else
                    rng.choice([0, _spread(rng, 1, 4000)]),
                    biased=rng.choice([0, _spread(rng, 1, 300)]),
                    masked=rng.choice([0.0, 0.0, 0.5, 1.0]), pad=rng.choice([0, 0, 11, 64]))
    size = rng.choice([1024, 2048, 4096, 8 * rng.randint(32, 512)])
    tokens = rng.choice([_spread(rng, 1, 64), _spread(rng, 1, 2048)])
    sequences = rng.choice([tokens if tokens <= 64 else 4, rng.randint(1, min(tokens, 12))])
    dtype = "bfloat16" if rng.random() < 0.75 else "float32"
    return dict(kind="adapted", tokens=tokens if dtype == "bfloat16" else min(tokens, 600),
                size_in=size, size_out=rng.choice([1024, 2048, 4096, 6144, rng.randint(200, 6000)]),
                rank=8 * rng.randint(1, 12), adapters=rng.randint(1, 8),
                sequences=min(sequences, 600), dtype=dtype, pad=rng.choice([0, 0, 8, 64]))


# ------------------------------------------------------------------ the inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)
    return g


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device="cuda")


def _pack_bits(flags):
    """bool [n, V] -> int32 [n, ceil(V / 32)], token i in bit i % 32 of word i // 32."""
    n, V = flags.shape
    words = (V + 31) // 32
    full = torch.zeros(n, words * 32, dtype=torch.bool, device=flags.device)
    full[:, :V] = flags
    weights = torch.ones(32, dtype=torch.int64, device=flags.device) << torch.arange(
        32, device=flags.device)
    packed = (full.view(n, words, 32) * weights).sum(-1)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)


def _rows_of(case, seed):
    """Logits with a few likely tokens a row, and what each row's request brings."""
    g, n, V = _generator(seed), case["rows"], case["vocab"]
    rng = random.Random(int(seed))
    wide = torch.randn(n, V + case["pad"], generator=g, device="cuda") * 2.2
    logits = wide[:, :V]
    likely = torch.randint(0, V, (n, 40), generator=g, device="cuda")
    logits.scatter_add_(1, likely, 2.0 + 9.0 * _rand(g, n, 40))
    s = dict(kind=case["kind"], logits=logits, history=None, bias=None, mask=None)
    if case["history"]:
        h = case["history"]
        lengths = torch.randint(1, h + 1, (n, 1), generator=g, device="cuda")
        lengths[0] = h
        place = torch.arange(h, device="cuda")[None]
        ids = (V * _rand(g, n, h) ** 3).long().clamp_(max=V - 1)
        said = ((place >= lengths // 2) & (place < lengths)).to(torch.int32)
        read = (place < lengths // 2).to(torch.int32)
        zero = lambda: torch.zeros(n, V, dtype=torch.int32, device="cuda")  # noqa: E731
        mine = zero().scatter_add_(1, ids, said)
        mine += (zero().scatter_add_(1, ids, read) > 0).to(torch.int32) * IN_PROMPT
        rows = torch.randperm(n + 2, generator=g, device="cuda")[:n]
        counts = torch.zeros(n + 2, V, dtype=torch.int32, device="cuda")
        counts[rows] = mine
        s["history"] = dict(
            counts=counts, seen=_pack_bits(counts != 0), rows=rows.to(torch.int32),
            repetition=1.0 + 0.3 * _rand(g, n), frequency=0.5 * _rand(g, n),
            presence=0.8 * _rand(g, n))
    if case["biased"]:
        ids, values, starts = [], [], [0]
        for r in range(n):
            some = sorted(rng.sample(range(V), rng.randint(0, min(V, case["biased"]))))
            ids += some
            values += [rng.choice([-math.inf, rng.uniform(-8.0, 8.0)]) for _ in some]
            starts.append(len(ids))
        s["bias"] = dict(starts=torch.tensor(starts, dtype=torch.int32, device="cuda"),
                         ids=torch.tensor(ids, dtype=torch.int32, device="cuda"),
                         values=torch.tensor(values, dtype=torch.float32, device="cuda"))
    if case["masked"]:
        masked = [r for r in range(n) if rng.random() < case["masked"]] or [n - 1]
        share = torch.tensor([rng.choice([0.002, 0.05, 0.9]) for _ in masked], device="cuda")
        allowed = _rand(g, len(masked), V) < share[:, None]
        allowed[:, V // 2] = True
        which = [-1] * n
        for i, r in enumerate(masked):
            which[r] = i
        s["mask"] = dict(bits=_pack_bits(allowed),
                         rows=torch.tensor(which, dtype=torch.int32, device="cuda"))
    if case["kind"] == "sample":
        temperature, top_k, top_p, min_p = [], [], [], []
        for _ in range(n):
            rule = case["rule"]
            if rule == "mixed":
                rule = rng.choice(["greedy", "plain", "top_k", "top_p", "min_p", "all"])
            temperature.append(0.0 if rule == "greedy" else rng.uniform(0.5, 1.3))
            top_k.append(rng.choice([1, 20, 50, 400]) if rule in ("top_k", "all") else 0)
            top_p.append(rng.choice([0.8, 0.9, 0.95]) if rule in ("top_p", "all") else 1.0)
            min_p.append(rng.choice([0.02, 0.1]) if rule in ("min_p", "all") else 0.0)
        f32 = lambda v: torch.tensor(v, dtype=torch.float32, device="cuda")  # noqa: E731
        i64 = lambda v: torch.tensor(v, dtype=torch.int64, device="cuda")  # noqa: E731
        s["rules"] = dict(temperature=f32(temperature),
                          top_k=torch.tensor(top_k, dtype=torch.int32, device="cuda"),
                          top_p=f32(top_p), min_p=f32(min_p),
                          streams=i64([rng.getrandbits(64) - (1 << 63) for _ in range(n)]),
                          steps=i64([rng.randint(0, 4000) for _ in range(n)]))
    return s


def _projection_of(case, seed):
    g, T, K, N, R = (_generator(seed), case["tokens"], case["size_in"], case["size_out"],
                     case["rank"])
    dtype = torch.bfloat16 if case["dtype"] == "bfloat16" else torch.float32
    rng = random.Random(int(seed))
    S = case["adapters"]
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    cuts = sorted(rng.sample(range(1, T), case["sequences"] - 1)) if T > 1 else []
    index = []
    for i, (start, end) in enumerate(zip([0] + cuts, cuts + [T])):
        # every adapter where there are sequences enough, and now and then a request without one
        index += [i % S if i < S else rng.randint(-1, S - 1)] * (end - start)
    return dict(kind="adapted", x=normal(T, K + case["pad"]).to(dtype)[:, :K],
                w=(0.02 * normal(N, K)).to(dtype), a=(normal(S, R, K) / math.sqrt(K)).to(dtype),
                b=(0.05 * normal(S, N, R)).to(dtype), scales=0.5 + 1.5 * _rand(g, S),
                index=torch.tensor(index, dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    return _projection_of(case, seed) if case["kind"] == "adapted" else _rows_of(case, seed)


# ------------------------------------------------------------------ plain forms
def _unpack_bits(bits, V):
    places = torch.arange(32, device=bits.device, dtype=torch.int32)
    return ((bits[:, :, None] >> places) & 1).reshape(bits.shape[0], -1)[:, :V] != 0


def _edited(s):
    """The edited logits, in 32 bits, each operation rounded by itself."""
    v = s["logits"]
    n, V = v.shape
    if s["history"] is not None:
        h = s["history"]
        held = h["counts"][h["rows"].long()]
        said = (held & (IN_PROMPT - 1)).to(torch.float32)
        rep = h["repetition"][:, None]
        v = torch.where(held != 0, torch.where(v > 0, v / rep, v * rep), v)
        v = torch.where(said > 0, (v - h["frequency"][:, None] * said) - h["presence"][:, None], v)
    if s["bias"] is not None:
        b = s["bias"]
        places = torch.arange(b["ids"].numel(), device=v.device)
        row = torch.bucketize(places, b["starts"][1:].long(), right=True)
        v = v.contiguous().view(-1).index_add(0, row * V + b["ids"].long(), b["values"]).view(n, V)
    if s["mask"] is not None:
        which = s["mask"]["rows"].long()
        allowed = _unpack_bits(s["mask"]["bits"], V)[which.clamp(min=0)] | (which < 0)[:, None]
        v = torch.where(allowed, v, torch.full_like(v, -math.inf))
    return v


def _shifted(z, bits):
    return (z >> bits) & ((1 << (64 - bits)) - 1)


def _signed(v):
    return v - (1 << 64) if v >= 1 << 63 else v


def _mixed(z):
    z = (z ^ _shifted(z, 30)) * _signed(M1)
    z = (z ^ _shifted(z, 27)) * _signed(M2)
    return z ^ _shifted(z, 31)


def _noise(streams, steps, V):
    """-log(-log u) of every token, u in (0, 1) from the row's stream and step."""
    ids = torch.arange(1, V + 1, device=streams.device)[None]
    z = _mixed(streams + (steps + 1) * _signed(GOLDEN))[:, None]
    z = _mixed(z + ids * _signed(GOLDEN))
    u = ((_shifted(z, 40).double() + 0.5) * 2.0 ** -24).float().clamp(max=LARGEST_U)
    return -torch.log(-torch.log(u.double()))


def _sampled(s):
    r, v = s["rules"], _edited(s)
    n, V = v.shape
    greedy = r["temperature"] <= 0
    T = torch.where(greedy, torch.ones_like(r["temperature"]), r["temperature"]).double()[:, None]
    best = v.max(1, keepdim=True).values
    z = (v.double() - best.double()) / T
    weight = torch.exp(z)
    # in order of value, the lower id first among equals
    order = torch.sort(v, dim=1, descending=True, stable=True).indices
    place = torch.arange(V, device=v.device)[None]
    k = torch.where(r["top_k"] > 0, r["top_k"], V).long()[:, None]
    sorted_weight = torch.where(place < k, weight.gather(1, order), 0.0)
    before = sorted_weight.cumsum(1) - sorted_weight
    p = r["top_p"].double()[:, None]
    kept = (place < k) & ((before < p * sorted_weight.sum(1, keepdim=True)) | (p >= 1))
    kept &= weight.gather(1, order) >= r["min_p"].double()[:, None]
    kept = torch.zeros_like(kept).scatter_(1, order, kept | (place == 0))
    score = z + _noise(r["streams"], r["steps"], V)
    score = torch.where(greedy[:, None], v.double(), torch.where(kept, score, -math.inf))
    first = torch.where(score == score.max(1, keepdim=True).values, place, V).min(1).values
    logprob = z.gather(1, first[:, None])[:, 0] - torch.log(weight.sum(1))
    return {"tokens": first.to(torch.int32), "logprobs": logprob.float()}


def _adapted(s):
    S, R, K = s["a"].shape
    x = s["x"].float()
    mine = s["index"][:, None] == torch.arange(S, device=x.device)[None]  # [T, S]
    low = (x @ s["a"].float().reshape(S * R, K).T).view(-1, S, R)
    low = low * torch.where(mine, s["scales"][None], 0.0)[:, :, None]
    up = s["b"].float().transpose(1, 2).reshape(S * R, -1)
    return (x @ s["w"].float().T + low.view(-1, S * R) @ up).to(s["x"].dtype)


# -------------------------------------------------------------------- one pass
def _edits(ops, s):
    h, b, m = s["history"], s["bias"], s["mask"]
    given = {}
    if h is not None:
        given.update(history=ops.TokenHistory(h["counts"], h["seen"]), history_rows=h["rows"],
                     repetition=h["repetition"], frequency=h["frequency"], presence=h["presence"])
    if b is not None:
        given.update(bias=ops.TokenBiases(b["starts"], b["ids"], b["values"]))
    if m is not None:
        given.update(allowed=m["bits"], allowed_rows=m["rows"])
    return ops.LogitEdits(**given)


def run(s):
    if own:
        from foundry_b200.kernels import ops
        if s["kind"] == "adapted":
            return ops.adapted_product(s["x"], s["w"], ops.AdapterBank(s["a"], s["b"], s["scales"]),
                                       s["index"])
        if s["kind"] == "edit":
            return ops.edit_logits(s["logits"], _edits(ops, s))
        r = s["rules"]
        tokens, logprobs = ops.sample_tokens(
            s["logits"], ops.SampleRules(r["temperature"], r["top_k"], r["top_p"], r["min_p"],
                                         r["streams"], r["steps"]), _edits(ops, s))
        return {"tokens": tokens, "logprobs": logprobs}
    if s["kind"] == "adapted":
        return _adapted(s)
    return _edited(s) if s["kind"] == "edit" else _sampled(s)


def work(case):
    if case["kind"] == "adapted":
        T, K, N, R = case["tokens"], case["size_in"], case["size_out"], case["rank"]
        used = min(case["adapters"], case["sequences"])
        size = 2 if case["dtype"] == "bfloat16" else 4
        return {"bytes": size * (T * K + N * K + T * N + used * R * (K + N)) + 4 * T,
                "flops": 2.0 * T * N * K + 2.0 * T * R * (K + N)}
    n, V = case["rows"], case["vocab"]
    # histories of half the longest on average, each token of one read once
    row = 4 * V + 2 * case["history"] + (V // 8 if case["history"] else 0) + 4 * case["biased"]
    row += case["masked"] * V / 8
    row += 4 * V if case["kind"] == "edit" else 48
    return {"bytes": float(n * row), "flops": float(n * V * (4 if case["kind"] == "edit" else 8))}


# ------------------------------------------------------------------- in 64 bits
def _bits_of(words, V):
    raw = np.ascontiguousarray(words.cpu().numpy()).view(np.uint8)
    return np.unpackbits(raw, axis=1, bitorder="little")[:, :V].astype(bool)


def _exact_logits(s):
    v = s["logits"].cpu().numpy().astype(np.float64)
    if s["history"] is not None:
        h = {k: t.cpu().numpy() for k, t in s["history"].items()}
        for r in range(v.shape[0]):
            held = h["counts"][h["rows"][r]]
            seen = np.nonzero(held)[0]
            rep = float(h["repetition"][r])
            row = v[r, seen]
            row = np.where(row > 0, row / rep, row * rep)
            times = (held[seen] % IN_PROMPT).astype(np.float64)
            row -= (float(h["frequency"][r]) * times + float(h["presence"][r])) * (times > 0)
            v[r, seen] = row
    if s["bias"] is not None:
        starts, ids, values = (s["bias"][k].cpu().numpy() for k in ("starts", "ids", "values"))
        for r in range(v.shape[0]):
            mine = slice(starts[r], starts[r + 1])
            v[r, ids[mine]] += values[mine]
    if s["mask"] is not None:
        allowed = _bits_of(s["mask"]["bits"], v.shape[1])
        for r, which in enumerate(s["mask"]["rows"].tolist()):
            if which >= 0:
                v[r, ~allowed[which]] = -np.inf
    return v


def _exact_uniform(stream, step, V):
    def mix(z):
        z = (z ^ (z >> np.uint64(30))) * np.uint64(M1)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(M2)
        return z ^ (z >> np.uint64(31))
    with np.errstate(over="ignore"):
        z = mix(np.uint64(stream % (1 << 64)) + np.uint64(GOLDEN) * np.uint64(step + 1))
        z = mix(z + np.uint64(GOLDEN) * np.arange(1, V + 1, dtype=np.uint64))
    u = ((z >> np.uint64(40)).astype(np.float64) + 0.5) / 16777216.0
    return np.minimum(u.astype(np.float32).astype(np.float64), LARGEST_U)


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "adapted":
        x, y = s["x"].double(), None
        y = x @ s["w"].double().T
        for a in range(s["a"].shape[0]):
            rows = (s["index"] == a).nonzero()[:, 0]
            low = x[rows] @ s["a"][a].double().T
            y[rows] += float(s["scales"][a]) * (low @ s["b"][a].double().T)
        return y
    v = _exact_logits(s)
    if case["kind"] == "edit":
        return v
    rules = {k: t.tolist() for k, t in s["rules"].items()}
    logprobs = []
    for r, row in enumerate(v):
        T = rules["temperature"][r]
        if T <= 0:
            token = int(np.argmax(row))
            logprobs.append(row[token] - row.max() - np.log(np.exp(row - row.max()).sum()))
            continue
        z = (row - row.max()) / T
        order = np.lexsort((np.arange(z.size), -z))
        if rules["top_k"][r] > 0:
            order = order[:rules["top_k"][r]]
        w = np.exp(z[order])
        if rules["top_p"][r] < 1:
            reach = np.searchsorted(np.cumsum(w), rules["top_p"][r] * w.sum())
            order, w = order[:reach + 1], w[:reach + 1]
        order = order[w >= rules["min_p"][r]]
        u = _exact_uniform(rules["streams"][r], rules["steps"][r], z.size)[order]
        token = order[np.argmax(z[order] - np.log(-np.log(u)))]
        logprobs.append(z[token] - np.log(np.exp(z).sum()))
    return {"tokens": None, "logprobs": np.array(logprobs)}
