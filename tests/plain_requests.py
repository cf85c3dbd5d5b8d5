"""Plain forms, in numpy, of what a request brings of its own: edits of its logits, the draw of its
token, its adapter beside a shared projection. Written from the formulas, apart from the kernels."""
import numpy as np

IN_PROMPT = 1 << 30


def pack_bits(flags):
    """bool [n, V] -> int32 [n, ceil(V / 32)], token i in bit i % 32 of word i // 32."""
    flags = np.asarray(flags, bool)
    n, V = flags.shape
    full = np.zeros((n, (V + 31) // 32 * 32), bool)
    full[:, :V] = flags
    return np.packbits(full, axis=1, bitorder="little").view(np.int32)


def counts_of(prompt, generated, vocab):
    counts = np.bincount(np.asarray(generated, np.int64), minlength=vocab).astype(np.int32)
    counts[np.unique(np.asarray(prompt, np.int64))] |= IN_PROMPT
    return counts


def edited(logits, counts=None, repetition=1.0, frequency=0.0, presence=0.0, bias=(), allowed=None,
           dtype=np.float32):
    """One row. In float32 every operation is rounded by itself, as the kernels round."""
    f = dtype
    v = np.array(logits, dtype=f)
    with np.errstate(all="ignore"):
        if counts is not None:
            said = (counts & (IN_PROMPT - 1)).astype(f)
            seen = counts != 0
            v = np.where(seen, np.where(v > 0, v / f(repetition), v * f(repetition)), v)
            v = np.where(said > 0, (v - f(frequency) * said) - f(presence), v)
        for token, value in bias:
            if 0 <= token < v.size:
                v[token] = v[token] + f(value)
        if allowed is not None:
            v = np.where(allowed, v, f(-np.inf))
    assert v.dtype == f
    return v


def noise(stream, step, vocab):
    """-log(-log u) of every token in 64 bits, u as the kernels make it (32 bits, below one)."""
    def mix(z):
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xbf58476d1ce4e5b9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94d049bb133111eb)
        return z ^ (z >> np.uint64(31))
    golden = np.uint64(0x9e3779b97f4a7c15)
    with np.errstate(over="ignore"):
        z = mix(np.uint64(stream % (1 << 64)) + golden * np.uint64(step + 1))
        z = mix(z + golden * np.arange(1, vocab + 1, dtype=np.uint64))
    u = (((z >> np.uint64(40)).astype(np.float64) + 0.5) * 2.0 ** -24).astype(np.float32)
    return -np.log(-np.log(np.minimum(u.astype(np.float64), 1.0 - 2.0 ** -24)))


def kept(v, temperature, top_k=0, top_p=1.0, min_p=0.0):
    """The tokens that the rules leave of a row of edited logits, in their order. The borders are the
    parameters as the kernels get them, in 32 bits."""
    v = np.where(np.isnan(v), -np.inf, v.astype(np.float64)) + 0.0
    best = v.max()
    with np.errstate(all="ignore"):
        z = np.where(v == best, 0.0, (v - best) / np.float64(np.float32(temperature)))
    order = np.lexsort((np.arange(v.size), -v))
    if top_k > 0:
        order = order[:top_k]
    w = np.exp(z[order])
    if top_p < 1:
        share = np.float64(np.float32(top_p)) * w.sum()
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        order, w = order[before < share], w[before < share]
    stays = w >= np.float64(np.float32(min_p))
    stays[0] = True
    return order[stays], z


def sampled(v, temperature=0.0, top_k=0, top_p=1.0, min_p=0.0, stream=0, step=0):
    """(token, log-probability) of one row of edited logits."""
    v = np.where(np.isnan(v), -np.inf, np.asarray(v, np.float64))
    if v.max() == -np.inf:
        return -1, -np.inf
    order, z = kept(v, temperature if temperature > 0 else 1.0, top_k, top_p, min_p)
    if temperature <= 0:
        token = int(np.argmax(v))
    else:
        order = np.sort(order)
        token = int(order[np.argmax(z[order] + noise(stream, step, v.size)[order])])
    return token, float(z[token] - np.log(np.exp(z).sum()))


def logprob_bound(v, token, temperature):
    """How far a 32-bit log-probability may be from the exact one: z = (v - M) / T takes three roundings
    (the difference, 1 / T, the product), exp of it two units more, the sum of the weights is 64-bit,
    the result one rounding. d log(sum) = sum w (3 |z| + 4) 2^-24 / sum w."""
    v = np.where(np.isnan(v), -np.inf, np.asarray(v, np.float64))
    z = np.where(v == v.max(), 0.0, (v - v.max()) / (temperature if temperature > 0 else 1.0))
    w = np.exp(z)
    size = np.where(w > 0, np.abs(np.where(np.isfinite(z), z, 0.0)), 0.0)
    lp = abs(z[token] - np.log(w.sum()))
    return 2.0 ** -24 * (3 * abs(z[token]) + lp + (w * (3 * size + 4)).sum() / w.sum()) + 1e-45


def adapted(x, w, a, b, scales, index):
    """y in 64 bits, the sum of |rank number x B| products, and the sum of |x w| products."""
    x, w, a, b = (np.asarray(t, np.float64) for t in (x, w, a, b))
    y = x @ w.T
    size, much = np.zeros_like(y), np.abs(x) @ np.abs(w).T
    for s in range(a.shape[0]):
        rows = np.nonzero(np.asarray(index) == s)[0]
        low = float(scales[s]) * (x[rows] @ a[s].T)
        much_low = abs(float(scales[s])) * (np.abs(x[rows]) @ np.abs(a[s]).T)
        y[rows] += low @ b[s].T
        size[rows] += np.abs(low) @ np.abs(b[s]).T
        much[rows] += much_low @ np.abs(b[s]).T
    return y, size, much


def adapted_bound(y, size, much, terms, bf16):
    """Per element: `terms` 32-bit additions of products whose absolute sum is `much` (each rounding at
    most 2^-24 of a partial sum, which is at most `much`); in bfloat16 also one rounding of every
    rank number (2^-8 of it, so 2^-8 of `size`) and the result's own 2^-8."""
    bound = terms * 2.0 ** -24 * much + 2.0 ** -24 * np.abs(y)
    return bound + 2.0 ** -8 * (size + np.abs(y)) * 1.01 if bf16 else bound
