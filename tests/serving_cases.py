"""Inputs and plain 64-bit forms that the tests of the serving operators share:
attention over packed prompts and behind a shared prefix, and logits under
penalties, biases and masks."""
import numpy as np

from funasrnet_amd import hip

CODES = {"f32": hip.TYPE_F32, "f16": hip.TYPE_F16, "bf16": hip.TYPE_BF16}
# Half a step of a value in [1, 2): the largest relative rounding error.
HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


def store(x, kind):
    """float array -> the type's bits (round to nearest even), as numpy holds them."""
    x = np.asarray(x, np.float32)
    if kind == "f32":
        return x.copy()
    if kind == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    u = x.view(np.uint32).astype(np.uint64)
    rounded = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), rounded)


def load(a, kind):
    """The type's bits -> float32 values."""
    if kind == "bf16":
        return (a.astype(np.uint32) << 16).view(np.float32)
    return a.astype(np.float32)


def attend(q, k, v, scale, seen):
    """One head in 64 bits: softmax(scale q k^T) v over the keys seen[i, j], and
    per output the sum of p |v| and the largest sum |q k| of a score, of which
    rounding errors are fractions. Values that are not seen are not read."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    out, weight, dots = np.zeros_like(q), np.zeros_like(q), np.zeros((len(q), 1))
    for i in range(len(q)):
        at = np.flatnonzero(seen[i])
        if at.size == 0:
            continue
        s = scale * (k[at] @ q[i])
        top = s.max()
        if top == -np.inf:
            continue
        p = np.exp(s - top)
        out[i] = p @ v[at] / p.sum()
        weight[i] = p @ np.abs(v[at]) / p.sum()
        dots[i] = scale * (np.abs(k[at]) @ np.abs(q[i])).max()
    return out, weight, dots


def attend_all(q, k, v, scale, offset):
    """attend() for many rows: row i sees the keys up to i + offset; finite values."""
    q, k, v = (np.asarray(a, np.float64) for a in (q, k, v))
    s = scale * (q @ k.T)
    seen = np.arange(len(k))[None, :] <= np.arange(len(q))[:, None] + offset
    top = np.where(seen, s, -np.inf).max(1, keepdims=True, initial=-np.inf)
    p = np.where(seen, np.exp(s - np.where(np.isfinite(top), top, 0.0)), 0.0)
    total = np.maximum(p.sum(1, keepdims=True), 1e-300)
    return p @ v / total, p @ np.abs(v) / total, scale * (np.abs(q) @ np.abs(k).T).max(1, keepdims=True)


def attention_bound(out, weight, dots, keys, size, kind):
    """How far a correct result may be off, from the roundings it makes:
    a score sums `size` products in 32 bits (size + 3 half steps of sum |q k|,
    the queries' split into two 16-bit parts 4 more), which e^s turns into a
    relative error of p; exp2 and its argument 4; the sum over the keys one a
    key; each p rounded once to the values' type where queries are 16 bits (for
    fp32 queries p is held in two parts, 2^-22); and the output once."""
    u = 2.0**-24
    p_step = {"f32": 2.0**-22, "f16": 2.0**-11, "bf16": 2.0**-8}[kind]
    relative = 2 * ((size + 7) * u * dots + 4 * u * (1 + dots)) + 2 * (keys + 16) * u + p_step
    return weight * relative + np.abs(out) * HALF_STEP[kind] + 1e-30


def adjusted(x, history, prompt, repetition, presence, frequency, bias, mask, kind):
    """One row of logits in 32 bits, step by step, and the token chosen.
    bias: list of (token, value); mask: bool per token or None."""
    x = x.astype(np.float32).copy()
    vocab = len(x)
    f = np.float32
    count = {}
    for i, t in enumerate(history):
        if 0 <= t < vocab:
            count[t] = count.get(t, 0) + (1 if i >= prompt else 0)
    with np.errstate(all="ignore"):
        for t, n in count.items():
            x[t] = x[t] / f(repetition) if x[t] > 0 else x[t] * f(repetition)
            if n:
                x[t] = f(x[t] - f(f(frequency) * f(n)))
                x[t] = f(x[t] - f(presence))
        for t, value in {t: value for t, value in bias if 0 <= t < vocab}.items():
            x[t] = f(x[t] + f(value))
    if mask is not None:
        x[~mask] = -np.inf
    written = store(x, kind)
    y = load(written, kind)
    open_ = np.flatnonzero(y > -np.inf)
    token = -1 if open_.size == 0 else int(open_[np.argmax(y[open_])])
    return written, token
