"""What a serving program asks of the attention and token-choice operators:
prompts of several recordings attended in one call, decoding over a prompt
prefix that every recording shares, and the choice of the next token under
penalties, biases and a grammar's mask.

`run` computes each operator from elementary torch operations in 32 bits, or,
with `own` set, calls the library's entry points (funasrnet_amd.hip). Sizes are
the decoder's (16 or 32 query heads and 8 K/V heads of 128, a vocabulary of
151936, an F16 K/V cache under fp32 activations) or generic.

torch is imported before the library: both then share one HIP runtime.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_VOCAB = 151936


def listed() -> list:
    return [
        # A spoken command's prompt: the smallest call, latency alone. Queries
        # are the decoder's fp32 rows, keys and values its F16 cache.
        {"name": "prompt_command", "kind": "packed", "sequences": 1, "rows_low": 37, "rows_high": 37, "cached_low": 0,
         "cached_high": 0, "heads": 16, "kv_heads": 8, "size": 128, "type": "f32", "cache": "f16"},
        # The prefix of one minute of audio.
        {"name": "prompt_minute", "kind": "packed", "sequences": 1, "rows_low": 750, "rows_high": 750, "cached_low": 0,
         "cached_high": 0, "heads": 16, "kv_heads": 8, "size": 128, "type": "f32", "cache": "f16"},
        # Recordings that arrived together, a second to a minute and a half each.
        {"name": "prompts_packed", "kind": "packed", "sequences": 24, "rows_low": 20, "rows_high": 1100, "cached_low": 0,
         "cached_high": 0, "heads": 16, "kv_heads": 8, "size": 128, "type": "f16", "cache": "f16"},
        # New audio behind transcripts that are cached already.
        {"name": "prompts_resumed", "kind": "packed", "sequences": 6, "rows_low": 1, "rows_high": 400, "cached_low": 500,
         "cached_high": 5000, "heads": 32, "kv_heads": 8, "size": 128, "type": "bf16", "cache": "bf16"},
        # The longest prompt: an hour's transcript to be revised.
        {"name": "prompt_longest", "kind": "packed", "sequences": 1, "rows_low": 8192, "rows_high": 8192, "cached_low": 0,
         "cached_high": 0, "heads": 32, "kv_heads": 8, "size": 128, "type": "bf16", "cache": "bf16"},
        # Two recordings behind an instruction and a few hot words.
        {"name": "prefix_pair", "kind": "prefix", "sequences": 2, "prefix": 300, "own_low": 1, "own_high": 150, "heads": 16,
         "kv_heads": 8, "size": 128, "type": "f32", "cache": "f16"},
        # A server's lock-step batch behind a long list of hot words.
        {"name": "prefix_sessions", "kind": "prefix", "sequences": 16, "prefix": 2048, "own_low": 100, "own_high": 750,
         "heads": 16, "kv_heads": 8, "size": 128, "type": "f32", "cache": "f16"},
        # Questions about one long document.
        {"name": "prefix_document", "kind": "prefix", "sequences": 61, "prefix": 8191, "own_low": 1, "own_high": 700,
         "heads": 32, "kv_heads": 8, "size": 128, "type": "bf16", "cache": "bf16"},
        # The largest batch, each with a minute of audio of its own.
        {"name": "prefix_batch", "kind": "prefix", "sequences": 256, "prefix": 4096, "own_low": 200, "own_high": 1400,
         "heads": 16, "kv_heads": 8, "size": 128, "type": "f16", "cache": "f16"},
        # One recording's next token: repeated text held back, hot words favoured.
        {"name": "choice_token", "kind": "choice", "rows": 1, "vocab": _VOCAB, "history": 300, "biases": 40, "masks": 0,
         "type": "f32"},
        # A lock-step batch whose rows follow a grammar's states.
        {"name": "choice_sessions", "kind": "choice", "rows": 16, "vocab": _VOCAB, "history": 1500, "biases": 200, "masks": 9,
         "type": "f32"},
        # The largest batch, in 16 bits.
        {"name": "choice_batch", "kind": "choice", "rows": 256, "vocab": _VOCAB, "history": 600, "biases": 64, "masks": 33,
         "type": "bf16"},
    ]


def _between(rng, low: int, high: int) -> int:
    """Log-uniform whole number of [low, high], low >= 1."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _draw_attention(rng) -> dict:
    kv_heads = rng.choice([8, 8, 8, 4, 2, 1, 3])
    group = rng.choice([2, 2, 4, 4, 1, 3, 5, 8])
    kind, cache = rng.choice([("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")])
    return {"heads": kv_heads * group, "kv_heads": kv_heads, "size": rng.choice([128, 128, 64, 96]), "type": kind,
            "cache": cache}


def _draw_once(rng) -> dict:
    kind = rng.choice(["packed", "packed", "prefix", "prefix", "choice"])
    if kind == "packed":
        sequences = rng.choice([1, _between(rng, 2, 64)])
        high = _between(rng, 1, 8192 if sequences == 1 else 2000)
        cached = rng.choice([0, 0, _between(rng, 1, 5000)])
        return {"kind": kind, "sequences": sequences, "rows_low": high if sequences == 1 else min(high, rng.choice([0, 1, 20])),
                "rows_high": high, "cached_low": cached // 4, "cached_high": cached, **_draw_attention(rng)}
    if kind == "prefix":
        high = _between(rng, 1, 1500)
        return {"kind": kind, "sequences": _between(rng, 1, 256), "prefix": _between(rng, 16, 8192),
                "own_low": min(high, rng.choice([0, 1, 200])), "own_high": high, **_draw_attention(rng)}
    return {"kind": kind, "rows": _between(rng, 1, 256), "vocab": rng.choice([_VOCAB, _between(rng, 2000, 160000)]),
            "history": rng.choice([0, _between(rng, 1, 4000)]), "biases": rng.choice([0, _between(rng, 1, 500)]),
            "masks": rng.choice([0, _between(rng, 1, 64)]), "type": rng.choice(list(_TYPES))}


def draw(rng) -> dict:
    """A case of these ranges that costs no more than the largest listed one of its kind."""
    most = {}
    for c in listed():
        w = work(c)
        for key in ("bytes", "flops"):
            most[c["kind"], key] = max(most.get((c["kind"], key), 0.0), w[key])
    while True:
        case = _draw_once(rng)
        w = work(case)
        if any(w[key] > most[case["kind"], key] for key in ("bytes", "flops")):
            continue
        if case["kind"] == "packed":
            queries, keys = _lengths(case)
            # The plain form pads every sequence to the longest one.
            if case["sequences"] * case["heads"] * max(queries) * max(keys, default=0) > 8192 * 8192 * 32 or sum(queries) < 1:
                continue
        return case


# ---- What a program has in hand -----------------------------------------------


def _spread(case: dict, salt: int, count: int, low: int, high: int) -> list:
    """`count` lengths of [low, high], spread over their logarithm, from the case's sizes alone."""
    rng = random.Random(count * 1_000_003 + low * 10_007 + high * 101 + case["heads"] + salt)
    return [min(high, max(low, round(math.exp(rng.uniform(math.log(low + 1), math.log(high + 1)))) - 1)) for _ in range(count)]


def _lengths(case: dict):
    """Query rows and key rows of each packed sequence."""
    queries = _spread(case, 1, case["sequences"], case["rows_low"], case["rows_high"])
    cached = _spread(case, 2, case["sequences"], case["cached_low"], case["cached_high"])
    return queries, [a + b for a, b in zip(queries, cached)]


def _owned(case: dict) -> list:
    """Each sequence's own cache rows behind the shared prefix."""
    return _spread(case, 3, case["sequences"], case["own_low"], case["own_high"])


def _offsets(lengths: list) -> torch.Tensor:
    total = [0]
    for n in lengths:
        total.append(total[-1] + n)
    return torch.tensor(total, dtype=torch.int32, device="cuda")


def _normal(gen, kind: str, *shape, scale: float = 1.0) -> torch.Tensor:
    return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(_TYPES[kind])


def _inputs(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "packed":
        queries, keys = _lengths(case)
        size, cache = case["size"], case["cache"]
        return {"q": _normal(gen, case["type"], sum(queries), case["heads"], size, scale=1.5),
                "k": _normal(gen, cache, sum(keys), case["kv_heads"], size),
                "v": _normal(gen, cache, sum(keys), case["kv_heads"], size),
                "query_offsets": _offsets(queries), "key_offsets": _offsets(keys)}
    if case["kind"] == "prefix":
        n, heads, size, cache = case["sequences"], case["kv_heads"], case["size"], case["cache"]
        # The decoder's cache order: heads, then positions; capacity to spare.
        capacity = case["own_high"] + 8
        return {"q": _normal(gen, case["type"], n, case["heads"], size, scale=1.5),
                "prefix_k": _normal(gen, cache, heads, case["prefix"], size),
                "prefix_v": _normal(gen, cache, heads, case["prefix"], size),
                "k": _normal(gen, cache, n, heads, capacity, size), "v": _normal(gen, cache, n, heads, capacity, size),
                "lengths": torch.tensor(_owned(case), dtype=torch.int32, device="cuda")}
    rows, vocab, history = case["rows"], case["vocab"], case["history"]

    def whole(low, high, *shape):
        return torch.randint(low, high, shape, generator=gen, device="cuda", dtype=torch.int32)

    def uniform(low, high, *shape):
        return torch.rand(*shape, generator=gen, device="cuda") * (high - low) + low

    v = {"logits": _normal(gen, case["type"], rows, vocab, scale=3.0)}
    if history:
        # Text repeats a few words often: three in four tokens are of a small set.
        words = whole(0, vocab, rows, max(1, history // 16))
        common = words.gather(1, whole(0, words.shape[1], rows, history).long())
        v["tokens"] = torch.where(uniform(0, 1, rows, history) < 0.75, common, whole(0, vocab, rows, history))
        v["counts"] = whole(history // 2, history + 1, rows)
        v["prompts"] = whole(0, history // 2 + 1, rows)
        v["repetition"] = uniform(1.0, 1.4, rows)
        v["presence"], v["frequency"] = uniform(0, 0.8, rows), uniform(0, 0.3, rows)
    if case["biases"]:
        v["bias_tokens"] = whole(0, vocab, rows, case["biases"])
        v["bias_values"] = uniform(-4, 8, rows, case["biases"])
    if case["masks"]:
        # Most states allow a part of the vocabulary, one allows nothing.
        words = (vocab + 31) // 32
        bits = torch.randint(0, 1 << 32, (2, case["masks"], words), generator=gen, device="cuda", dtype=torch.int64)
        both = bits[0] & bits[1]
        both[-1] = 0 if case["masks"] > 8 else both[-1]
        v["mask"] = torch.where(both >= 1 << 31, both - (1 << 32), both).to(torch.int32)
        v["states"] = whole(-1, case["masks"], rows)
    return v


def prepare(case: dict, seed: int) -> dict:
    if own:
        _backend()  # before the inputs: they are made on its stream
    v = _inputs(case, seed)
    # What the host knows of device-side lengths: bounds.
    state = {"case": case, **v}
    if case["kind"] == "packed":
        queries, keys = _lengths(case)
        state["longest"] = max(queries), max(keys)
    if own:
        _call(state)
    return state


# ---- The library's calls -----------------------------------------------------------

_shared: dict = {}


def _backend():
    """The context. torch works on the context's stream from here on: inputs are
    written before the calls that read them, outputs read after the calls that
    write them, and tensors given back to the allocator while calls still use
    them are not handed out to work ahead of those."""
    from funasrnet_amd import hip

    if "backend" not in _shared:
        _shared["backend"] = hip.HipBackend(0)
        _shared["stream"] = torch.cuda.ExternalStream(_shared["backend"].stream, device=0)
    torch.cuda.set_stream(_shared["stream"])
    return _shared["backend"], hip


def _call(state: dict) -> None:
    """The call's descriptor, output and workspace, kept as a program keeps them from step to step."""
    backend, hip = _backend()
    case = state["case"]
    types = {"f32": hip.TYPE_F32, "f16": hip.TYPE_F16, "bf16": hip.TYPE_BF16}
    if case["kind"] == "packed":
        q, k, v = state["q"], state["k"], state["v"]
        out = torch.empty_like(q)
        args = hip.PackedAttention(
            query=q.data_ptr(), key=k.data_ptr(), value=v.data_ptr(), output=out.data_ptr(),
            query_row=q.stride(0), query_head=q.stride(1), key_row=k.stride(0), key_head=k.stride(1),
            value_row=v.stride(0), value_head=v.stride(1), output_row=out.stride(0), output_head=out.stride(1),
            query_offsets=state["query_offsets"].data_ptr(), key_offsets=state["key_offsets"].data_ptr(),
            sequences=case["sequences"], query_rows=q.shape[0], key_rows=k.shape[0], longest_query=state["longest"][0],
            longest_key=state["longest"][1], heads=case["heads"], kv_heads=case["kv_heads"], head_size=case["size"],
            query_type=types[case["type"]], cache_type=types[case["cache"]], scale=case["size"] ** -0.5)
        bytes_ = backend.attention_packed_workspace(args)
    elif case["kind"] == "prefix":
        q, k, v, pk, pv = state["q"], state["k"], state["v"], state["prefix_k"], state["prefix_v"]
        out = torch.empty_like(q)
        args = hip.PrefixAttention(
            query=q.data_ptr(), prefix_key=pk.data_ptr(), prefix_value=pv.data_ptr(), key=k.data_ptr(), value=v.data_ptr(),
            output=out.data_ptr(), lengths=state["lengths"].data_ptr(), query_sequence=q.stride(0), query_head=q.stride(1),
            prefix_key_row=pk.stride(1), prefix_key_head=pk.stride(0), prefix_value_row=pv.stride(1),
            prefix_value_head=pv.stride(0), key_sequence=k.stride(0), key_row=k.stride(2), key_head=k.stride(1),
            value_sequence=v.stride(0), value_row=v.stride(2), value_head=v.stride(1), output_sequence=out.stride(0),
            output_head=out.stride(1), sequences=case["sequences"], prefix=case["prefix"], capacity=k.shape[2],
            longest=case["own_high"], heads=case["heads"], kv_heads=case["kv_heads"], head_size=case["size"],
            query_type=types[case["type"]], cache_type=types[case["cache"]], scale=case["size"] ** -0.5)
        bytes_ = backend.attention_prefix_workspace(args)
    else:
        logits = state["logits"]
        out = {"logits": torch.empty_like(logits), "tokens": torch.empty(case["rows"], dtype=torch.int32, device="cuda")}
        args = hip.LogitsAdjust(logits=logits.data_ptr(), output=out["logits"].data_ptr(), tokens=out["tokens"].data_ptr(),
                                logits_stride=logits.stride(0), output_stride=logits.stride(0), rows=case["rows"],
                                vocab=case["vocab"], type=types[case["type"]])
        if case["history"]:
            args.history, args.history_stride = state["tokens"].data_ptr(), case["history"]
            args.history_capacity, args.history_counts = case["history"], state["counts"].data_ptr()
            args.prompt_counts, args.repetition = state["prompts"].data_ptr(), state["repetition"].data_ptr()
            args.presence, args.frequency = state["presence"].data_ptr(), state["frequency"].data_ptr()
        if case["biases"]:
            args.bias_tokens, args.bias_values = state["bias_tokens"].data_ptr(), state["bias_values"].data_ptr()
            args.bias_stride = args.bias_capacity = case["biases"]
        if case["masks"]:
            args.masks, args.mask_stride = state["mask"].data_ptr(), state["mask"].stride(0)
            args.mask_rows, args.mask_index = case["masks"], state["states"].data_ptr()
        bytes_ = backend.logits_adjust_workspace(args)
    state["workspace"] = torch.empty(max(bytes_, 1), dtype=torch.uint8, device="cuda")
    args.workspace, args.workspace_bytes = state["workspace"].data_ptr(), bytes_
    state["args"], state["out"] = args, out


def _run_own(state: dict):
    backend, kind = _shared["backend"], state["case"]["kind"]
    if kind == "packed":
        backend.attention_packed_device(state["args"])
    elif kind == "prefix":
        backend.attention_prefix_device(state["args"])
    else:
        backend.logits_adjust_device(state["args"])
    return state["out"]


# ---- The plain forms ----------------------------------------------------------------


def _softmax_values(scores: torch.Tensor, values: torch.Tensor) -> torch.Tensor:
    """softmax(scores) values; 0 for rows whose every score is -inf."""
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, torch.matmul(p, values) / total, 0.0)


def _packed_plain(state: dict) -> torch.Tensor:
    case, q = state["case"], state["q"]
    n, heads, size = case["sequences"], case["kv_heads"], case["size"]
    group = case["heads"] // heads
    rows, keys = state["longest"]
    begin, key_begin = state["query_offsets"].long(), state["key_offsets"].long()
    count, key_count = begin[1:] - begin[:-1], key_begin[1:] - key_begin[:-1]
    i, j = torch.arange(rows, device="cuda"), torch.arange(keys, device="cuda")
    # Every sequence padded to the longest: [n, heads, group * rows, size] and [n, heads, keys, size].
    at = (begin[:-1, None] + i).clamp(max=q.shape[0] - 1)
    key_at = (key_begin[:-1, None] + j).clamp(max=state["k"].shape[0] - 1)
    x = q[at].float().reshape(n, rows, heads, group, size).permute(0, 2, 3, 1, 4).reshape(n, heads, group * rows, size)
    k = state["k"][key_at].float().permute(0, 2, 3, 1).contiguous()
    v = state["v"][key_at].float().permute(0, 2, 1, 3).contiguous()
    last = (i + (key_count - count)[:, None])[:, :, None]
    seen = (j <= last) & (j < key_count[:, None, None])
    scores = (torch.matmul(x, k) * size**-0.5).reshape(n, heads, group, rows, keys)
    scores = scores.masked_fill(~seen[:, None, None], -math.inf).reshape(n, heads, group * rows, keys)
    out = _softmax_values(scores, v).reshape(n, heads, group, rows, size).permute(0, 3, 1, 2, 4)
    out = out.reshape(n, rows, case["heads"], size)
    row = torch.arange(q.shape[0], device="cuda")
    sequence = (row[:, None] >= begin[1:]).sum(1)
    return out[sequence, row - begin[sequence]].to(q.dtype)


def _prefix_plain(state: dict) -> torch.Tensor:
    case = state["case"]
    n, heads, size = case["sequences"], case["kv_heads"], case["size"]
    group = case["heads"] // heads
    q = state["q"].float().reshape(n, heads, group, size)
    x = q.permute(1, 0, 2, 3).reshape(heads, n * group, size)
    shared = torch.matmul(x, state["prefix_k"].float().transpose(1, 2).contiguous()).reshape(heads, n, group, -1)
    keys = min(case["own_high"], state["k"].shape[2])
    k, v = state["k"][:, :, :keys].float(), state["v"][:, :, :keys].float()
    mine = torch.matmul(q, k.transpose(2, 3).contiguous())
    mine = mine.masked_fill((torch.arange(keys, device="cuda") >= state["lengths"][:, None])[:, None, None], -math.inf)
    scores = torch.cat([shared.permute(1, 0, 2, 3), mine], -1) * size**-0.5
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    total, prefix = p.sum(-1, keepdim=True), case["prefix"]
    first = torch.matmul(p[..., :prefix].permute(1, 0, 2, 3).reshape(heads, n * group, prefix), state["prefix_v"].float())
    out = first.reshape(heads, n, group, size).permute(1, 0, 2, 3) + torch.matmul(p[..., prefix:], v)
    return (out / total).reshape(n, case["heads"], size).to(state["q"].dtype)


def _choice_plain(state: dict) -> dict:
    case, logits = state["case"], state["logits"]
    rows, vocab = logits.shape
    x = logits.float()
    if case["history"]:
        at = torch.arange(case["history"], device="cuda")
        held = at < state["counts"][:, None]
        written = held & (at >= state["prompts"][:, None])
        tokens = state["tokens"].long()
        count = torch.zeros(rows, vocab, dtype=torch.int32, device="cuda")
        seen = count.clone().scatter_add_(1, tokens, held.int()) > 0
        count.scatter_add_(1, tokens, written.int())
        repetition = state["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
        x = x - state["frequency"][:, None] * count.float()
        x = x - torch.where(count > 0, state["presence"][:, None], 0.0)
    if case["biases"]:
        # The last entry of a token is its bias.
        at = torch.arange(case["biases"], device="cuda").expand(rows, -1)
        entry = torch.full((rows, vocab), -1, dtype=torch.int64, device="cuda")
        entry.scatter_reduce_(1, state["bias_tokens"].long(), at, "amax")
        x = torch.where(entry >= 0, x + state["bias_values"].gather(1, entry.clamp(min=0)), x)
    if case["masks"]:
        t = torch.arange(vocab, device="cuda")
        states = state["states"].long()
        words = state["mask"][states.clamp(min=0)][:, t // 32]
        x = torch.where(((words >> (t % 32)) & 1 == 1) | (states < 0)[:, None], x, -math.inf)
    out = x.to(logits.dtype)
    value = out.float()
    best = value.amax(1, keepdim=True)
    index = torch.where(value == best, torch.arange(vocab, device="cuda"), vocab).amin(1)
    return {"logits": out, "tokens": torch.where(best[:, 0] > -math.inf, index, -1).int()}


_PLAIN = {"packed": _packed_plain, "prefix": _prefix_plain, "choice": _choice_plain}


def run(state: dict):
    if own:
        return _run_own(state)
    return _PLAIN[state["case"]["kind"]](state)


# ---- What the work cannot do without ------------------------------------------------


def work(case: dict) -> dict:
    wide = {"f32": 4, "f16": 2, "bf16": 2}
    if case["kind"] == "packed":
        queries, keys = _lengths(case)
        pairs = sum(a * (b - a) + a * (a + 1) // 2 for a, b in zip(queries, keys))
        return {"bytes": float(2 * sum(queries) * case["heads"] * case["size"] * wide[case["type"]]
                               + 2 * sum(keys) * case["kv_heads"] * case["size"] * wide[case["cache"]]),
                "flops": 4.0 * pairs * case["heads"] * case["size"]}
    if case["kind"] == "prefix":
        n, owned = case["sequences"], sum(_owned(case))
        return {"bytes": float(2 * n * case["heads"] * case["size"] * wide[case["type"]]
                               + 2 * (case["prefix"] + owned) * case["kv_heads"] * case["size"] * wide[case["cache"]]),
                "flops": 4.0 * (n * case["prefix"] + owned) * case["heads"] * case["size"]}
    rows, vocab = case["rows"], case["vocab"]
    lists = 4 * rows * case["history"] + 8 * rows * case["biases"] + 4 * min(rows, case["masks"]) * ((vocab + 31) // 32)
    return {"bytes": float(2 * rows * vocab * wide[case["type"]] + lists), "flops": float(rows * vocab)}


# ---- The same in 64 bits ------------------------------------------------------------


def _attend64(q, k, v, scale: float, offset) -> torch.Tensor:
    """[rows, size] of one head's softmax(scale q k^T) v in 64 bits; row i sees keys up to i + offset (None: all)."""
    s = (q.double() @ k.double().T.contiguous()) * scale
    if offset is not None:
        at = torch.arange(s.shape[0], device="cuda")[:, None] + offset
        s = torch.where(torch.arange(s.shape[1], device="cuda") <= at, s, -math.inf)
    return torch.softmax(s, 1) @ v.double()


def exact(case: dict, seed: int):
    v = _inputs(case, seed)
    if case["kind"] == "packed":
        queries, keys = _lengths(case)
        group, out, a, b = case["heads"] // case["kv_heads"], torch.zeros(v["q"].shape, dtype=torch.float64, device="cuda"), 0, 0
        for m, n in zip(queries, keys):
            for h in range(case["heads"]):
                g = h // group
                out[a:a + m, h] = _attend64(v["q"][a:a + m, h], v["k"][b:b + n, g], v["v"][b:b + n, g], case["size"] ** -0.5, n - m)
            a, b = a + m, b + n
        return out
    if case["kind"] == "prefix":
        group, out = case["heads"] // case["kv_heads"], torch.zeros(v["q"].shape, dtype=torch.float64, device="cuda")
        for s, n in enumerate(_owned(case)):
            for g in range(case["kv_heads"]):
                k = torch.cat([v["prefix_k"][g], v["k"][s, g, :n]])
                w = torch.cat([v["prefix_v"][g], v["v"][s, g, :n]])
                heads = slice(g * group, (g + 1) * group)
                out[s, heads] = _attend64(v["q"][s, heads], k, w, case["size"] ** -0.5, None)
        return out
    rows = []
    for r in range(case["rows"]):
        x = v["logits"][r].double()
        if case["history"]:
            count = int(v["counts"][r])
            tokens, first = v["tokens"][r, :count].long(), min(int(v["prompts"][r]), count)
            seen = torch.zeros(case["vocab"], dtype=torch.bool, device="cuda")
            seen[tokens] = True
            times = torch.bincount(tokens[first:], minlength=case["vocab"]).double()
            factor = v["repetition"][r].double()
            x = torch.where(seen, torch.where(x > 0, x / factor, x * factor), x)
            x = x - v["frequency"][r].double() * times - v["presence"][r].double() * (times > 0)
        if case["biases"]:
            last = dict(zip(v["bias_tokens"][r].tolist(), v["bias_values"][r].double().tolist()))
            x[torch.tensor(list(last), device="cuda")] += torch.tensor(list(last.values()), dtype=torch.float64, device="cuda")
        if case["masks"] and int(v["states"][r]) >= 0:
            words = v["mask"][int(v["states"][r])].long() & 0xFFFFFFFF
            bits = (words[:, None] >> torch.arange(32, device="cuda")) & 1
            x = torch.where(bits.reshape(-1)[:case["vocab"]] == 1, x, -math.inf)
        rows.append(x)
    return {"logits": torch.stack(rows), "tokens": None}
