"""The serving operators on the device against their definitions in 64 bits:
packed causal prompts, single tokens behind a shared prefix, and the choice of a
token, at the sizes and masks where they can go wrong."""
import numpy as np
import pytest

from serving_cases import CODES, adjusted, attend, attention_bound, load, store

pytestmark = pytest.mark.gpu

TYPES = [("f32", "f16"), ("f16", "f16"), ("bf16", "bf16")]


@pytest.fixture(scope="module")
def backend():
    from funasrnet_amd.hip import HipBackend
    b = HipBackend(0)
    yield b
    b.close()


def to_device(a):
    from funasrnet_amd.device import DeviceArray
    return DeviceArray.from_numpy(a)


def workspace_of(bytes_, extra=0):
    """A workspace that holds NaN patterns."""
    return to_device(np.full(max(bytes_, 16) + extra, 0xFF, np.uint8))


# ---- Packed prompts -----------------------------------------------------------------


def packed_inputs(seed, queries, keys, heads, kv_heads, size, types):
    rng = np.random.default_rng(seed)
    q = store(rng.standard_normal((sum(queries), heads, size)) * 1.5, types[0])
    k = store(rng.standard_normal((sum(keys), kv_heads, size)), types[1])
    v = store(rng.standard_normal((sum(keys), kv_heads, size)), types[1])
    return q, k, v


def offsets(lengths, before=0):
    return np.concatenate([[before], before + np.cumsum(lengths)]).astype(np.int32)


def run_packed(backend, q, k, v, query_offsets, key_offsets, types, scale=None, pad=0, keep=None):
    """The output rows, from buffers whose rows are `pad` elements longer than needed."""
    from funasrnet_amd import hip
    (rows, heads, size), (key_rows, kv_heads, _) = q.shape, k.shape

    def spaced(a):
        wide = np.full((a.shape[0], a.shape[1] * size + pad), 77, a.dtype)
        wide[:, :a.shape[1] * size] = a.reshape(a.shape[0], -1)
        return wide

    dq, dk, dv = to_device(spaced(q)), to_device(spaced(k)), to_device(spaced(v))
    start = np.full((rows, heads * size + pad), 55, q.dtype) if keep is None else keep
    out = to_device(start)
    dqo, dko = to_device(query_offsets), None if key_offsets is None else to_device(key_offsets)
    ko = query_offsets if key_offsets is None else key_offsets
    call = hip.PackedAttention(
        query=dq.ptr, key=dk.ptr, value=dv.ptr, output=out.ptr, query_row=heads * size + pad, query_head=size,
        key_row=kv_heads * size + pad, key_head=size, value_row=kv_heads * size + pad, value_head=size,
        output_row=heads * size + pad, output_head=size, query_offsets=dqo.ptr, key_offsets=dko.ptr if dko else None,
        sequences=len(query_offsets) - 1, query_rows=rows, key_rows=key_rows,
        longest_query=int(np.diff(query_offsets).max(initial=0)), longest_key=int(np.diff(ko).max(initial=0)), heads=heads,
        kv_heads=kv_heads, head_size=size, query_type=CODES[types[0]], cache_type=CODES[types[1]], scale=scale or size**-0.5)
    need = backend.attention_packed_workspace(call)
    ws = workspace_of(need, 64)
    call.workspace, call.workspace_bytes = ws.ptr, need
    assert backend.attention_packed_device(call) == hip.OK
    backend.synchronize()
    assert np.all(ws.numpy()[max(need, 16):] == 0xFF)
    got = out.numpy()
    assert pad == 0 or np.array_equal(got[:, heads * size:], start[:, heads * size:])
    return got[:, :heads * size].reshape(rows, heads, size)


def check_packed(got, q, k, v, query_offsets, key_offsets, types, scale=None):
    heads, kv_heads, size = q.shape[1], k.shape[1], q.shape[2]
    fq, fk, fv, fg = load(q, types[0]), load(k, types[1]), load(v, types[1]), load(got, types[0])
    ko = query_offsets if key_offsets is None else key_offsets
    for s in range(len(query_offsets) - 1):
        (a, b), (c, d) = query_offsets[s:s + 2], ko[s:s + 2]
        seen = np.arange(d - c)[None, :] <= np.arange(b - a)[:, None] + (d - c) - (b - a)
        for h in range(heads):
            g = h // (heads // kv_heads)
            out, weight, dots = attend(fq[a:b, h], fk[c:d, g], fv[c:d, g], scale or size**-0.5, seen)
            off = np.abs(fg[a:b, h] - out)
            limit = attention_bound(out, weight, dots, max(d - c, 1), size, types[0])
            assert np.all(off <= limit), (s, h, float((off / limit).max()))


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("queries,extra,heads,kv_heads,size", [
    ([1], [0], 2, 1, 128),                                   # one token, one key
    ([37], [0], 4, 2, 128),
    ([64, 1, 0, 65], [0, 0, 0, 0], 4, 4, 128),               # an empty sequence
    ([33, 128, 5], [0, 0, 0], 8, 2, 64),
    ([3, 1, 0, 70], [100, 33, 9, 250], 6, 2, 96),            # resumed, three heads a K/V head
    ([1, 1, 1], [1000, 0, 511], 16, 2, 128),                 # single tokens over long caches
    ([17, 9], [-5, -9], 5, 1, 128),                          # queries that see nothing
    ([40], [0], 3, 3, 8),
    ([29], [3], 2, 1, 120),
    ([300], [13], 2, 2, 128),
    ([2, 5, 130], [1, 0, 700], 40, 8, 72),
], ids=str)
def test_packed(backend, types, queries, extra, heads, kv_heads, size):
    keys = [a + b for a, b in zip(queries, extra)]
    q, k, v = packed_inputs(sum(queries) + size, queries, keys, heads, kv_heads, size, types)
    qo, ko = offsets(queries), offsets(keys)
    print(f"packed {queries} {extra} {heads}/{kv_heads} x {size} {types}", flush=True)
    got = run_packed(backend, q, k, v, qo, None if not any(extra) else ko, types, pad=24)
    check_packed(got, q, k, v, qo, ko, types)


# ---- A shared prefix ----------------------------------------------------------------


def run_prefix(backend, q, pk, pv, k, v, lengths, types, scale=None, heads_first=True):
    """pk, pv [prefix][kv_heads][size], k, v [sequences][capacity][kv_heads][size]; laid out
    with heads before positions (the decoder's cache) or as they are."""
    from funasrnet_amd import hip
    n, heads, size = q.shape
    prefix, kv_heads = pk.shape[:2]
    capacity = k.shape[1]
    if heads_first:
        dpk, dpv = (to_device(np.swapaxes(a, 0, 1)) for a in (pk, pv))
        dk, dv = (to_device(np.swapaxes(a, 1, 2)) for a in (k, v))
        strides = dict(row=size, prefix_head=prefix * size, head=capacity * size)
    else:
        dpk, dpv, dk, dv = (to_device(a) for a in (pk, pv, k, v))
        strides = dict(row=kv_heads * size, prefix_head=size, head=size)
    dq, out, dl = to_device(q), to_device(np.full_like(q, 55)), to_device(np.asarray(lengths, np.int32))
    own = max(capacity * kv_heads * size, 0)
    call = hip.PrefixAttention(
        query=dq.ptr, prefix_key=dpk.ptr, prefix_value=dpv.ptr, key=dk.ptr, value=dv.ptr, output=out.ptr, lengths=dl.ptr,
        query_sequence=heads * size, query_head=size, prefix_key_row=strides["row"], prefix_key_head=strides["prefix_head"],
        prefix_value_row=strides["row"], prefix_value_head=strides["prefix_head"], key_sequence=own, key_row=strides["row"],
        key_head=strides["head"], value_sequence=own, value_row=strides["row"], value_head=strides["head"],
        output_sequence=heads * size, output_head=size, sequences=n, prefix=prefix, capacity=capacity,
        longest=int(min(max(max(lengths), 0), capacity)), heads=heads, kv_heads=kv_heads, head_size=size,
        query_type=CODES[types[0]], cache_type=CODES[types[1]], scale=scale or size**-0.5)
    need = backend.attention_prefix_workspace(call)
    ws = workspace_of(need, 64)
    call.workspace, call.workspace_bytes = ws.ptr, need
    assert backend.attention_prefix_device(call) == hip.OK
    backend.synchronize()
    assert np.all(ws.numpy()[max(need, 16):] == 0xFF)
    return out.numpy()


def prefix_inputs(seed, n, prefix, capacity, heads, kv_heads, size, types):
    rng = np.random.default_rng(seed)
    q = store(rng.standard_normal((n, heads, size)) * 1.5, types[0])
    pk, pv = (store(rng.standard_normal((prefix, kv_heads, size)), types[1]) for _ in range(2))
    k, v = (store(rng.standard_normal((n, capacity, kv_heads, size)), types[1]) for _ in range(2))
    return q, pk, pv, k, v


def check_prefix(got, q, pk, pv, k, v, lengths, types, scale=None):
    n, heads, size = q.shape
    kv_heads, capacity = pk.shape[1], k.shape[1]
    fq, fg = load(q, types[0]), load(got, types[0])
    fpk, fpv, fk, fv = (load(a, types[1]) for a in (pk, pv, k, v))
    for s in range(n):
        own = min(max(int(lengths[s]), 0), capacity)
        for g in range(kv_heads):
            keys = np.concatenate([fpk[:, g], fk[s, :own, g]])
            values = np.concatenate([fpv[:, g], fv[s, :own, g]])
            hs = slice(g * (heads // kv_heads), (g + 1) * (heads // kv_heads))
            seen = np.ones((heads // kv_heads, len(keys)), bool)
            out, weight, dots = attend(fq[s, hs], keys, values, scale or size**-0.5, seen)
            off = np.abs(fg[s, hs] - out)
            limit = attention_bound(out, weight, dots, max(len(keys), 1), size, types[0])
            assert np.all(off <= limit), (s, g, float((off / limit).max()))


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("lengths,prefix,capacity,heads,kv_heads,size", [
    ([1], 1, 1, 2, 1, 128),
    ([0], 0, 4, 2, 1, 128),                                  # nothing to see
    ([0, 5, -3, 900], 0, 20, 4, 2, 128),                     # no prefix; lengths beyond both ends
    ([0, 1, 33, 64, 65], 100, 70, 16, 8, 128),
    ([7, 200], 1000, 200, 4, 1, 64),
    ([50] * 17, 129, 50, 6, 2, 96),
    ([3], 5000, 10, 8, 1, 128),
    ([700, 1], 63, 701, 10, 2, 120),
    (list(range(70)), 65, 70, 2, 2, 8),
], ids=str)
def test_prefix(backend, types, lengths, prefix, capacity, heads, kv_heads, size):
    arrays = prefix_inputs(prefix + size, len(lengths), prefix, capacity, heads, kv_heads, size, types)
    print(f"prefix {lengths[:4]} {prefix} {capacity} {heads}/{kv_heads} x {size} {types}", flush=True)
    for heads_first in (True, False):
        got = run_prefix(backend, *arrays, lengths, types, heads_first=heads_first)
        check_prefix(got, *arrays, lengths, types)


# ---- The choice of a token ------------------------------------------------------------


def choice_inputs(seed, rows, vocab, history, biases, masks, kind):
    rng = np.random.default_rng(seed)
    v = {"logits": store(rng.standard_normal((rows, vocab)) * 3, kind)}
    if history:
        words = rng.integers(0, vocab, max(1, history // 8))
        lists = np.where(rng.random((rows, history)) < 0.7, rng.choice(words, (rows, history)),
                         rng.integers(-1, vocab + 2, (rows, history)))
        v["history"] = lists.astype(np.int32)
        v["counts"] = rng.integers(0, history + 1, rows).astype(np.int32)
        v["prompts"] = rng.integers(0, history + 1, rows).astype(np.int32)
        v["repetition"] = rng.uniform(0.8, 1.5, rows).astype(np.float32)
        v["presence"] = rng.uniform(-0.5, 1, rows).astype(np.float32)
        v["frequency"] = rng.uniform(0, 0.5, rows).astype(np.float32)
    if biases:
        # Few tokens, so that entries repeat; some outside the vocabulary.
        v["bias_tokens"] = rng.choice(np.concatenate([rng.integers(0, vocab, biases), [-1, vocab]]), (rows, biases)).astype(np.int32)
        v["bias_values"] = rng.uniform(-4, 8, (rows, biases)).astype(np.float32)
        v["bias_counts"] = rng.integers(0, biases + 1, rows).astype(np.int32)
    if masks:
        v["masks"] = rng.integers(0, 1 << 32, (masks, (vocab + 31) // 32), dtype=np.uint64).astype(np.uint32)
        v["masks"][-1] = 0  # allows nothing
        v["index"] = rng.integers(-1, masks + 1, rows).astype(np.int32)
    return v


def run_choice(backend, v, kind, pad=0, in_place=False, tokens=True):
    from funasrnet_amd import hip
    rows, vocab = v["logits"].shape
    wide = np.full((rows, vocab + pad), 9, v["logits"].dtype)
    wide[:, :vocab] = v["logits"]
    logits = to_device(wide)
    out = logits if in_place else to_device(np.full_like(wide, 7))
    chosen = to_device(np.full(rows + 1, -5, np.int32))
    held = {n: to_device(a) for n, a in v.items() if n != "logits"}
    call = hip.LogitsAdjust(logits=logits.ptr, output=out.ptr, tokens=chosen.ptr if tokens else None,
                            logits_stride=vocab + pad, output_stride=vocab + pad, rows=rows, vocab=vocab, type=CODES[kind])
    if "history" in v:
        call.history, call.history_stride = held["history"].ptr, v["history"].shape[1]
        call.history_capacity = v["history"].shape[1]
        call.history_counts, call.prompt_counts = held["counts"].ptr, held["prompts"].ptr
        call.repetition, call.presence, call.frequency = (held[n].ptr for n in ("repetition", "presence", "frequency"))
    if "bias_tokens" in v:
        call.bias_tokens, call.bias_values = held["bias_tokens"].ptr, held["bias_values"].ptr
        call.bias_stride = call.bias_capacity = v["bias_tokens"].shape[1]
        call.bias_counts = held["bias_counts"].ptr
    if "masks" in v:
        call.masks, call.mask_stride, call.mask_rows = held["masks"].ptr, v["masks"].shape[1], v["masks"].shape[0]
        call.mask_index = held["index"].ptr
    need = backend.logits_adjust_workspace(call)
    ws = workspace_of(need, 64)
    call.workspace, call.workspace_bytes = ws.ptr, need
    assert backend.logits_adjust_device(call) == hip.OK
    backend.synchronize()
    assert np.all(ws.numpy()[max(need, 16):] == 0xFF)
    got, picked = out.numpy(), chosen.numpy()
    assert np.array_equal(got[:, vocab:], (wide if in_place else np.full_like(wide, 7))[:, vocab:])
    assert picked[rows] == -5 and (tokens or np.all(picked == -5))
    return got[:, :vocab], picked[:rows]


def check_choice(got, picked, v, kind):
    rows, vocab = v["logits"].shape
    for r in range(rows):
        history, prompt, factors, bias, mask = [], 0, (1, 0, 0), [], None
        if "history" in v:
            history, prompt = v["history"][r, :v["counts"][r]].tolist(), int(v["prompts"][r])
            factors = v["repetition"][r], v["presence"][r], v["frequency"][r]
        if "bias_tokens" in v:
            n = v["bias_counts"][r]
            bias = list(zip(v["bias_tokens"][r, :n].tolist(), v["bias_values"][r, :n]))
        if "masks" in v and 0 <= v["index"][r] < len(v["masks"]):
            mask = np.unpackbits(v["masks"][v["index"][r]].view(np.uint8), bitorder="little")[:vocab] == 1
        expected, token = adjusted(load(v["logits"][r], kind), history, prompt, *factors, bias, mask, kind)
        # fp32 steps in a fixed order: the same bits.
        assert np.array_equal(got[r].view(np.uint8), expected.view(np.uint8)), r
        assert picked is None or picked[r] == token, (r, picked[r], token)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,vocab,history,biases,masks,pad", [
    (1, 1, 1, 1, 0, 0), (1, 1023, 0, 0, 0, 0), (3, 1025, 10, 0, 0, 3), (2, 4096, 0, 5, 0, 0), (5, 2049, 0, 0, 4, 1),
    (4, 5003, 700, 40, 3, 2), (1, 151936, 300, 40, 0, 0), (17, 151936, 50, 9, 5, 0), (9, 8191, 64, 3, 2, 1), (1, 40, 5000, 600, 1, 0),
], ids=str)
def test_choice(backend, kind, rows, vocab, history, biases, masks, pad):
    print(f"choice {rows} x {vocab} {history} {biases} {masks} {pad} {kind}", flush=True)
    v = choice_inputs(rows * 7 + vocab, rows, vocab, history, biases, masks, kind)
    got, picked = run_choice(backend, v, kind, pad)
    check_choice(got, picked, v, kind)
    again, same = run_choice(backend, v, kind, pad, in_place=True)
    assert np.array_equal(got.view(np.uint8), again.view(np.uint8)) and np.array_equal(picked, same)
    alone, _ = run_choice(backend, v, kind, pad, tokens=False)
    assert np.array_equal(got.view(np.uint8), alone.view(np.uint8))
