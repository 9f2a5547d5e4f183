"""The serving operators on the device against their definitions in 64 bits:
packed causal prompts, single tokens behind a shared prefix, and the choice of a
token, at the sizes and masks where they can go wrong."""
import numpy as np
import pytest

from serving_cases import CODES, adjusted, attend, attend_all, attention_bound, load, store

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


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("queries,extra,heads,kv_heads,size", [
    ([1100], [0], 64, 64, 128),             # 128 rows a workgroup
    ([700, 3, 450], [0, 0, 0], 64, 64, 64),
    ([400], [2500], 64, 64, 128),           # and the keys in shares
    ([390], [2110], 64, 32, 96),
    ([60, 45], [1500, 3000], 8, 4, 128),    # 64 rows, shares
    ([1, 1, 1], [4000, 1200, 2600], 8, 8, 128),
    ([7], [9000], 4, 1, 64),
], ids=str)
def test_packed_large(backend, types, queries, extra, heads, kv_heads, size):
    keys = [a + b for a, b in zip(queries, extra)]
    q, k, v = packed_inputs(sum(keys), queries, keys, heads, kv_heads, size, types)
    qo, ko = offsets(queries), offsets(keys)
    print(f"packed {queries} {extra} {heads}/{kv_heads} x {size} {types}", flush=True)
    got = run_packed(backend, q, k, v, qo, ko, types)
    fq, fk, fv, fg = load(q, types[0]), load(k, types[1]), load(v, types[1]), load(got, types[0])
    for s in range(len(queries)):
        (a, b), (c, d) = qo[s:s + 2], ko[s:s + 2]
        for h in sorted({0, 1, heads // 2, heads - 1}):
            g = h // (heads // kv_heads)
            out, weight, dots = attend_all(fq[a:b, h], fk[c:d, g], fv[c:d, g], size**-0.5, extra[s])
            off = np.abs(fg[a:b, h] - out)
            limit = attention_bound(out, weight, dots, d - c, size, types[0])
            assert np.all(off <= limit), (s, h, float((off / limit).max()))


@pytest.mark.parametrize("count", [63, 64, 65, 300, 4200])
def test_packed_many_sequences(backend, count):
    """The search for a tile's sequence, with empty ones among them."""
    rng = np.random.default_rng(count)
    queries = rng.integers(0, 6, count).tolist()
    keys = [a + int(b) for a, b in zip(queries, rng.integers(0, 3, count))]
    types = ("f16", "f16")
    q, k, v = packed_inputs(count, queries, keys, 2, 1, 64, types)
    qo, ko = offsets(queries), offsets(keys)
    got = run_packed(backend, q, k, v, qo, ko, types)
    check_packed(got, q, k, v, qo, ko, types)


def test_packed_rows_of_no_sequence_are_left(backend):
    types = ("f32", "f16")
    queries, keys = [20, 0, 33], [25, 4, 33]
    q, k, v = packed_inputs(5, [70], [90], 4, 2, 128, types)
    qo, ko = offsets(queries, 9), offsets(keys, 3)
    keep = np.random.default_rng(1).standard_normal((70, 4 * 128)).astype(np.float32)
    got = run_packed(backend, q, k, v, qo, ko, types, keep=keep)
    check_packed(got, q, k, v, qo, ko, types)
    kept = keep.reshape(70, 4, 128)
    assert np.array_equal(got[:9], kept[:9]) and np.array_equal(got[9 + 53:], kept[9 + 53:])


def test_packed_offsets_outside_the_rows(backend):
    """Taken as the nearer end."""
    types = ("f16", "f16")
    q, k, v = packed_inputs(6, [50], [60], 2, 2, 64, types)
    got = run_packed(backend, q, k, v, np.array([-7, 30, 1000], np.int32), np.array([-100, 40, 2**31 - 1], np.int32), types)
    check_packed(got, q, k, v, np.array([0, 30, 50]), np.array([0, 40, 60]), types)


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("rows,heads,kv_heads,extra", [(90, 2, 1, 0), (1100, 64, 64, 0), (400, 64, 64, 2500), (3, 4, 1, 700)])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_packed_masked_places_may_hold_anything(backend, types, rows, heads, kv_heads, extra, bad):
    """A late key and value only reach the rows that see them."""
    keys = rows + extra
    q, k, v = packed_inputs(rows, [rows], [keys], heads, kv_heads, 128, types)
    at = keys - 2  # seen by the last two rows
    plain = run_packed(backend, q, k, v, offsets([rows]), offsets([keys]), types)
    spoilt_k, spoilt_v = k.copy(), v.copy()
    spoilt_k[at] = store(np.full(spoilt_k[at].shape, bad), types[1])
    spoilt_v[at] = store(np.full(spoilt_v[at].shape, bad), types[1])
    got = load(run_packed(backend, q, spoilt_k, spoilt_v, offsets([rows]), offsets([keys]), types), types[0])
    plain = load(plain, types[0])
    # Rows before it: as without it, but for the order in which a row is summed.
    limit = 2 * attention_bound(plain, np.abs(plain) + 4.0, 60.0, keys, 128, types[0])
    assert np.all(np.isfinite(got[:rows - 2])) and np.all(np.abs(got[:rows - 2] - plain[:rows - 2]) <= limit[:rows - 2])
    if bad != -np.inf:
        assert not np.any(np.isfinite(got[rows - 2:]))


def test_packed_row_of_minus_infinity_scores(backend):
    types = ("f16", "f16")
    q, k, v = packed_inputs(8, [40], [40], 2, 2, 64, types)
    q[:] = store(np.abs(load(q, "f16")) + 0.1, "f16")
    k[:3] = store(np.full((3, 2, 64), -np.inf), "f16")  # rows 0 to 2 only see these
    got = load(run_packed(backend, q, k, v, offsets([40]), None, types), "f16")
    assert np.all(got[:3] == 0)
    fq, fk, fv = load(q, "f16"), load(k, "f16"), load(v, "f16")
    for h in range(2):
        out, weight, dots = attend_all(fq[3:, h], fk[3:, h], fv[3:, h], 64**-0.5, 0)
        assert np.all(np.abs(got[3:, h] - out) <= attention_bound(out, weight, dots, 37, 64, "f16"))


@pytest.mark.parametrize("rows,heads,kv_heads", [(40, 2, 2), (300, 16, 1)])
@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
def test_packed_infinite_queries(backend, types, rows, heads, kv_heads):
    """-infinity against keys above 0: every score is -infinity, the row zeros; other rows as ever."""
    q, k, v = packed_inputs(10, [rows], [rows], heads, kv_heads, 128, types)
    k[:, :, 5] = store(np.abs(load(k[:, :, 5], types[1])) + 0.125, types[1])
    plain = load(run_packed(backend, q, k, v, offsets([rows]), None, types), types[0])
    q[3::7, :, 5] = store(np.full(q[3::7, :, 5].shape, -np.inf), types[0])
    q[5::7, :, 5] = store(np.full(q[5::7, :, 5].shape, np.inf), types[0])  # infinity - infinity
    got = load(run_packed(backend, q, k, v, offsets([rows]), None, types), types[0])
    assert np.all(got[3::7] == 0)
    assert np.all(np.isnan(got[5::7]))
    others = np.isin(np.arange(rows) % 7, [3, 5], invert=True)
    assert np.array_equal(got[others], plain[others])


@pytest.mark.parametrize("magnitude", [1e-30, 1e-6, 1e4, 1e30])
def test_packed_fp32_queries_of_any_size(backend, magnitude):
    types = ("f32", "f16")
    q, k, v = packed_inputs(9, [70], [70], 4, 2, 128, types)
    q *= np.float32(magnitude)
    scale = float(np.float32(128**-0.5 / magnitude))
    got = run_packed(backend, q, k, v, offsets([70]), None, types, scale=scale)
    check_packed(got, q, k, v, offsets([70]), None, types, scale=scale)


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
def test_packed_sharp_and_rising_scores(backend, types):
    """Weights that differ by far, largest scores that keep rising."""
    q, k, v = packed_inputs(10, [200], [200], 2, 1, 64, types)
    k[:] = store(load(k, types[1]) * np.linspace(0.01, 12, 200)[:, None, None], types[1])
    got = run_packed(backend, q, k, v, offsets([200]), None, types)
    check_packed(got, q, k, v, offsets([200]), None, types)


def test_packed_broadcast_and_cache_order(backend):
    """One K/V head's rows for all (stride 0), and a cache with heads before rows."""
    from funasrnet_amd import hip
    types, heads, rows = ("f32", "f16"), 4, 45
    q, k, v = packed_inputs(11, [rows], [rows], heads, 2, 128, types)
    for shared in (True, False):
        kk = np.repeat(k[:, :1], 2, 1) if shared else k
        vv = np.repeat(v[:, :1], 2, 1) if shared else v
        dk, dv = ((to_device(k[:, 0]), to_device(v[:, 0])) if shared else
                  (to_device(np.swapaxes(k, 0, 1)), to_device(np.swapaxes(v, 0, 1))))
        dq, out, do = to_device(q), to_device(np.zeros_like(q)), to_device(offsets([rows]))
        head = 0 if shared else rows * 128
        call = hip.PackedAttention(query=dq.ptr, key=dk.ptr, value=dv.ptr, output=out.ptr, query_row=heads * 128, query_head=128,
                                   key_row=128, key_head=head, value_row=128, value_head=head, output_row=heads * 128,
                                   output_head=128, query_offsets=do.ptr, sequences=1, query_rows=rows, key_rows=rows,
                                   longest_query=rows, longest_key=rows, heads=heads, kv_heads=2, head_size=128,
                                   query_type=hip.TYPE_F32, cache_type=hip.TYPE_F16, scale=128**-0.5)
        assert backend.attention_packed_device(call) == hip.OK
        backend.synchronize()
        check_packed(out.numpy(), q, kk, vv, offsets([rows]), None, types)


def test_packed_hints_only_steer(backend):
    """Lengths beyond the hints are attended all the same."""
    from funasrnet_amd import hip
    types = ("bf16", "bf16")
    q, k, v = packed_inputs(12, [300, 10], [1500, 1700], 4, 2, 128, types)
    results = []
    for longest in ((0, 0), (1, 1), (300, 1700), (100000, 100000)):
        dq, dk, dv, out = to_device(q), to_device(k), to_device(v), to_device(np.zeros_like(q))
        qo, ko = to_device(offsets([300, 10])), to_device(offsets([1500, 1700]))
        call = hip.PackedAttention(query=dq.ptr, key=dk.ptr, value=dv.ptr, output=out.ptr, query_row=512, query_head=128,
                                   key_row=256, key_head=128, value_row=256, value_head=128, output_row=512, output_head=128,
                                   query_offsets=qo.ptr, key_offsets=ko.ptr, sequences=2, query_rows=310, key_rows=3200,
                                   longest_query=longest[0], longest_key=longest[1], heads=4, kv_heads=2, head_size=128,
                                   query_type=hip.TYPE_BF16, cache_type=hip.TYPE_BF16, scale=128**-0.5)
        need = backend.attention_packed_workspace(call)
        ws = workspace_of(need)
        call.workspace, call.workspace_bytes = ws.ptr, need
        assert backend.attention_packed_device(call) == hip.OK
        backend.synchronize()
        results.append(out.numpy())
        check_packed(results[-1], q, k, v, offsets([300, 10]), offsets([1500, 1700]), types)


def test_offsets_past_32_bits(backend):
    """Keys and values more than 2^32 elements into their buffers."""
    import ctypes
    from funasrnet_amd import device, hip
    rows, step = 40, (1 << 32) // 8 // 128 * 128  # 9 sequences, each half a Gi elements on
    types = ("f16", "f16")
    n = 9
    arrays = prefix_inputs(13, n, 33, rows, 4, 2, 128, types)
    q, pk, pv, k, v = arrays
    big = [ctypes.c_void_p() for _ in range(2)]
    run = device.runtime()
    lengths = np.full(n, rows, np.int32)
    try:
        for p, a in zip(big, (k, v)):
            assert run.hipMalloc(ctypes.byref(p), (step * n) * 2) == 0
            for s in range(n):
                block = np.ascontiguousarray(a[s])
                assert run.hipMemcpy(p.value + s * step * 2, block.ctypes.data, block.nbytes, device.H2D) == 0
        dq, dpk, dpv, dl, out = to_device(q), to_device(pk), to_device(pv), to_device(lengths), to_device(np.zeros_like(q))
        call = hip.PrefixAttention(
            query=dq.ptr, prefix_key=dpk.ptr, prefix_value=dpv.ptr, key=big[0].value, value=big[1].value, output=out.ptr,
            lengths=dl.ptr, query_sequence=512, query_head=128, prefix_key_row=256, prefix_key_head=128, prefix_value_row=256,
            prefix_value_head=128, key_sequence=step, key_row=256, key_head=128, value_sequence=step, value_row=256,
            value_head=128, output_sequence=512, output_head=128, sequences=n, prefix=33, capacity=rows, longest=rows, heads=4,
            kv_heads=2, head_size=128, query_type=hip.TYPE_F16, cache_type=hip.TYPE_F16, scale=128**-0.5)
        need = backend.attention_prefix_workspace(call)
        ws = workspace_of(need)
        call.workspace, call.workspace_bytes = ws.ptr, need
        assert backend.attention_prefix_device(call) == hip.OK
        backend.synchronize()
        check_prefix(out.numpy(), *arrays, lengths, types)
        # The last sequence's rows as a packed prompt whose rows are 2^24 elements apart.
        far = 1 << 24
        for p, a in zip(big, (k, v)):
            for r in range(rows):
                block = np.ascontiguousarray(a[n - 1, r])
                assert run.hipMemcpy(p.value + r * far * 2, block.ctypes.data, block.nbytes, device.H2D) == 0
        qq = np.ascontiguousarray(np.resize(q, (rows, 4, 128)))
        dq, out, do = to_device(qq), to_device(np.zeros_like(qq)), to_device(offsets([rows]))
        call = hip.PackedAttention(query=dq.ptr, key=big[0].value, value=big[1].value, output=out.ptr, query_row=512,
                                   query_head=128, key_row=far, key_head=128, value_row=far, value_head=128, output_row=512,
                                   output_head=128, query_offsets=do.ptr, sequences=1, query_rows=rows, key_rows=rows,
                                   longest_query=rows, longest_key=rows, heads=4, kv_heads=2, head_size=128,
                                   query_type=hip.TYPE_F16, cache_type=hip.TYPE_F16, scale=128**-0.5)
        assert backend.attention_packed_device(call) == hip.OK
        backend.synchronize()
        check_packed(out.numpy(), qq, k[n - 1], v[n - 1], offsets([rows]), None, types)
    finally:
        for p in big:
            if p.value:
                run.hipFree(p.value)


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


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("count,prefix,longest,heads,kv_heads,size", [
    (300, 700, 90, 16, 8, 64),       # 64 rows of the prefix a workgroup
    (1100, 130, 5, 64, 8, 8),        # 128
    (40, 1500, 900, 8, 4, 128),      # own rows in one share
    (2, 4000, 3000, 4, 2, 128),      # and in several
    (70, 65, 40, 40, 1, 128),        # more heads a group than a tile has rows
], ids=str)
def test_prefix_large(backend, types, count, prefix, longest, heads, kv_heads, size):
    rng = np.random.default_rng(count)
    lengths = rng.integers(0, longest + 1, count)
    arrays = prefix_inputs(count, count, prefix, longest, heads, kv_heads, size, types)
    print(f"prefix {count} {prefix} {longest} {heads}/{kv_heads} x {size} {types}", flush=True)
    got = run_prefix(backend, *arrays, lengths, types)
    some = np.unique(np.concatenate([rng.integers(0, count, 25), [0, count - 1]]))
    check_prefix(got[some], arrays[0][some], *arrays[1:3], arrays[3][some], arrays[4][some], lengths[some], types)


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("count,heads,kv_heads,size", [(300, 4, 2, 128), (1100, 64, 2, 128), (300, 4, 4, 96)], ids=str)
def test_prefix_capacities_past_the_caches(backend, types, count, heads, kv_heads, size):
    """Own rows that count as more than the caches hold; the sequences' cache rows overlap, 16 apart."""
    from funasrnet_amd import hip
    rng = np.random.default_rng(count + size)
    capacity, step, prefix = 4096, 16, 100
    rows = capacity + step * count
    q = store(rng.standard_normal((count, heads, size)) * 1.5, types[0])
    pk, pv = (store(rng.standard_normal((prefix, kv_heads, size)), types[1]) for _ in range(2))
    k, v = (store(rng.standard_normal((rows, kv_heads, size)), types[1]) for _ in range(2))
    lengths = np.where(rng.random(count) < 0.02, capacity, rng.integers(0, 200, count)).astype(np.int32)
    dq, dpk, dpv, dk, dv, dl = (to_device(x) for x in (q, pk, pv, k, v, lengths))
    out = to_device(np.full_like(q, 55))
    line = kv_heads * size
    call = hip.PrefixAttention(
        query=dq.ptr, prefix_key=dpk.ptr, prefix_value=dpv.ptr, key=dk.ptr, value=dv.ptr, output=out.ptr, lengths=dl.ptr,
        query_sequence=heads * size, query_head=size, prefix_key_row=line, prefix_key_head=size, prefix_value_row=line,
        prefix_value_head=size, key_sequence=step * line, key_row=line, key_head=size, value_sequence=step * line,
        value_row=line, value_head=size, output_sequence=heads * size, output_head=size, sequences=count, prefix=prefix,
        capacity=capacity, longest=capacity, heads=heads, kv_heads=kv_heads, head_size=size, query_type=CODES[types[0]],
        cache_type=CODES[types[1]], scale=size**-0.5)
    need = backend.attention_prefix_workspace(call)
    ws = workspace_of(need)
    call.workspace, call.workspace_bytes = ws.ptr, need
    assert backend.attention_prefix_device(call) == hip.OK
    backend.synchronize()
    some = np.unique(np.concatenate([rng.integers(0, count, 12), np.flatnonzero(lengths == capacity)[:2], [0, count - 1]]))
    own_k, own_v = (np.stack([a[step * i:step * i + capacity] for i in some]) for a in (k, v))
    check_prefix(out.numpy()[some], q[some], pk, pv, own_k, own_v, lengths[some], types)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_prefix_rows_behind_the_length_may_hold_anything(backend, bad):
    types = ("f32", "f16")
    lengths = [0, 1, 31, 32, 33, 100]
    for prefix in (0, 50, 1500):
        q, pk, pv, k, v = prefix_inputs(prefix + 3, len(lengths), prefix, 128, 4, 2, 128, types)
        for s, n in enumerate(lengths):
            k[s, n:] = bad
            v[s, n:] = bad
        got = run_prefix(backend, q, pk, pv, k, v, lengths, types)
        check_prefix(got, q, pk, pv, k, v, lengths, types)


@pytest.mark.parametrize("prefix", [300, 2000])
def test_prefix_value_that_is_infinite(backend, prefix):
    """An infinite value reaches every row, a NaN of one sequence that one alone."""
    types = ("bf16", "bf16")
    q, pk, pv, k, v = prefix_inputs(4, 5, prefix, 64, 4, 2, 64, types)
    lengths = [64, 3, 50, 0, 20]
    v[2, 7, 1] = store(np.full(64, np.nan), "bf16")
    pv[11, 0] = store(np.full(64, np.inf), "bf16")
    got = load(run_prefix(backend, q, pk, pv, k, v, lengths, types), "bf16")
    assert np.all(got[:, :2] == np.inf)
    assert np.all(np.isnan(got[2, 2:])) and np.all(np.isfinite(got[[0, 1, 3, 4], 2:]))


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("count,heads,kv_heads", [(1, 1, 1), (3, 1, 1), (17, 6, 2), (5, 35, 7), (1, 3, 3)], ids=str)
@pytest.mark.parametrize("size", [64, 104])
def test_prefix_odd_partial_rows(backend, types, count, heads, kv_heads, size):
    """Shares of both ranges whose rows are odd in number."""
    rng = np.random.default_rng(count + heads)
    lengths = rng.integers(0, 900, count)
    lengths[0] = 900
    arrays = prefix_inputs(count * heads, count, 1300, 900, heads, kv_heads, size, types)
    got = run_prefix(backend, *arrays, lengths, types)
    check_prefix(got, *arrays, lengths, types)


def test_attention_is_deterministic(backend):
    types = ("f32", "f16")
    arrays = prefix_inputs(5, 20, 1800, 400, 8, 4, 128, types)
    lengths = np.random.default_rng(5).integers(0, 400, 20)
    first = run_prefix(backend, *arrays, lengths, types)
    q, k, v = packed_inputs(6, [300, 40], [1800, 2500], 8, 4, 128, types)
    packed = run_packed(backend, q, k, v, offsets([300, 40]), offsets([1800, 2500]), types)
    for _ in range(3):
        assert np.array_equal(first.view(np.uint32), run_prefix(backend, *arrays, lengths, types).view(np.uint32))
        again = run_packed(backend, q, k, v, offsets([300, 40]), offsets([1800, 2500]), types)
        assert np.array_equal(packed.view(np.uint32), again.view(np.uint32))


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


@pytest.mark.parametrize("kind,rows", [("f32", 120), ("f32", 330), ("f32", 430), ("bf16", 250), ("bf16", 870)])
def test_choice_of_large_batches(backend, kind, rows):
    """Workgroups that take several chunks of a row, lists that name few or nearly all tokens of a chunk."""
    vocab, history, biases = 20011, 3500, 700
    v = choice_inputs(rows, rows, vocab, history, biases, 3, kind)
    rng = np.random.default_rng(rows)
    for r in range(rows):
        if r % 3 == 0:    # few
            v["counts"][r], v["bias_counts"][r] = 40, 9
        elif r % 3 == 1:  # every token of a range, in any order
            start = int(rng.integers(0, vocab - history))
            v["history"][r] = start + rng.permutation(history)
            v["bias_tokens"][r] = start + rng.permutation(biases) - 50
            v["counts"][r], v["bias_counts"][r] = history, biases
        else:             # one token
            v["history"][r] = r
    got, picked = run_choice(backend, v, kind, pad=5)
    for at in (slice(0, 40), slice(rows // 2, rows // 2 + 9), slice(rows - 9, rows)):
        some = {n: a if n == "masks" else a[at] for n, a in v.items()}
        check_choice(got[at], picked[at], some, kind)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_choice_of_unusual_values(backend, kind):
    v = choice_inputs(3, 6, 700, 30, 5, 0, kind)
    x = load(v["logits"], kind)
    x[0, ::3] = np.nan
    x[1] = -np.inf
    x[2, 5], x[2, 600] = np.inf, np.inf
    x[3] = np.nan
    x[4] = -0.0
    x[4, 300] = 0.0
    v["logits"] = store(x, kind)
    v["counts"][:] = [30, 0, 30, 30, 0, 30]
    v["bias_counts"][:] = [5, 0, 0, 0, 0, 5]
    got, picked = run_choice(backend, v, kind)
    check_choice(got, picked, v, kind)
    assert picked[1] == -1 and picked[3] == -1 and picked[4] == 0


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_choice_lists_and_masks_shared_by_rows(backend, kind):
    """Stride 0 lists, one mask for all, no index, no counts, unaligned and differently aligned rows."""
    from funasrnet_amd import hip
    from funasrnet_amd.device import DeviceArray
    rng = np.random.default_rng(17)
    rows, vocab = 5, 3001
    v = choice_inputs(18, rows, vocab, 12, 4, 1, kind)
    v["masks"][0] = rng.integers(0, 1 << 32, v["masks"].shape[1], dtype=np.uint64)
    for lead_in, lead_out in ((0, 0), (1, 1), (3, 2), (5, 0)):
        width = 4 if kind == "f32" else 2
        wide = np.full(rows * (vocab + 6) + 8, 3, v["logits"].dtype)
        for r in range(rows):
            wide[lead_in + r * (vocab + 6):][:vocab] = v["logits"][r]
        logits, out = to_device(wide), to_device(np.full_like(wide, 4))
        chosen = DeviceArray(rows, np.int32)
        held = {n: to_device(a[0] if n in ("history", "bias_tokens", "bias_values") else a) for n, a in v.items() if n != "logits"}
        call = hip.LogitsAdjust(logits=logits.ptr + lead_in * width, output=out.ptr + lead_out * width, tokens=chosen.ptr,
                                logits_stride=vocab + 6, output_stride=vocab + 6, rows=rows, vocab=vocab, type=CODES[kind],
                                history=held["history"].ptr, history_stride=0, history_capacity=12,
                                repetition=held["repetition"].ptr, bias_tokens=held["bias_tokens"].ptr,
                                bias_values=held["bias_values"].ptr, bias_stride=0, bias_capacity=4, masks=held["masks"].ptr,
                                mask_stride=v["masks"].shape[1], mask_rows=1)
        need = backend.logits_adjust_workspace(call)
        ws = workspace_of(need)
        call.workspace, call.workspace_bytes = ws.ptr, need
        assert backend.logits_adjust_device(call) == hip.OK
        backend.synchronize()
        got, picked = out.numpy(), chosen.numpy()
        mask = np.unpackbits(v["masks"][0].view(np.uint8), bitorder="little")[:vocab] == 1
        for r in range(rows):
            bias = list(zip(v["bias_tokens"][0].tolist(), v["bias_values"][0]))
            expected, token = adjusted(load(v["logits"][r], kind), v["history"][0].tolist(), 0, v["repetition"][r], 0, 0, bias,
                                       mask, kind)
            row = got[lead_out + r * (vocab + 6):]
            assert np.array_equal(row[:vocab].view(np.uint8), expected.view(np.uint8)) and picked[r] == token
            assert np.all(row[vocab:vocab + 6] == 4)


def test_choice_counts_out_of_range(backend):
    """Counts below 0 and above the capacity, prompts longer than the history."""
    v = choice_inputs(19, 4, 500, 20, 6, 0, "f32")
    v["counts"][:] = [-3, 21, 20, 2**31 - 1]
    v["prompts"][:] = [0, -5, 2**31 - 1, 3]
    v["bias_counts"][:] = [7, -1, 2**31 - 1, 0]
    got, picked = run_choice(backend, v, "f32")
    v["counts"][:] = [0, 20, 20, 20]
    v["bias_counts"][:] = [6, 0, 6, 0]
    check_choice(got, picked, v, "f32")


# ---- Refusals that need a context -----------------------------------------------------


def test_refusals_with_a_context(backend):
    from funasrnet_amd import hip
    lib = hip.load()
    import ctypes
    types = ("f32", "f16")
    q, k, v = packed_inputs(1, [4], [3000], 2, 1, 128, types)
    dq, dk, dv, out = to_device(q), to_device(k), to_device(v), to_device(np.full_like(q, 5))
    qo, ko = to_device(offsets([4])), to_device(offsets([3000]))

    def call(**changes):
        a = hip.PackedAttention(query=dq.ptr, key=dk.ptr, value=dv.ptr, output=out.ptr, query_row=256, query_head=128,
                                key_row=128, key_head=128, value_row=128, value_head=128, output_row=256, output_head=128,
                                query_offsets=qo.ptr, key_offsets=ko.ptr, sequences=1, query_rows=4, key_rows=3000,
                                longest_query=4, longest_key=3000, heads=2, kv_heads=1, head_size=128,
                                query_type=hip.TYPE_F32, cache_type=hip.TYPE_F16, scale=0.1)
        need = backend.attention_packed_workspace(a)
        assert need > 0
        a.workspace_bytes = need
        for name, value in changes.items():
            setattr(a, name, value)
        return lib.fah_attention_packed_device(backend.handle, ctypes.byref(a))

    ws = workspace_of(1 << 22)
    assert call() == hip.ERROR_ARGUMENT and b"workspace" in lib.fah_last_error()          # none given
    assert call(workspace=ws.ptr, workspace_bytes=16) == hip.ERROR_ARGUMENT               # too small
    assert call(workspace=ws.ptr + 4) == hip.ERROR_ARGUMENT                               # off its boundary
    for name in ("query", "key", "value", "output", "query_offsets"):
        assert call(workspace=ws.ptr, **{name: None}) == hip.ERROR_ARGUMENT, name
    for name, at in (("query", dq.ptr), ("key", dk.ptr), ("value", dv.ptr), ("output", out.ptr)):
        assert call(workspace=ws.ptr, **{name: at + 2}) == hip.DECLINED, name
    assert np.all(out.numpy() == 5)
    assert call(workspace=ws.ptr, sequences=0) == hip.OK and call(workspace=ws.ptr, query_rows=0) == hip.OK
    backend.synchronize()
    assert np.all(out.numpy() == 5)
    a = hip.LogitsAdjust(logits=dq.ptr, output=out.ptr, logits_stride=100, output_stride=100, rows=2, vocab=100)
    for changes in (dict(logits=None), dict(output=None), dict(output_stride=99), dict(logits=dq.ptr + 2),
                    dict(history_capacity=1), dict(bias_capacity=1), dict(mask_rows=1), dict(logits=out.ptr, logits_stride=128),
                    dict(vocab=0), dict(tokens=qo.ptr)):
        b = hip.LogitsAdjust.from_buffer_copy(a)
        for name, value in changes.items():
            setattr(b, name, value)
        assert lib.fah_logits_adjust_device(backend.handle, ctypes.byref(b)) == hip.ERROR_ARGUMENT, changes
    assert np.all(out.numpy() == 5)


# ---- Together, in graphs, on threads -----------------------------------------------------


class Serving:
    """A batch behind a shared prefix: its prompts, a decode step and the choice of a token."""

    def __init__(self, backend, seed, count=6, prefix=600, own=70, heads=8, kv_heads=4, vocab=4000):
        from funasrnet_amd import hip
        from funasrnet_amd.device import DeviceArray
        self.backend, self.types, size = backend, ("f32", "f16"), 128
        rng = np.random.default_rng(seed)
        self.q, self.pk, self.pv, self.k, self.v = prefix_inputs(seed, count, prefix, own, heads, kv_heads, size, self.types)
        self.lengths = rng.integers(1, own + 1, count).astype(np.int32)
        self.choice = choice_inputs(seed, count, vocab, 40, 8, 3, "f32")
        self.hold = {n: to_device(a) for n, a in dict(q=self.q, pk=self.pk, pv=self.pv, k=self.k, v=self.v, lengths=self.lengths,
                                                      **self.choice).items()}
        d = self.hold
        self.out, self.adjusted = DeviceArray(self.q.shape, np.float32), DeviceArray((count, vocab), np.float32)
        self.tokens = DeviceArray(count, np.int32)
        row = kv_heads * size
        self.attend = hip.PrefixAttention(
            query=d["q"].ptr, prefix_key=d["pk"].ptr, prefix_value=d["pv"].ptr, key=d["k"].ptr, value=d["v"].ptr,
            output=self.out.ptr, lengths=d["lengths"].ptr, query_sequence=heads * size, query_head=size, prefix_key_row=row,
            prefix_key_head=size, prefix_value_row=row, prefix_value_head=size, key_sequence=own * row, key_row=row,
            key_head=size, value_sequence=own * row, value_row=row, value_head=size, output_sequence=heads * size,
            output_head=size, sequences=count, prefix=prefix, capacity=own, longest=own, heads=heads, kv_heads=kv_heads,
            head_size=size, query_type=hip.TYPE_F32, cache_type=hip.TYPE_F16, scale=size**-0.5)
        self.pick = hip.LogitsAdjust(
            logits=d["logits"].ptr, output=self.adjusted.ptr, tokens=self.tokens.ptr, logits_stride=vocab, output_stride=vocab,
            rows=count, vocab=vocab, type=hip.TYPE_F32, history=d["history"].ptr, history_stride=40, history_capacity=40,
            history_counts=d["counts"].ptr, prompt_counts=d["prompts"].ptr, repetition=d["repetition"].ptr,
            presence=d["presence"].ptr, frequency=d["frequency"].ptr, bias_tokens=d["bias_tokens"].ptr,
            bias_values=d["bias_values"].ptr, bias_stride=8, bias_capacity=8, bias_counts=d["bias_counts"].ptr,
            masks=d["masks"].ptr, mask_stride=self.choice["masks"].shape[1], mask_rows=3, mask_index=d["index"].ptr)
        # The prefix's own rows as a packed prompt, with the first sequence's queries repeated.
        self.prompt_q = np.ascontiguousarray(np.resize(self.q, (prefix, heads, size)))
        self.prompt_out = DeviceArray(self.prompt_q.shape, np.float32)
        self.hold["prompt_q"], self.hold["offsets"] = to_device(self.prompt_q), to_device(offsets([prefix]))
        self.prompt = hip.PackedAttention(
            query=d["prompt_q"].ptr, key=d["pk"].ptr, value=d["pv"].ptr, output=self.prompt_out.ptr, query_row=heads * size,
            query_head=size, key_row=row, key_head=size, value_row=row, value_head=size, output_row=heads * size,
            output_head=size, query_offsets=d["offsets"].ptr, sequences=1, query_rows=prefix, key_rows=prefix,
            longest_query=prefix, longest_key=prefix, heads=heads, kv_heads=kv_heads, head_size=size,
            query_type=hip.TYPE_F32, cache_type=hip.TYPE_F16, scale=size**-0.5)
        self.spaces = []
        for a, need in ((self.attend, backend.attention_prefix_workspace(self.attend)),
                        (self.pick, backend.logits_adjust_workspace(self.pick)),
                        (self.prompt, backend.attention_packed_workspace(self.prompt))):
            self.spaces.append(workspace_of(need))
            a.workspace, a.workspace_bytes = self.spaces[-1].ptr, need

    def enqueue(self):
        from funasrnet_amd import hip
        assert self.backend.attention_packed_device(self.prompt) == hip.OK
        assert self.backend.attention_prefix_device(self.attend) == hip.OK
        assert self.backend.logits_adjust_device(self.pick) == hip.OK

    def results(self):
        return self.prompt_out.numpy(), self.out.numpy(), self.adjusted.numpy(), self.tokens.numpy()

    def clear(self):
        for a in (self.prompt_out, self.out, self.adjusted, self.tokens):
            a.fill_zero()
        for a in self.spaces:
            a.upload(np.full(a.shape, 0xFF, np.uint8))

    def check(self):
        prompt, out, logits, tokens = self.results()
        check_packed(prompt, self.prompt_q, self.pk, self.pv, offsets([len(self.pk)]), None, self.types)
        check_prefix(out, self.q, self.pk, self.pv, self.k, self.v, self.lengths, self.types)
        check_choice(logits, tokens, self.choice, "f32")


def same(a, b):
    return all(np.array_equal(x.view(np.uint8), y.view(np.uint8)) for x, y in zip(a, b))


def test_a_serving_step(backend):
    """Prompts, decode behind the prefix, choice, one behind the other on the context's stream."""
    s = Serving(backend, 21)
    s.clear()
    s.enqueue()
    backend.synchronize()
    s.check()
    # A sequence that decodes the last row of its own prompt gets that row's result.
    n, heads = int(s.lengths[0]), s.q.shape[1]
    k = np.concatenate([s.pk, s.k[0, :n]])
    v = np.concatenate([s.pv, s.v[0, :n]])
    queries = np.ascontiguousarray(np.resize(s.q, (n, heads, 128)))
    queries[-1] = s.q[0]
    got = run_packed(backend, queries, k, v, offsets([n]), offsets([len(k)]), s.types)
    assert np.abs(got[-1] - s.results()[1][0]).max() < 1e-5


def test_graphs_replay_the_calls(backend):
    """Two graphs with workspaces of their own, replayed several times with other
    work and changed inputs between, against the calls made one by one."""
    import ctypes
    from funasrnet_amd import device
    run = device.runtime()
    vp = ctypes.c_void_p
    both = [Serving(backend, 31), Serving(backend, 32, count=3, prefix=2500, own=300)]
    graphs = []
    for s in both:
        s.enqueue()  # once before, as a program warms up
        backend.synchronize()
        graph, made = vp(), vp()
        assert run.hipStreamBeginCapture(vp(backend.stream), 2) == 0  # relaxed
        s.enqueue()
        assert run.hipStreamEndCapture(vp(backend.stream), ctypes.byref(graph)) == 0
        assert run.hipGraphInstantiate(ctypes.byref(made), graph, None, None, ctypes.c_size_t(0)) == 0
        graphs.append((graph, made))
    rng = np.random.default_rng(33)
    for turn in range(4):
        for s in both:
            s.q = (rng.standard_normal(s.q.shape) * 1.5).astype(np.float32)
            s.lengths = rng.integers(1, s.k.shape[1] + 1, len(s.lengths)).astype(np.int32)
            s.hold["q"].upload(s.q)
            s.hold["lengths"].upload(s.lengths)
            s.clear()
        for _, made in graphs:
            assert run.hipGraphLaunch(made, vp(backend.stream)) == 0
        backend.synchronize()
        replayed = [s.results() for s in both]
        for s, r in zip(both, replayed):
            s.check()
            s.clear()
            s.enqueue()
            backend.synchronize()
            assert same(r, s.results()), turn
    for graph, made in graphs:
        run.hipGraphExecDestroy(made)
        run.hipGraphDestroy(graph)


def test_two_contexts_on_two_threads():
    import threading
    from funasrnet_amd.hip import HipBackend
    backends = [HipBackend(0), HipBackend(0)]
    try:
        work = [Serving(b, 41 + i, count=5 + i) for i, b in enumerate(backends)]
        for s in work:
            s.enqueue()
            s.backend.synchronize()
        alone = [s.results() for s in work]
        for s in work:
            s.clear()
        errors = []

        def turn(s, expected):
            try:
                for _ in range(30):
                    s.enqueue()
                    s.backend.synchronize()
                if not same(expected, s.results()):
                    errors.append("results differ")
            except Exception as e:  # reported below
                errors.append(repr(e))

        threads = [threading.Thread(target=turn, args=(s, r)) for s, r in zip(work, alone)]
        for t in threads:
            t.start()
        for t in threads:
            t.join(timeout=60)
        assert not any(t.is_alive() for t in threads) and not errors, errors
    finally:
        for b in backends:
            b.close()


# ---- The decoder's own loop -----------------------------------------------------------


@pytest.mark.parametrize("persistent", ["1", "0"])
def test_decoder_choose(persistent, monkeypatch, oracle_lib):
    """choose() adjusts the step's logits, and generate() goes on with its token."""
    from funasrnet_amd import hip, model
    monkeypatch.setenv("FAH_PERSISTENT", persistent)
    weights = model.synthetic(model.small_config(layers=2, vocab=2048), seed=3)
    x = np.random.default_rng(0).standard_normal((6, weights.config.width)).astype(np.float32)
    backend = hip.HipBackend(0)
    gpu, ref = hip.HipDecoder(backend, weights, capacity=64), oracle_lib.Decoder(weights, capacity=64)
    try:
        with pytest.raises(RuntimeError, match="no logits"):
            gpu.choose()
        logits = gpu.decode(x, 6)
        expected = ref.decode(x, 6)
        rng = np.random.default_rng(7)
        written, prompt = [5, 9, 5], 2
        for step in range(8):
            mask = rng.random(2048) < 0.7
            biases = {int(t): float(b) for t, b in zip(rng.integers(0, 2048, 4), rng.uniform(-2, 2, 4))}
            seen = np.empty(2048, np.float32)
            token = gpu.choose(written, prompt, 1.3, 0.4, 0.2, biases, mask, seen)
            want, choice = adjusted(logits, written, prompt, 1.3, 0.4, 0.2, list(biases.items()), mask, "f32")
            assert np.array_equal(seen.view(np.uint32), want.view(np.uint32)) and token == choice
            assert gpu.greedy() == token
            # Its row's logits: the oracle's after the same token.
            assert gpu.generate(1).tolist() == [token]
            expected = ref.decode(ref.embed([token]), 1)
            written.append(token)
            logits = np.empty(2048, np.float32)
            gpu.choose(logits=logits)  # as they are
            assert np.abs(logits - expected).max() < 1e-2
        assert gpu.position == 6 + 8
        # Nothing left to choose.
        assert gpu.choose(mask=np.zeros(2048, bool)) == -1
        with pytest.raises(RuntimeError, match="no logits"):
            gpu.generate(1)
        gpu.set_position(6)
        gpu.decode(x[:1], 1)
        # A lock-step step keeps no logits.
        hip.HipDecoder.generate_sessions([gpu], 1)
        with pytest.raises(RuntimeError, match="lock-step"):
            gpu.choose()
    finally:
        gpu.close()
        ref.close()
        backend.close()


# ---- Scores and values far from 1 -------------------------------------------------------


def whole_scores(rng, rows, keys, heads, kv_heads, size, types, shift):
    """Queries and keys of few bits, so that every score is exact in 32 bits: `shift` powers of two times a whole number."""
    limit = {"f32": 100, "f16": 13, "bf16": 60}[types[0]]
    up = min(shift, limit)
    q = store(rng.integers(-1, 2, (rows, heads, size)) * np.exp2(up), types[0])
    k = store(rng.integers(-8, 9, (keys, kv_heads, size)) * np.exp2(shift - up), types[1])
    return q, k


def check_exact_scores(got, q, k, v, offset, types, scale, span):
    """Scores without rounding errors: only those of the weights (of scores at most `span` below the largest), sums and output stay."""
    heads, kv_heads, size = q.shape[1], k.shape[1], q.shape[2]
    fq, fk, fv, fg = load(q, types[0]), load(k, types[1]), load(v, types[1]), load(got, types[0])
    for h in range(heads):
        g = h // (heads // kv_heads)
        out, weight, _ = attend_all(fq[:, h], fk[:, g], fv[:, g], scale, offset)
        off = np.abs(fg[:, h] - out)
        limit = attention_bound(out, weight, span, len(k), size, types[0])
        assert np.all(off <= limit), (h, float((off / limit).max()))


@pytest.mark.parametrize("types,shifts", [(("f32", "f16"), (12, 20, 24, 28, 32, 40, 100)), (("f16", "f16"), (12, 20, 23)),
                                          (("bf16", "bf16"), (12, 20, 24, 28, 32, 40, 100))], ids=lambda t: "-".join(map(str, t)))
@pytest.mark.parametrize("rows,heads,kv_heads,extra", [(130, 2, 1, 0), (1100, 64, 64, 0), (40, 4, 2, 3000), (1, 4, 4, 500)])
def test_packed_scores_of_any_size(backend, types, shifts, rows, heads, kv_heads, extra):
    """From thousands to 2^100 and more: the keys with the largest score share the weight."""
    for shift in shifts:
        rng = np.random.default_rng(shift * 7 + rows)
        print(f"scores {shift} {rows} {heads}/{kv_heads} {extra} {types}", flush=True)
        q, k = whole_scores(rng, rows, rows + extra, heads, kv_heads, 128, types, shift)
        v = store(rng.standard_normal(k.shape), types[1])
        got = run_packed(backend, q, k, v, offsets([rows]), offsets([rows + extra]), types)
        # (Other scores are at least 2^12 128^-0.5 below: weight 0.)
        some = [0, 1, heads // 2, heads - 1] if heads > 4 else range(heads)
        for h in some:
            g = h // (heads // kv_heads)
            check_exact_scores(got[:, h:h + 1], q[:, h:h + 1], k[:, g:g + 1], v[:, g:g + 1], extra, types, 128**-0.5, 1.0)


def close_scores(rng, queries, keys, size, types, power, order):
    """Scores 2^power + n units, n below 12, with the keys in the order of n or in any: a unit is the step of a 32-bit value there."""
    unit = power - 23
    n = rng.integers(0, 12, keys)
    if order == "rising":
        n.sort()
    q, k = np.zeros((queries, 1, size)), np.zeros((keys, 1, size))
    big = {"f32": 14, "f16": 14, "bf16": 40}[types[0]]
    q[:, 0, 0], k[:, 0, 0] = np.exp2(min(big, power)), np.exp2(power - min(big, power))
    q[:, 0, 1:3], k[:, 0, 1] = np.exp2(max(unit, 0)), n * np.exp2(min(unit, 0))
    return store(q, types[0]), store(k, types[1])


@pytest.mark.parametrize("types,powers", [(("f32", "f16"), (15, 22, 25, 27)), (("f16", "f16"), (15, 22, 25, 28)),
                                          (("bf16", "bf16"), (15, 23, 28, 36, 60))], ids=lambda t: "-".join(map(str, t)))
@pytest.mark.parametrize("order", ["rising", "any"])
@pytest.mark.parametrize("unit", [0.02, 0.3, 2.0, 9.0])
def test_scores_whose_differences_are_their_last_bits(backend, types, powers, order, unit):
    """Scores of up to 2^27 and more after scaling, a few of their last bits apart: whole weights, and shares that agree."""
    size = 64
    for power in powers:
        rng = np.random.default_rng(power)
        scale = float(np.float32(unit * 2.0**(23 - power)))
        for queries, keys in ((90, 90), (3, 1400)):
            q, k = close_scores(rng, queries, keys, size, types, power, order)
            v = store(rng.standard_normal(k.shape), types[1])
            got = run_packed(backend, q, k, v, offsets([queries]), offsets([keys]), types, scale=scale)
            check_exact_scores(got, q, k, v, keys - queries, types, scale, 12 * unit)
        q, k = close_scores(rng, 5, 2100, size, types, power, order)
        v = store(rng.standard_normal(k.shape), types[1])
        lengths = np.array([100, 0, 37, 64, 1])
        own_k, own_v = (np.stack([a[2000:]] * 5) for a in (k, v))
        got = run_prefix(backend, q, k[:2000], v[:2000], own_k, own_v, lengths, types, scale=scale)
        for s, n in enumerate(lengths):
            check_exact_scores(got[s:s + 1], q[s:s + 1], k[:2000 + n], v[:2000 + n], 2000 + n, types, scale, 12 * unit)


@pytest.mark.parametrize("magnitude,scale", [(1e36, 1e-38), (1e30, 1e-31), (1e-6, 1e5), (1e-30, 1e29), (1e-37, 1e36)])
def test_shares_of_fp32_queries_of_any_size(backend, magnitude, scale):
    """Joined rows whose scores before scaling are beyond 32 bits, or close to nothing."""
    types, f = ("f32", "f16"), np.float32(scale)
    q, k, v = packed_inputs(14, [60, 3], [2100, 1300], 4, 2, 128, types)
    q *= np.float32(magnitude)
    k = store(load(k, "f16") * 40, "f16") if magnitude > 1e30 else k
    qo, ko = offsets([60, 3]), offsets([2100, 1300])
    check_packed(run_packed(backend, q, k, v, qo, ko, types, scale=float(f)), q, k, v, qo, ko, types, scale=float(f))
    lengths = [3, 400, 0, 77]
    q, pk, pv, k, v = prefix_inputs(15, 4, 1500, 400, 4, 2, 128, types)
    q *= np.float32(magnitude)
    pk, k = (store(load(x, "f16") * 40, "f16") if magnitude > 1e30 else x for x in (pk, k))
    for heads_first in (True, False):
        got = run_prefix(backend, q, pk, pv, k, v, lengths, types, scale=float(f), heads_first=heads_first)
        check_prefix(got, q, pk, pv, k, v, lengths, types, scale=float(f))
    # A value that is not finite, where rows are formed again.
    v[1, 399, 1] = np.inf
    got = run_prefix(backend, q, pk, pv, k, v, lengths, types, scale=float(f))
    assert np.all(got[1, 2:] == np.inf)
    check_prefix(got[[0, 2, 3]], q[[0, 2, 3]], pk, pv, k[[0, 2, 3]], v[[0, 2, 3]], [3, 0, 77], types, scale=float(f))


def test_calls_without_any_keys(backend):
    """No key rows at all, and their buffers NULL: zeros."""
    from funasrnet_amd import hip
    rng = np.random.default_rng(2)
    for kinds, dtype in ((("f32", "f16"), np.float32), (("f16", "f16"), np.float16), (("bf16", "bf16"), np.uint16)):
        q = to_device(store(rng.standard_normal((9, 4, 64)), kinds[0]))
        assert q.dtype == dtype
        codes = dict(query_type=CODES[kinds[0]], cache_type=CODES[kinds[1]], scale=0.125, heads=4, kv_heads=2, head_size=64)
        zero, at = to_device(np.zeros(10, np.int32)), to_device(np.array([0, 4, 9], np.int32))
        out = to_device(np.full((9, 4, 64), 3, dtype))
        call = hip.PackedAttention(query=q.ptr, output=out.ptr, query_row=256, query_head=64, key_row=128, key_head=64, value_row=128,
                                   value_head=64, output_row=256, output_head=64, query_offsets=at.ptr, key_offsets=zero.ptr,
                                   sequences=2, query_rows=9, longest_query=5, **codes)
        assert backend.attention_packed_workspace(call) == 0 and backend.attention_packed_device(call) == hip.OK
        backend.synchronize()
        assert np.all(load(out.numpy(), kinds[0]) == 0)
        out = to_device(np.full((9, 4, 64), 3, dtype))
        call = hip.PrefixAttention(query=q.ptr, output=out.ptr, lengths=zero.ptr, query_sequence=256, query_head=64, prefix_key_row=64,
                                   prefix_value_row=64, key_row=64, value_row=64, output_sequence=256, output_head=64, sequences=9,
                                   **codes)
        assert backend.attention_prefix_workspace(call) == 0 and backend.attention_prefix_device(call) == hip.OK
        backend.synchronize()
        assert np.all(load(out.numpy(), kinds[0]) == 0)


@pytest.mark.parametrize("power", [126, 118, -112])
@pytest.mark.parametrize("queries,keys,heads,kv_heads,size", [(130, 130, 4, 2, 128), (1100, 1100, 64, 64, 64), (9, 3000, 4, 2, 128)],
                         ids=str)
def test_bf16_values_of_any_size(backend, power, queries, keys, heads, kv_heads, size):
    """Values near either end of the type's range: rows of every tile, and partial ones."""
    types = ("bf16", "bf16")
    q, k, v = packed_inputs(power + 200, [queries], [keys], heads, kv_heads, size, types)
    v = store(np.clip(load(v, "bf16"), -3.5, 3.5) * np.float32(2.0**power), "bf16")
    assert np.all(np.isfinite(load(v, "bf16")))
    got = run_packed(backend, q, k, v, offsets([queries]), offsets([keys]), types)
    fq, fk, fv, fg = load(q, "bf16"), load(k, "bf16"), load(v, "bf16") * 2.0**-power, load(got, "bf16") * 2.0**-power
    for h in sorted({0, 1, heads - 1}):
        g = h // (heads // kv_heads)
        out, weight, dots = attend_all(fq[:, h], fk[:, g], fv[:, g], size**-0.5, keys - queries)
        # Sums of small values end in the 32-bit numbers below the normal ones: a step of 2^-149 a key.
        floor = 2.0 * keys * 2.0**(-149 + 24 - power) if power < 0 else 0.0
        assert np.all(np.abs(fg[:, h] - out) <= attention_bound(out, weight, dots, keys, size, "bf16") + floor), h
    lengths = [0, 1, 40, 70]
    for prefix in (0, 2000):
        q, pk, pv, k, v = prefix_inputs(power + 201, len(lengths), prefix, 70, heads, kv_heads, size, types)
        pv, v = (store(np.clip(load(x, "bf16"), -3.5, 3.5) * np.float32(2.0**power), "bf16") for x in (pv, v))
        got = run_prefix(backend, q, pk, pv, k, v, lengths, types)
        assert np.all(np.isfinite(load(got, "bf16")))
        if power > 0:
            down = [store(load(x, "bf16") * np.float32(2.0**-power), "bf16") for x in (got, pv, v)]
            check_prefix(down[0], q, pk, down[1], k, down[2], lengths, types)


# ---- Values that are not finite ------------------------------------------------------------


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("rows,extra,heads,kv_heads,size", [(40, 0, 2, 2, 128), (300, 0, 6, 2, 64), (1100, 0, 64, 64, 128), (400, 2500, 64, 64, 64),
                                                            (60, 2000, 8, 4, 104), (5, 900, 4, 4, 128)], ids=str)
def test_values_that_are_not_finite(backend, types, rows, extra, heads, kv_heads, size):
    """Each channel by itself: NaN or infinite from the first key that holds one on, whatever its tile masks, and as ever in the others."""
    keys = rows + extra
    q, k, v = packed_inputs(rows + size, [rows], [keys], heads, kv_heads, size, types)
    late = [keys - 1 - n for n in (0, min(rows - 1, 3), rows // 2, rows - 1)]  # keys that some rows see
    spoilt = load(v, types[1]).astype(np.float32)
    spoilt[0, :, 2], spoilt[:, :, 5] = np.nan, np.inf                # from the first key on; everywhere
    spoilt[extra // 2, :, 7] = -np.inf
    spoilt[late[1], :, 11], spoilt[late[2], :, 13], spoilt[late[3], :, 17] = np.nan, np.inf, -np.inf
    spoilt[late[0]] = np.nan                                         # the last key: one row alone
    clean = np.where(np.isfinite(spoilt), spoilt, 0.0)
    got = load(run_packed(backend, q, k, store(spoilt, types[1]), offsets([rows]), offsets([keys]), types), types[0])
    fq, fk = load(q, types[0]), load(k, types[1])
    seen = np.arange(keys)[None, :] <= np.arange(rows)[:, None] + extra
    for h in sorted({0, 1, heads // 2, heads - 1}):
        g = h // (heads // kv_heads)
        out, weight, dots = attend_all(fq[:, h], fk[:, g], clean[:, g], size**-0.5, extra)
        limit = attention_bound(out, weight, dots, keys, size, types[0])
        for kind, test in (("nan", np.isnan), ("inf", np.isposinf), ("-inf", np.isneginf)):
            spoilt_by = (seen.astype(np.float32) @ test(spoilt[:, g]).astype(np.float32)) > 0  # [rows, size]
            if kind == "nan":
                nan = spoilt_by
            elif kind == "inf":
                up = spoilt_by
            else:
                down = spoilt_by
        nan |= up & down
        assert np.array_equal(np.isnan(got[:, h]), nan), h
        assert np.array_equal(np.isposinf(got[:, h]), up & ~nan) and np.array_equal(np.isneginf(got[:, h]), down & ~nan), h
        finite = ~(nan | up | down)
        assert np.all(np.abs(got[:, h] - out)[finite] <= limit[finite]), h


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("rows,extra,heads,kv_heads", [(150, 0, 2, 2), (1100, 0, 64, 64), (70, 3000, 4, 2)], ids=str)
def test_rows_of_minus_infinity_scores_over_any_values(backend, types, rows, extra, heads, kv_heads):
    """Zeros, whatever the values are."""
    q, k, v = packed_inputs(rows, [rows], [rows + extra], heads, kv_heads, 64, types)
    q[:] = store(np.abs(load(q, types[0])) + 0.1, types[0])
    k[:] = store(np.full(k.shape, -np.inf), types[1])
    v[::3] = store(np.full(v[::3].shape, np.nan), types[1])
    v[1::3] = store(np.full(v[1::3].shape, np.inf), types[1])
    got = load(run_packed(backend, q, k, v, offsets([rows]), offsets([rows + extra]), types), types[0])
    assert np.all(got == 0)
    for prefix in (0, 1500):
        q, pk, pv, k, v = prefix_inputs(9, 3, prefix, 90, heads, kv_heads, 64, types)
        q = store(np.abs(load(q, types[0])) + 0.1, types[0])
        pk, k = (store(np.full(x.shape, -np.inf), types[1]) for x in (pk, k))
        pv, v = (store(np.full(x.shape, np.nan), types[1]) for x in (pv, v))
        assert np.all(load(run_prefix(backend, q, pk, pv, k, v, [90, 0, 33], types), types[0]) == 0)


@pytest.mark.parametrize("types", TYPES, ids=lambda t: "-".join(t))
@pytest.mark.parametrize("rows,extra,heads,kv_heads,size", [(70, 0, 2, 2, 64), (1100, 0, 64, 64, 128), (400, 2500, 64, 64, 64), (60, 2000, 8, 4, 104),
                                                            (3, 900, 4, 4, 128)], ids=str)
def test_infinite_keys(backend, types, rows, extra, heads, kv_heads, size):
    """Scores of -infinity weigh nothing, whatever their values are short of NaN and infinity; those of infinity make the row NaN."""
    keys = rows + extra
    q, k, v = packed_inputs(rows + 3, [rows], [keys], heads, kv_heads, size, types)
    # Channel 5 of queries: above 0, but for every seventh row.
    side = np.where(np.arange(rows) % 7 == 3, -1.0, 1.0)
    q[:, :, 5] = store(side[:, None] * (np.abs(load(q[:, :, 5], types[0])) + 0.125), types[0])
    k[::5, :, 5] = store(np.full(k[::5, :, 5].shape, -np.inf), types[1])
    got = load(run_packed(backend, q, k, v, offsets([rows]), offsets([keys]), types), types[0])
    fq, fk, fv = load(q, types[0]), load(k, types[1]), load(v, types[1])
    at, others = np.arange(keys) % 5 != 0, side > 0
    seen = np.arange(keys)[None, :] <= np.arange(rows)[:, None] + extra
    for h in sorted({0, heads // 2, heads - 1}):
        g = h // (heads // kv_heads)
        assert np.all(np.isnan(got[~others, h])), h
        for r in np.flatnonzero(others)[:: max(1, rows // 40)]:
            out, weight, dots = attend(fq[r:r + 1, h], fk[at, g], fv[at, g], size**-0.5, seen[r:r + 1, at])
            assert np.all(np.abs(got[r, h] - out[0]) <= attention_bound(out, weight, dots, keys, size, types[0])[0]), (h, r)
    for prefix in (0, 1200):
        lengths = [90, 1, 33]
        q, pk, pv, k, v = prefix_inputs(10, 3, prefix, 90, heads, kv_heads, size, types)
        q[:, :, 5] = store(np.abs(load(q[:, :, 5], types[0])) + 0.125, types[0])
        drop = [np.arange(n) % 3 == 1 for n in (prefix, 90)]
        pk[drop[0], :, 5], k[:, drop[1], :, 5] = (store(np.float32(-np.inf), types[1]) for _ in range(2))
        got = run_prefix(backend, q, pk, pv, k, v, lengths, types)
        kept = [int(np.sum(~drop[1][:n])) for n in lengths]
        check_prefix(got, q, pk[~drop[0]], pv[~drop[0]], k[:, ~drop[1]], v[:, ~drop[1]], kept, types)


# ---- Captures beside another context's steps ------------------------------------------------


@pytest.mark.parametrize("order", ["step first", "call first"])
def test_capture_beside_another_contexts_steps(backend, order):
    """A decoder of another context steps (persistent, lock-step) while the calls are captured: neither notices."""
    import ctypes
    from funasrnet_amd import device, hip, model
    run, vp = device.runtime(), ctypes.c_void_p
    weights = model.synthetic(model.small_config(layers=2, vocab=2048), seed=5)
    x = np.random.default_rng(1).standard_normal((6, weights.config.width)).astype(np.float32)
    other = hip.HipBackend(0)
    decoder = hip.HipDecoder(other, weights, capacity=64)
    s = Serving(backend, 61, count=4)
    try:
        def steps():
            decoder.set_position(0)
            decoder.decode(x, 6)
            tokens = decoder.generate(3).tolist()
            return tokens + hip.HipDecoder.generate_sessions([decoder], 3).reshape(-1).tolist() + [decoder.position]

        expected = steps()
        s.enqueue()
        backend.synchronize()
        results = s.results()
        graph, made = vp(), vp()
        assert run.hipStreamBeginCapture(vp(backend.stream), 2) == 0  # relaxed
        if order == "call first":
            s.enqueue()
        print("steps beside a capture", flush=True)
        assert steps() == expected
        if order == "step first":
            s.enqueue()
        assert run.hipStreamEndCapture(vp(backend.stream), ctypes.byref(graph)) == 0
        assert run.hipGraphInstantiate(ctypes.byref(made), graph, None, None, ctypes.c_size_t(0)) == 0
        for _ in range(3):
            s.clear()
            assert run.hipGraphLaunch(made, vp(backend.stream)) == 0
            backend.synchronize()
            assert same(results, s.results())
            assert steps() == expected
        run.hipGraphExecDestroy(made)
        run.hipGraphDestroy(graph)
    finally:
        decoder.close()
        other.close()
