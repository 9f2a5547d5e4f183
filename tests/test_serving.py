"""Refusals and sizes of the serving operators that need no device: the
*_workspace calls check a descriptor as the device calls do."""
import ctypes
import os
from types import SimpleNamespace

import numpy as np
import pytest

from funasrnet_amd import hip


def packed(**changes):
    a = hip.PackedAttention(query_row=2048, query_head=128, key_row=1024, key_head=128, value_row=1024, value_head=128,
                            output_row=2048, output_head=128, sequences=3, query_rows=100, key_rows=120, longest_query=50,
                            longest_key=60, heads=16, kv_heads=8, head_size=128, query_type=hip.TYPE_F32,
                            cache_type=hip.TYPE_F16, scale=0.1)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


def prefix(**changes):
    a = hip.PrefixAttention(query_sequence=2048, query_head=128, prefix_key_row=128, prefix_key_head=128 * 500,
                            prefix_value_row=128, prefix_value_head=128 * 500, key_sequence=1 << 20, key_row=128,
                            key_head=1 << 17, value_sequence=1 << 20, value_row=128, value_head=1 << 17,
                            output_sequence=2048, output_head=128, sequences=5, prefix=500, capacity=1024, longest=700,
                            heads=16, kv_heads=8, head_size=128, query_type=hip.TYPE_F32, cache_type=hip.TYPE_F16, scale=0.1)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


def logits(**changes):
    a = hip.LogitsAdjust(logits_stride=1000, output_stride=1000, rows=4, vocab=1000, type=hip.TYPE_F32, tokens=16)
    for name, value in changes.items():
        setattr(a, name, value)
    return a


CALLS = {"packed": ("fah_attention_packed", packed), "prefix": ("fah_attention_prefix", prefix),
         "logits": ("fah_logits_adjust", logits)}


def workspace(kind, **changes):
    name, make = CALLS[kind]
    v = ctypes.c_int64(-7)
    rc = getattr(hip.load(), name + "_workspace")(ctypes.byref(make(**changes)), ctypes.byref(v))
    return rc, v.value


@pytest.mark.parametrize("kind", CALLS)
def test_workspace_is_given(kind):
    rc, n = workspace(kind)
    assert rc == hip.OK and n >= 0


@pytest.mark.parametrize("kind", CALLS)
def test_null_arguments(kind):
    lib, (name, make) = hip.load(), CALLS[kind]
    v = ctypes.c_int64()
    assert getattr(lib, name + "_workspace")(None, ctypes.byref(v)) == hip.ERROR_ARGUMENT
    assert getattr(lib, name + "_workspace")(ctypes.byref(make()), None) == hip.ERROR_ARGUMENT
    assert getattr(lib, name + "_device")(None, ctypes.byref(make())) == hip.ERROR_ARGUMENT


@pytest.mark.parametrize("kind,changes", [
    ("packed", dict(sequences=-1)), ("packed", dict(query_rows=-1)), ("packed", dict(key_rows=-1)),
    ("packed", dict(longest_query=-1)), ("packed", dict(longest_key=-1)), ("packed", dict(heads=0)),
    ("packed", dict(kv_heads=0)), ("packed", dict(kv_heads=3)), ("packed", dict(head_size=0)), ("packed", dict(scale=0.0)),
    ("packed", dict(scale=-1.0)), ("packed", dict(scale=float("nan"))), ("packed", dict(scale=float("inf"))),
    ("packed", dict(query_rows=2**31 - 1)), ("packed", dict(sequences=2**31 - 1)), ("packed", dict(key_rows=2**31 - 1)),
    ("prefix", dict(prefix=2**31 - 1)), ("prefix", dict(capacity=2**31 - 1)),
    ("prefix", dict(sequences=-1)), ("prefix", dict(prefix=-1)), ("prefix", dict(capacity=-1)), ("prefix", dict(longest=-1)),
    ("prefix", dict(heads=15)), ("prefix", dict(kv_heads=-8)), ("prefix", dict(scale=0.0)),
    ("prefix", dict(sequences=2**31 - 1)),
    ("logits", dict(rows=-1)), ("logits", dict(vocab=-1)), ("logits", dict(rows=70000)), ("logits", dict(history_capacity=-1)),
    ("logits", dict(bias_capacity=-1)), ("logits", dict(mask_rows=-1)), ("logits", dict(vocab=2**31 - 1)),
])
def test_invalid_sizes_are_errors(kind, changes):
    rc, n = workspace(kind, **changes)
    assert rc == hip.ERROR_ARGUMENT and n == -7
    assert hip.load().fah_last_error()


@pytest.mark.parametrize("kind,changes", [
    ("packed", dict(head_size=12)), ("packed", dict(head_size=136)), ("packed", dict(query_type=hip.TYPE_F32, cache_type=0)),
    ("packed", dict(query_type=hip.TYPE_F16, cache_type=hip.TYPE_BF16)), ("packed", dict(query_type=7)),
    ("packed", dict(query_row=2046)), ("packed", dict(output_head=130)), ("packed", dict(key_row=1028)),
    ("packed", dict(value_head=-128)), ("packed", dict(key_row=(1 << 25) + 8)), ("packed", dict(heads=65544, kv_heads=8)),
    ("prefix", dict(value_row=(1 << 25) + 8)),
    ("prefix", dict(head_size=100)), ("prefix", dict(cache_type=hip.TYPE_BF16)), ("prefix", dict(prefix_key_row=132)),
    ("prefix", dict(key_sequence=(1 << 20) + 4)), ("prefix", dict(query_head=2)), ("prefix", dict(output_sequence=-2048)),
    ("logits", dict(type=3)), ("logits", dict(type=-1)),
])
def test_unsupported_forms_are_declined(kind, changes):
    rc, n = workspace(kind, **changes)
    assert rc == hip.DECLINED and n == -7


@pytest.mark.parametrize("kind,size", [("packed", "key_rows"), ("prefix", "prefix"), ("prefix", "capacity")])
def test_keys_whose_shares_end_past_32_bits(kind, size):
    """256 shares of 2^31 - 4097 keys in tiles of 128 are 65536 tiles each: the last one's end, 2^31, is no 32-bit number."""
    keys = 2**31 - 4097
    tiles = -(-keys // 128)
    assert -(-tiles // 256) * 128 * 256 == 2**31
    rc, _ = workspace(kind, **{size: keys, "longest_key" if kind == "packed" else "longest": keys})
    assert rc == hip.ERROR_ARGUMENT and b"keys" in hip.load().fah_last_error()
    keys = 2**31 - 2**19 - 1
    rc, _ = workspace(kind, **{size: keys, "longest_key" if kind == "packed" else "longest": keys})
    assert rc == hip.OK


def test_choose_arguments(monkeypatch):
    """HipDecoder.choose: masks that are lists, logits that are not contiguous, and refusals ahead of the library's call."""
    seen = {}

    class Library:
        @staticmethod
        def fah_decoder_choose(handle, history, count, prompt, repetition, presence, frequency, tokens, values, biases, mask, out, token):
            seen["mask"] = None if mask is None else [mask[0], mask[1]]
            for i in range(40 if out is not None else 0):
                out[i] = i + 0.5
            token._obj.value = 7
            return hip.OK

    monkeypatch.setattr(hip, "load", lambda: Library)
    decoder = object.__new__(hip.HipDecoder)
    decoder.handle, decoder.config = 1, SimpleNamespace(vocab=40)
    allowed = [i % 3 == 0 for i in range(40)]
    assert decoder.choose([1, 2], mask=allowed) == 7
    assert seen["mask"] == [sum(1 << i for i in range(0, 32, 3)), sum(1 << (i - 32) for i in range(33, 40, 3))]
    wide = np.zeros((40, 2), np.float32)
    assert decoder.choose(logits=wide[:, 1]) == 7
    assert np.array_equal(wide[:, 1], np.arange(40) + 0.5) and np.all(wide[:, 0] == 0)
    fixed = np.zeros(40, np.float32)
    fixed.flags.writeable = False
    seen.clear()
    for bad in (dict(logits=fixed), dict(logits=np.zeros(40)), dict(logits=np.zeros(39, np.float32)), dict(mask=allowed[:39]),
                dict(mask=np.ones((1, 40), bool))):
        with pytest.raises(ValueError):
            decoder.choose(**bad)
    assert not seen and np.all(fixed == 0)
    decoder.handle = None  # nothing to destroy


def test_choose_is_reached_from_csharp():
    """The binding's import has a caller, which the core's interface names."""
    folder = os.path.join(os.path.dirname(hip.__file__), "csharp")
    step = open(os.path.join(folder, "FunAsrNet.Hip", "HipDecoderStep.cs")).read()
    core = open(os.path.join(folder, "FunAsrNet.CorePatch", "IDecoderStepBackend.cs")).read()
    assert "Native.fah_decoder_choose(Handle" in step and "public int Choose(TokenRules rules, float[]? logits)" in step
    assert "int Choose(TokenRules rules, float[]? logits);" in core
