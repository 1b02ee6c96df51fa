"""Refusals of the shared-prefix operators through the C ABI: all before any
device is touched, each with its reason.  The pointers are never read."""
import ctypes as C

import pytest

import dolittle_b200 as dl
from dolittle_b200 import _lib

P = 1 << 20  # a plausible, aligned address


def attention(**change):
    a = _lib.SharedAttention(4, 1, 32, 8, 128, 0, 0, P, P, 100, 1024, P, P, P, 50, 1024, 51200, P)
    for k, v in change.items():
        setattr(a, k, v)
    return a


def eviction(**change):
    e = _lib.CacheEviction(2, 8, 128, 100, 50, 4, 8, P, P, 1024, 102400, P, P, P, P, P, 100, 1024, 102400, P, P, P)
    for k, v in change.items():
        setattr(e, k, v)
    return e


ATTENTION = [
    (dict(batch=0), _lib.DL_INVALID_ARGUMENT, b"empty"),
    (dict(rows=0), _lib.DL_INVALID_ARGUMENT, b"empty"),
    (dict(kv_heads=0), _lib.DL_INVALID_ARGUMENT, b"empty"),
    (dict(width=96), _lib.DL_UNSUPPORTED, b"width"),
    (dict(query_heads=30), _lib.DL_UNSUPPORTED, b"query heads"),
    (dict(query_heads=8 * 65), _lib.DL_UNSUPPORTED, b"group"),
    (dict(query_stride=4095), _lib.DL_UNSUPPORTED, b"stride"),
    (dict(query_stride=4088), _lib.DL_UNSUPPORTED, b"stride"),
    (dict(output_stride=12), _lib.DL_UNSUPPORTED, b"stride"),
    (dict(prefix_key=None), _lib.DL_INVALID_ARGUMENT, b"prefix"),
    (dict(prefix_lengths=None), _lib.DL_INVALID_ARGUMENT, b"prefix"),
    (dict(prefix_value=P + 8), _lib.DL_UNSUPPORTED, b"aligned"),
    (dict(prefix_row_stride=1023), _lib.DL_UNSUPPORTED, b"prefix rows"),
    (dict(prefix_row_stride=1016), _lib.DL_UNSUPPORTED, b"prefix rows"),
    (dict(suffix_value=None), _lib.DL_INVALID_ARGUMENT, b"suffix"),
    (dict(suffix_lengths=None), _lib.DL_INVALID_ARGUMENT, b"suffix"),
    (dict(suffix_sequence_stride=51201), _lib.DL_UNSUPPORTED, b"suffix rows"),
    (dict(batch=1 << 17), _lib.DL_UNSUPPORTED, b"out of range"),
    (dict(rows=1 << 40), _lib.DL_UNSUPPORTED, b"out of range"),
    (dict(prefix_capacity=1 << 40), _lib.DL_UNSUPPORTED, b"out of range"),
]


@pytest.mark.parametrize("change,status,reason", ATTENTION)
def test_attention_refusals(change, status, reason):
    L = dl.lib()
    a = attention(**change)
    assert L.dl_attention_shared(C.byref(a), P, P, None, None, None, P, None) == status
    assert reason in L.dl_last_error()
    assert L.dl_attention_shared_workspace_bytes(C.byref(a), 1) == 0


def test_attention_refuses_null_and_misaligned_pointers():
    L = dl.lib()
    a = C.byref(attention())
    assert L.dl_attention_shared(None, P, P, None, None, None, P, None) == _lib.DL_INVALID_ARGUMENT
    for query, out, workspace in ((None, P, P), (P, None, P), (P, P, None)):
        assert L.dl_attention_shared(a, query, out, None, None, None, workspace, None) == _lib.DL_INVALID_ARGUMENT
    for query, out, workspace in ((P + 2, P, P), (P, P + 8, P), (P, P, P + 16)):
        assert L.dl_attention_shared(a, query, out, None, None, None, workspace, None) == _lib.DL_UNSUPPORTED


def test_workspace_grows_with_the_call_and_its_weights():
    L = dl.lib()
    sizes = [L.dl_attention_shared_workspace_bytes(C.byref(attention(batch=b, prefix_capacity=p)), w)
             for b, p, w in ((2, 64, 0), (32, 8192, 0), (32, 8192, 1))]
    assert 0 < sizes[0] < sizes[1] < sizes[2]
    assert L.dl_cache_evict_workspace_bytes(C.byref(eviction())) == 2 * 8 * (3 * 50 + 1) * 4


EVICTION = [
    (dict(caches=0), _lib.DL_INVALID_ARGUMENT, b"empty"),
    (dict(budget=0), _lib.DL_INVALID_ARGUMENT, b"empty"),
    (dict(first=30, recent=21), _lib.DL_INVALID_ARGUMENT, b"first + recent"),
    (dict(recent=1 << 63), _lib.DL_INVALID_ARGUMENT, b"first + recent"),
    (dict(out_capacity=49), _lib.DL_INVALID_ARGUMENT, b"capacity"),
    (dict(width=100), _lib.DL_UNSUPPORTED, b"multiples of 8"),
    (dict(row_stride=1025), _lib.DL_UNSUPPORTED, b"multiples of 8"),
    (dict(row_stride=1016), _lib.DL_UNSUPPORTED, b"row stride"),
    (dict(capacity=1 << 23), _lib.DL_UNSUPPORTED, b"slots"),
    (dict(caches=1 << 40), _lib.DL_UNSUPPORTED, b"out of range"),
    (dict(key=None), _lib.DL_INVALID_ARGUMENT, b"null"),
    (dict(lengths_out=None), _lib.DL_INVALID_ARGUMENT, b"null"),
    (dict(value_out=P + 8), _lib.DL_UNSUPPORTED, b"aligned"),
    (dict(out_capacity=60), _lib.DL_INVALID_ARGUMENT, b"in place"),
    (dict(key_out=P + 1024), _lib.DL_INVALID_ARGUMENT, b"overlap"),
    (dict(weights_out=P + 64), _lib.DL_INVALID_ARGUMENT, b"overlap"),
]


@pytest.mark.parametrize("change,status,reason", EVICTION)
def test_eviction_refusals(change, status, reason):
    L = dl.lib()
    e = eviction(**change)
    assert L.dl_cache_evict(C.byref(e), P, None) == status
    assert reason in L.dl_last_error()


def test_torch_calls_are_built_and_check_their_arguments():
    import torch

    from dolittle_b200 import shared
    assert shared._extension() is shared._extension()
    t = torch.zeros(1, 1, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        shared.attention_shared(t, t[0], t[0], t, t, None, None)
    with pytest.raises(ValueError, match="tensor"):
        shared.attention_shared(None, None, None, None, None, None, None)
    with pytest.raises(ValueError, match="CUDA"):
        shared.cache_evict(t, t, None, None, None, 1)
