"""Serving a batch of sequences that continue one prompt, on torch tensors
over the C ABI: attention over a shared prefix cache and per-sequence suffix
caches, the sums of the weight each key receives, and eviction by them.

The reference runs every continuation of a prompt (its steered and unsteered
branches, src/experiment/run.cpp:871-929) through a plan and a cache of its
own; here the prompt's cache is held and read once.  Every call only enqueues
work on torch's current stream of the tensors' device; wrong types, shapes and
strides raise ValueError, refusals of the library DolittleError.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import _lib
from ._lib import check, lib


def _cache(t, name: str, dims: int):
    """(row stride, outer stride) of a cache tensor [..., positions, heads, width]."""
    if t.dtype != torch.bfloat16 or t.dim() != dims or not t.is_cuda:
        raise ValueError(f"{name} must be a bfloat16 CUDA tensor of {dims} dimensions")
    s = t.stride()
    if (s[-1] != 1 and t.shape[-1] > 1) or (s[-2] != t.shape[-1] and t.shape[-2] > 1):
        raise ValueError(f"{name}: the heads of a position must be contiguous")
    row = t.shape[-1] * t.shape[-2]
    # A stride torch left arbitrary (one position, one cache) is not used.
    inner = s[-3] if t.shape[-3] > 1 else row
    return inner, (s[0] if dims == 4 and t.shape[0] > 1 else inner * t.shape[-3])


def _flat(t, name: str, dtype, shape, device):
    if t.dtype != dtype or tuple(t.shape) != tuple(shape) or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {tuple(shape)} on {device}")
    return t.data_ptr()


def _pair(key, value, name: str, dims: int, device):
    row, outer = _cache(key, f"{name}_key", dims)
    if value.shape != key.shape or value.device != device or key.device != device:
        raise ValueError(f"{name}_key and {name}_value must have one shape, on the query's device")
    if _cache(value, f"{name}_value", dims) != (row, outer):
        raise ValueError(f"{name}_key and {name}_value must have the same strides")
    return row, outer


def attention_shared(query, prefix_key, prefix_value, suffix_key, suffix_value, prefix_lengths, suffix_lengths, *,
                     prefix_weights=None, suffix_weights=None, out=None, lse=None):
    """Attention of `query` [B, rows, Hq, d] over the shared prefix cache
    [P, Hkv, d] and each sequence's suffix cache [B, S, Hkv, d]: sequence b's
    rows see prefix keys j < prefix_lengths[b], and row i suffix keys
    j < suffix_lengths[b] - (rows - 1 - i) (int64 tensors [B]).  Either side
    may be None.  Returns (out [B, rows, Hq, d] bfloat16, lse [B, rows, Hq]
    float32); a row without keys gives zeros and -inf.  prefix_weights
    [Hkv, P] and suffix_weights [B, Hkv, S] (float32) are added to: the softmax
    weight each key received from every row and query head."""
    if query.dtype != torch.bfloat16 or query.dim() != 4 or not query.is_cuda:
        raise ValueError("query must be a bfloat16 CUDA tensor [batch, rows, heads, width]")
    device = query.device
    batch, rows, heads, width = query.shape
    token, inner = heads * width, query.stride()
    stride = inner[1] if rows > 1 else inner[0] if batch > 1 else token
    if ((width > 1 and inner[3] != 1) or (heads > 1 and inner[2] != width) or
            (rows > 1 and batch > 1 and inner[0] != rows * stride)):
        raise ValueError("query: heads contiguous, one stride between tokens")
    a = _lib.SharedAttention(batch=batch, rows=rows, query_heads=heads, width=width, query_stride=stride)
    if prefix_key is not None:
        a.prefix_row_stride, _ = _pair(prefix_key, prefix_value, "prefix", 3, device)
        a.prefix_capacity, a.kv_heads = prefix_key.shape[0], prefix_key.shape[1]
        if prefix_key.shape[2] != width:
            raise ValueError("prefix caches must have the query's head width")
        a.prefix_key, a.prefix_value = prefix_key.data_ptr(), prefix_value.data_ptr()
        a.prefix_lengths = _flat(prefix_lengths, "prefix_lengths", torch.int64, (batch,), device)
    if suffix_key is not None:
        a.suffix_row_stride, a.suffix_sequence_stride = _pair(suffix_key, suffix_value, "suffix", 4, device)
        if suffix_key.shape[0] != batch or suffix_key.shape[3] != width or (
                prefix_key is not None and suffix_key.shape[2] != a.kv_heads):
            raise ValueError("suffix caches must be [batch, positions, the prefix's KV heads, the query's head width]")
        a.suffix_capacity, a.kv_heads = suffix_key.shape[1], suffix_key.shape[2]
        a.suffix_key, a.suffix_value = suffix_key.data_ptr(), suffix_value.data_ptr()
        a.suffix_lengths = _flat(suffix_lengths, "suffix_lengths", torch.int64, (batch,), device)
    if prefix_key is None and suffix_key is None:
        raise ValueError("a prefix or a suffix cache is required")
    pw = sw = None
    if prefix_weights is not None:
        pw = _flat(prefix_weights, "prefix_weights", torch.float32, (a.kv_heads, a.prefix_capacity), device)
    if suffix_weights is not None:
        sw = _flat(suffix_weights, "suffix_weights", torch.float32, (batch, a.kv_heads, a.suffix_capacity), device)
    if out is None:
        out = torch.empty((batch, rows, heads, width), dtype=torch.bfloat16, device=device)
    else:
        _flat(out, "out", torch.bfloat16, query.shape, device)
    if lse is None:
        lse = torch.empty((batch, rows, heads), dtype=torch.float32, device=device)
    else:
        _flat(lse, "lse", torch.float32, (batch, rows, heads), device)
    with torch.cuda.device(device):
        ref = C.byref(a)
        need = lib().dl_attention_shared_workspace_bytes(ref, pw is not None or sw is not None)
        if not need:
            raise _lib.DolittleError(_lib.DL_INVALID_ARGUMENT, lib().dl_last_error().decode())
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
        check(lib().dl_attention_shared(ref, query.data_ptr(), out.data_ptr(), lse.data_ptr(), pw, sw,
                                        workspace.data_ptr(), torch.cuda.current_stream().cuda_stream))
    return out, lse


def cache_evict(key, value, weights, positions, lengths, budget: int, *, first: int = 0, recent: int = 0, out=None):
    """Keep the min(length, budget) slots of every (cache, KV head) that were
    looked at most.  key/value [N, C, Hkv, d] bfloat16, weights [N, Hkv, C]
    float32, positions [N, Hkv, C] int32 (the token each slot holds), lengths
    [N] int64.  Protected slots (position < first, or above the head's largest
    position - recent) stay before any other; the rest by weight, largest
    first, ties to the lowest slot.  Kept slots below the new length stay in
    place, kept slots beyond it move into the vacated ones.  out = (key, value,
    weights, positions, lengths) receives the result, None evicts in place.
    Returns the five tensors that hold it."""
    device = key.device
    row, outer = _pair(key, value, "cache", 4, device)
    n, capacity, heads, width = key.shape
    e = _lib.CacheEviction(caches=n, kv_heads=heads, width=width, capacity=capacity, budget=budget, first=first,
                           recent=recent, row_stride=row, cache_stride=outer)
    e.key, e.value = key.data_ptr(), value.data_ptr()
    e.weights = _flat(weights, "weights", torch.float32, (n, heads, capacity), device)
    e.positions = _flat(positions, "positions", torch.int32, (n, heads, capacity), device)
    e.lengths = _flat(lengths, "lengths", torch.int64, (n,), device)
    if out is None:
        out = (key, value, weights, positions, lengths)
    key_out, value_out, weights_out, positions_out, lengths_out = out
    e.out_row_stride, e.out_cache_stride = _pair(key_out, value_out, "out", 4, device)
    room = key_out.shape[1]
    if tuple(key_out.shape) != (n, room, heads, width):
        raise ValueError("the output caches must be [caches, positions, heads, width] like the inputs")
    e.key_out, e.value_out, e.out_capacity = key_out.data_ptr(), value_out.data_ptr(), room
    e.weights_out = _flat(weights_out, "weights (output)", torch.float32, (n, heads, room), device)
    e.positions_out = _flat(positions_out, "positions (output)", torch.int32, (n, heads, room), device)
    e.lengths_out = _flat(lengths_out, "lengths (output)", torch.int64, (n,), device)
    with torch.cuda.device(device):
        ref = C.byref(e)
        need = lib().dl_cache_evict_workspace_bytes(ref)
        if not need:
            raise _lib.DolittleError(_lib.DL_INVALID_ARGUMENT, lib().dl_last_error().decode())
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
        check(lib().dl_cache_evict(ref, workspace.data_ptr(), torch.cuda.current_stream().cuda_stream))
    return out
