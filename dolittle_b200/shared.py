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
import functools

import torch

from . import _lib
from ._lib import check, lib

_BF16, _F32, _I32, _I64 = torch.bfloat16, torch.float32, torch.int32, torch.int64
# The stream's address without building a Stream object (a decode step makes
# one call per block).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream",
                      lambda device: torch.cuda.current_stream(device).cuda_stream)


def _pair(key, value, name: str, dims: int, device: int):
    """(shape, row stride, outer stride) of key and value caches [..., positions, heads, width]."""
    shape, stride = key.shape, key.stride()
    if (key.dtype is not _BF16 or value.dtype is not _BF16 or len(shape) != dims or value.shape != shape or
            key.get_device() != device or value.get_device() != device):
        raise ValueError(f"{name}_key and {name}_value must be bfloat16 tensors of one shape and {dims} dimensions, "
                         "on the query's device")
    width, heads, positions = shape[-1], shape[-2], shape[-3]
    # torch leaves the stride of a dimension of size 1 arbitrary; it is not used.
    row = stride[-3] if positions > 1 else heads * width
    outer = stride[0] if dims == 4 and shape[0] > 1 else row * positions
    if (stride[-1] != 1 and width > 1) or (stride[-2] != width and heads > 1):
        raise ValueError(f"{name}_key: the heads of a position must be contiguous")
    if value.stride() != stride and any(a != b for a, b, n in zip(value.stride(), stride, shape) if n > 1):
        raise ValueError(f"{name}_key and {name}_value must have the same strides")
    return shape, row, outer


def _flat(t, name: str, dtype, shape: tuple, device: int) -> int:
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} tensor {tuple(shape)} on the query's device")
    return t.data_ptr()


def _on(device: int, call):
    """call(stream) with `device` current."""
    if torch.cuda.current_device() == device:
        return check(call(_raw_stream(device)))
    with torch.cuda.device(device):
        return check(call(_raw_stream(device)))


@functools.lru_cache(maxsize=512)
def _attention_workspace(device: int, batch, rows, heads, kv_heads, width, prefix, suffix, weights: bool) -> int:
    # The size depends on the shapes alone; the pointers only have to be plausible here.
    a = _lib.SharedAttention(batch, rows, heads, kv_heads, width, 0, 0, 16, 16, prefix, kv_heads * width, 16, 16, 16,
                             suffix, kv_heads * width, kv_heads * width * suffix, 16)
    with torch.cuda.device(device):
        return lib().dl_attention_shared_workspace_bytes(C.byref(a), weights)


@functools.lru_cache(maxsize=512)
def _evict_workspace(device: int, caches, kv_heads, width, capacity, budget) -> int:
    e = _lib.CacheEviction(caches=caches, kv_heads=kv_heads, width=width, capacity=capacity, budget=budget,
                           row_stride=kv_heads * width, out_row_stride=kv_heads * width, out_capacity=capacity)
    with torch.cuda.device(device):
        return lib().dl_cache_evict_workspace_bytes(C.byref(e))


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
    shape, inner, device = query.shape, query.stride(), query.get_device()
    if query.dtype is not _BF16 or len(shape) != 4 or device < 0:
        raise ValueError("query must be a bfloat16 CUDA tensor [batch, rows, heads, width]")
    batch, rows, heads, width = shape
    stride = inner[1] if rows > 1 else inner[0] if batch > 1 else heads * width
    if ((inner[3] != 1 and width > 1) or (inner[2] != width and heads > 1) or
            (rows > 1 and batch > 1 and inner[0] != rows * stride)):
        raise ValueError("query: heads contiguous, one stride between tokens")
    kv_heads = pk = pv = pl = sk = sv = sl = None
    prefix = p_row = suffix = s_row = s_seq = 0
    if prefix_key is not None:
        (prefix, kv_heads, w), p_row, _ = _pair(prefix_key, prefix_value, "prefix", 3, device)
        if w != width:
            raise ValueError("prefix caches must have the query's head width")
        pk, pv = prefix_key.data_ptr(), prefix_value.data_ptr()
        pl = _flat(prefix_lengths, "prefix_lengths", _I64, (batch,), device)
    if suffix_key is not None:
        (n, suffix, h, w), s_row, s_seq = _pair(suffix_key, suffix_value, "suffix", 4, device)
        if n != batch or w != width or (kv_heads is not None and h != kv_heads):
            raise ValueError("suffix caches must be [batch, positions, the prefix's KV heads, the query's head width]")
        kv_heads = h
        sk, sv = suffix_key.data_ptr(), suffix_value.data_ptr()
        sl = _flat(suffix_lengths, "suffix_lengths", _I64, (batch,), device)
    if kv_heads is None:
        raise ValueError("a prefix or a suffix cache is required")
    pw = sw = None
    if prefix_weights is not None:
        pw = _flat(prefix_weights, "prefix_weights", _F32, (kv_heads, prefix), device)
    if suffix_weights is not None:
        sw = _flat(suffix_weights, "suffix_weights", _F32, (batch, kv_heads, suffix), device)
    if out is None:
        out = torch.empty(shape, dtype=_BF16, device=query.device)
    else:
        _flat(out, "out", _BF16, shape, device)
    if lse is None:
        lse = torch.empty((batch, rows, heads), dtype=_F32, device=query.device)
    else:
        _flat(lse, "lse", _F32, (batch, rows, heads), device)
    a = _lib.SharedAttention(batch, rows, heads, kv_heads, width, stride, 0, pk, pv, prefix, p_row, pl, sk, sv, suffix,
                             s_row, s_seq, sl)
    # 0 when the library refuses the shape: the call below then says why.
    need = _attention_workspace(device, batch, rows, heads, kv_heads, width, prefix, suffix,
                                pw is not None or sw is not None)
    workspace = torch.empty(need, dtype=torch.uint8, device=query.device)
    _on(device, lambda stream: lib().dl_attention_shared(C.byref(a), query.data_ptr(), out.data_ptr(), lse.data_ptr(),
                                                         pw, sw, workspace.data_ptr(), stream))
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
    device = key.get_device()
    if device < 0:
        raise ValueError("the caches must be CUDA tensors")
    (n, capacity, heads, width), row, outer = _pair(key, value, "cache", 4, device)
    if out is None:
        out = (key, value, weights, positions, lengths)
        room, out_row, out_outer = capacity, row, outer
    else:
        (m, room, h, w), out_row, out_outer = _pair(out[0], out[1], "out", 4, device)
        if m != n or h != heads or w != width:
            raise ValueError("the output caches must be [caches, positions, heads, width] like the inputs")
    slots, out_slots = (n, heads, capacity), (n, heads, room)
    if budget < 0 or first < 0 or recent < 0:
        raise ValueError("budget, first and recent must not be negative")
    e = _lib.CacheEviction(n, heads, width, capacity, budget, first, recent, key.data_ptr(), value.data_ptr(), row,
                           outer, _flat(weights, "weights", _F32, slots, device),
                           _flat(positions, "positions", _I32, slots, device),
                           _flat(lengths, "lengths", _I64, (n,), device), out[0].data_ptr(), out[1].data_ptr(), room,
                           out_row, out_outer, _flat(out[2], "weights (output)", _F32, out_slots, device),
                           _flat(out[3], "positions (output)", _I32, out_slots, device),
                           _flat(out[4], "lengths (output)", _I64, (n,), device))
    need = _evict_workspace(device, n, heads, width, capacity, budget)
    workspace = torch.empty(need, dtype=torch.uint8, device=key.device)
    _on(device, lambda stream: lib().dl_cache_evict(C.byref(e), workspace.data_ptr(), stream))
    return out
