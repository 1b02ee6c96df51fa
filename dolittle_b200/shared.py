"""Serving a batch of sequences that continue one prompt, on torch tensors
over the C ABI: attention over a shared prefix cache and per-sequence suffix
caches, the sums of the weight each key receives, and eviction by them.

The reference runs every continuation of a prompt (its steered and unsteered
branches, src/experiment/run.cpp:871-929) through a plan and a cache of its
own; here the prompt's cache is held and read once.  Every call only enqueues
work on torch's current stream of the tensors' device; wrong types, shapes and
strides raise ValueError, refusals of the library DolittleError.  Nothing here
is recorded for gradients.
"""
from __future__ import annotations

import ctypes as C
import importlib.machinery
import importlib.util
import os

import torch  # noqa: F401  (its libraries must be loaded before the extension's)

from . import _lib
from ._lib import lib

_calls = None


def _extension():
    """The in-tree extension module that checks the tensors and makes the calls."""
    global _calls
    if _calls is None:
        path = _lib.torch_calls_path()
        if not os.path.exists(path):
            raise ImportError(f"{path} is missing: run `python -m dolittle_b200.build`")
        spec = importlib.util.spec_from_loader(
            "dolittle_b200._torch_shared", importlib.machinery.ExtensionFileLoader("dolittle_b200._torch_shared", path))
        module = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(module)
        functions = ("dl_attention_shared_workspace_bytes", "dl_attention_shared", "dl_cache_evict_workspace_bytes",
                     "dl_cache_evict", "dl_last_error")
        module.bind(*[C.cast(getattr(lib(), f), C.c_void_p).value for f in functions], _lib.DolittleError)
        _calls = module
    return _calls


def attention_shared(query, prefix_key, prefix_value, suffix_key, suffix_value, prefix_lengths, suffix_lengths, *,
                     prefix_weights=None, suffix_weights=None, out=None, lse=None):
    """Attention of `query` [B, rows, Hq, d] over the shared prefix cache
    [P, Hkv, d] and each sequence's suffix cache [B, S, Hkv, d]: sequence b's
    rows see prefix keys j < prefix_lengths[b], and row i suffix keys
    j < suffix_lengths[b] - (rows - 1 - i) (int64 tensors [B]).  Either side
    may be None.  Returns (out [B, rows, Hq, d] bfloat16, lse [B, rows, Hq]
    float32); a row without keys gives zeros and -inf.  prefix_weights
    [Hkv, P] and suffix_weights [B, Hkv, S] (float32) are added to: the softmax
    weight each key received from every row and query head.  The query's tokens
    lie apart, and `out` shares no memory with them; one suffix may be expanded
    over the batch.  The work is cut by the caches' sizes P and S, whatever the
    lengths: a cache far larger than what it holds costs time."""
    return (_calls or _extension()).attention_shared(query, prefix_key, prefix_value, suffix_key, suffix_value,
                                                     prefix_lengths, suffix_lengths, prefix_weights, suffix_weights,
                                                     out, lse)


def cache_evict(key, value, weights, positions, lengths, budget: int, *, first: int = 0, recent: int = 0, out=None):
    """Keep the min(length, budget) slots of every (cache, KV head) that were
    looked at most.  key/value [N, C, Hkv, d] bfloat16, weights [N, Hkv, C]
    float32, positions [N, Hkv, C] int32 (the token each slot holds), lengths
    [N] int64.  Protected slots (position < first, or above the head's largest
    position - recent) stay before any other; the rest by weight, largest
    first, ties to the lowest slot.  Kept slots below the new length stay in
    place, kept slots beyond it move into the vacated ones.  out = (key, value,
    weights, positions, lengths) receives the result, None evicts in place.
    Returns the five tensors that hold it, rows that are written apart from one
    another."""
    return (_calls or _extension()).cache_evict(key, value, weights, positions, lengths, budget, first, recent, out)
