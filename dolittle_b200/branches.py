"""Continuations of one prompt, decoded together: the prompt's keys and values
stay where an Engine's prompt pass left them and are read once per step for the
whole batch; every branch holds only what came after.

The reference runs each continuation through a plan and a cache of its own
(steered and unsteered branches, src/experiment/run.cpp:871-929; sixteen
verbalizer samples of one prefix).  A step here is the engine's block recipe
(src/models/qwen3/model.cpp:343-409) on the engine's own weights, with
`shared.attention_shared` for its attention; with `weights=True` every step
also sums the weight each key receives, and `evict_prefix` / `evict_suffix` cut
the caches by those sums (`shared.cache_evict`).

The branches go in lockstep: one length for all, the whole prompt for each, and
no steering (the batched server steers).  Batches whose sequences differ in
length, or leave the prompt at different tokens, call `attention_shared` with
lengths of their own.  A step launches about twenty kernels a block from
Python, which bounds it: with the Qwen3-8B shapes 16 branches of a 2048-token
prompt take 6.6 ms a step (5.4 on the device; the server with its full caches
4.7), 32 of 8192 tokens 6.9 ms (the server 10.6).

    engine.consume_view(prompt, dl.DL_PREFILL_FAST)
    branches = Branches(engine, batch=16, capacity=128)
    logits = branches.step(tokens)             # [16, rows] ids -> [16, V]
"""
from __future__ import annotations

import torch

from . import _lib, shared
from ._lib import check, lib
from .engine import Engine

_BF16, _F32 = torch.bfloat16, torch.float32


class _Device:
    """Device memory that something else owns, for torch.as_tensor."""

    def __init__(self, pointer: int, shape: tuple, owner):
        self.owner = owner
        self.__cuda_array_interface__ = {"data": (pointer, False), "shape": shape, "typestr": "<i2", "version": 3}


class Branches:
    """`batch` sequences that continue what `engine` has consumed so far, in
    lockstep; each may grow by `capacity` tokens.  The engine's cache is read in
    place: it must not be reset or extended while branches use it (until
    `evict_prefix` has made a copy), and the engine, whose weights they use,
    stays open.  Head width 64 or 128, other widths as the
    tensor-core projections want them (hidden a multiple of 64, projections a
    multiple of 128 rows)."""

    def __init__(self, engine: Engine, batch: int, capacity: int, weights: bool = False):
        c = engine.config
        if engine.position < 1 or batch < 1 or capacity < 1:
            raise ValueError("a consumed prompt, a batch and a capacity are required")
        self.engine, self.config, self.batch, self.capacity = engine, c, batch, capacity
        self.prefix, self.position, self.length = engine.position, engine.position, 0
        d = c.head_width

        def cache(layer, values):
            pointer, stride = engine.kv_device(layer, values)
            rows = torch.as_tensor(_Device(pointer, (self.prefix, stride), engine)).view(_BF16)
            return rows.view(self.prefix, c.kv_heads, d)

        self._device = dev = cache(0, False).device  # the engine's, whichever is current
        self._prefix = [(cache(i, False), cache(i, True)) for i in range(c.layers)]
        kv = (c.layers, batch, capacity, c.kv_heads, d)
        self._suffix_key, self._suffix_value = torch.zeros(kv, dtype=_BF16, device=dev), torch.zeros(kv, dtype=_BF16,
                                                                                                  device=dev)
        self._prefix_lengths = torch.full((batch,), self.prefix, dtype=torch.int64, device=dev)
        self._suffix_lengths = torch.zeros(batch, dtype=torch.int64, device=dev)
        self._unknown = torch.zeros(batch, dtype=torch.bool, device=dev)  # branches that were given unknown ids
        self._next = torch.full((1,), self.position, dtype=torch.int64, device=dev)  # position of the next token
        self.prefix_weights = self.suffix_weights = None
        if weights:
            self.prefix_weights = [torch.zeros(c.kv_heads, self.prefix, device=dev) for _ in range(c.layers)]
            self.suffix_weights = torch.zeros(c.layers, batch, c.kv_heads, capacity, device=dev)
            # The token that each slot holds: evictions move slots, not positions.
            slots = torch.arange(self.prefix, dtype=torch.int32, device=dev)
            self._prefix_positions = [slots.expand(1, c.kv_heads, -1).contiguous() for _ in range(c.layers)]
            self._suffix_positions = torch.zeros(c.layers, batch, c.kv_heads, capacity, dtype=torch.int32, device=dev)
        self._weight = [engine.tensor_device(i)[0] for i in range(c.tensor_count())]
        q, k, v = (self._weight[3 + role] for role in (1, 2, 3))
        if k - q != 2 * c.query_heads * d * c.hidden or v - k != 2 * c.kv_heads * d * c.hidden:
            raise ValueError("the engine's q, k and v weights must be one matrix")
        self._scratch = None

    def _open(self):
        """The weights are the engine's, and so is the prompt's cache at first."""
        if not self.engine._h:
            raise ValueError("the branches' engine is closed")

    # ---- one step ----------------------------------------------------------
    def step(self, tokens) -> torch.Tensor:
        """The next tokens of every branch, [batch, rows] (or [batch]) ids;
        returns the last row's logits, [batch, V] BF16.  Ids outside the
        vocabulary raise ValueError where the host has them; on the device they
        are not waited for, and their branch's logits are NaN from there on."""
        self._open()
        tokens = torch.as_tensor(tokens).to(torch.int64)
        tokens = tokens if tokens.dim() == 2 else tokens[:, None]
        batch, rows = tokens.shape
        if batch != self.batch or rows < 1 or self.length + rows > self.capacity:
            raise ValueError("tokens must be [batch, rows] and fit the capacity")
        unknown = (tokens < 0) | (tokens >= self.config.vocabulary)
        if tokens.is_cuda:  # the embedding's rows are read as the ids say
            self._unknown |= unknown.any(1)
            tokens = tokens.masked_fill(unknown, 0)
        elif bool(unknown.any()):
            raise ValueError("token ids must be below the vocabulary's size")
        tokens = tokens.to(self._device, torch.int32).contiguous()
        with torch.cuda.device(self._device):
            return self._step(tokens, batch, rows)

    def _step(self, tokens, batch: int, rows: int) -> torch.Tensor:
        c, d = self.config, self.config.head_width
        stream = torch.cuda.current_stream().cuda_stream
        q_width, kv_width, m = c.query_heads * d, c.kv_heads * d, batch * rows
        new = dict(dtype=_BF16, device=self._device)
        x = torch.empty((m, c.hidden), **new)
        check(lib().dl_embedding(_lib.DL_BF16, tokens.data_ptr(), self._weight[0], x.data_ptr(), m, c.hidden, stream))
        normed = torch.empty_like(x)
        qkv = torch.empty((m, q_width + 2 * kv_width), **new)
        hidden = torch.empty((m, c.mlp_width), **new)
        attended = torch.empty((batch, rows, c.query_heads, d), **new)
        lse = torch.empty((batch, rows, c.query_heads), dtype=_F32, device=self._device)
        slots = self._suffix_lengths[:1] + torch.arange(rows, device=self._device)
        self._suffix_lengths += rows
        if self.suffix_weights is not None:
            at = (self._next + torch.arange(rows, device=self._device)).to(torch.int32)
            self._suffix_positions.index_copy_(3, slots, at.expand(*self._suffix_positions.shape[:3], rows))
            self.suffix_weights.index_fill_(3, slots, 0.0)
        for layer in range(c.layers):
            w = self._weight[3 + 11 * layer:14 + 11 * layer]
            self._norm(x, w[0], normed, m, c.hidden, stream)
            self._project(normed, w[1], qkv, q_width + 2 * kv_width, c.hidden, 0, stream)
            q = self._rotate(qkv[:, :q_width], w[4], batch, rows, c.query_heads, stream)
            k = self._rotate(qkv[:, q_width:q_width + kv_width], w[5], batch, rows, c.kv_heads, stream)
            self._suffix_key[layer].index_copy_(1, slots, k)
            self._suffix_value[layer].index_copy_(1, slots, qkv[:, q_width + kv_width:].reshape(k.shape))
            shared.attention_shared(
                q, *self._prefix[layer], self._suffix_key[layer], self._suffix_value[layer], self._prefix_lengths,
                self._suffix_lengths, out=attended, lse=lse,
                prefix_weights=None if self.prefix_weights is None else self.prefix_weights[layer],
                suffix_weights=None if self.suffix_weights is None else self.suffix_weights[layer])
            self._project(attended.view(m, q_width), w[6], x, c.hidden, q_width, 1, stream)
            self._norm(x, w[7], normed, m, c.hidden, stream)
            self._project(normed, w[8], hidden, 2 * c.mlp_width, c.hidden, 3, stream)  # gate and up rows interleaved
            self._project(hidden, w[10], x, c.hidden, c.mlp_width, 1, stream)
        self._next += rows
        self.position += rows
        self.length += rows
        last = x.view(batch, rows, c.hidden)[:, -1].contiguous()
        self._norm(last, self._weight[1], normed, batch, c.hidden, stream)
        logits = torch.empty((batch, c.vocabulary), **new)
        self._project(normed[:batch], self._weight[2], logits, c.vocabulary, c.hidden, 0, stream)
        return logits.masked_fill_(self._unknown[:, None], float("nan"))

    def _norm(self, x, weight, out, rows, width, stream):
        check(lib().dl_rms_norm(_lib.DL_BF16, x.data_ptr(), weight, out.data_ptr(), rows, width, self.config.epsilon,
                                stream))

    def _project(self, x, weight, out, n, k, epilogue, stream):
        """out = epilogue(x W^T); few rows as a split-K product."""
        m = x.shape[0]
        if m > 32:
            check(lib().dl_gemm_bf16(x.data_ptr(), k, weight, out.data_ptr(), out.shape[1], m, n, k, epilogue, stream))
            return
        need = lib().dl_gemm_bf16_parts_workspace_bytes(m, n, k, 0)
        if self._scratch is None or self._scratch.numel() < need:
            self._scratch = torch.empty(need, dtype=torch.uint8, device=self._device)
        check(lib().dl_gemm_bf16_parts(x.data_ptr(), k, weight, out.data_ptr(), out.shape[1], m, n, k, epilogue, 0,
                                       self._scratch.data_ptr(), stream))

    def _rotate(self, x, norm, batch, rows, heads, stream):
        """QK-norm and rotary embedding of [batch * rows, heads * d] rows at
        positions next ..; the branches of one position rotate as more heads."""
        d = self.config.head_width
        x = x.reshape(batch, rows, heads, d).transpose(0, 1).contiguous()
        normed, out = torch.empty_like(x), torch.empty_like(x)
        self._norm(x, norm, normed, x.numel() // d, d, stream)
        check(lib().dl_rotary(_lib.DL_BF16, normed.data_ptr(), out.data_ptr(), rows, batch * heads, d, 0,
                              self.config.theta, stream, self._next.data_ptr(), 0))
        return out.transpose(0, 1).contiguous()

    # ---- eviction ----------------------------------------------------------
    def _summed(self):
        if self.suffix_weights is None:
            raise ValueError("eviction needs branches made with weights=True")

    def evict_prefix(self, budget: int, first: int = 4, recent: int = 0) -> None:
        """Keep `budget` prompt keys per block and KV head, those the branches
        looked at most (and the `first` and `recent` positions, together at
        most `budget`), or all of a shorter prompt, in a cache of the branches'
        own; the engine's is left as it is."""
        self._summed()
        self._open()
        kept = min(budget, self.prefix)
        lengths = torch.full((1,), self.prefix, dtype=torch.int64, device=self._device)
        for i, (key, value) in enumerate(self._prefix):
            out = [torch.empty((1, kept, *key.shape[1:]), dtype=_BF16, device=self._device) for _ in range(2)]
            out += [torch.empty((1, key.shape[1], kept), device=self._device),
                    torch.empty((1, key.shape[1], kept), dtype=torch.int32, device=self._device),
                    torch.empty_like(lengths)]
            shared.cache_evict(key[None], value[None], self.prefix_weights[i][None], self._prefix_positions[i], lengths,
                               budget, first=first, recent=recent, out=out)
            self._prefix[i] = (out[0][0], out[1][0])
            self.prefix_weights[i], self._prefix_positions[i] = out[2][0], out[3]
        self.prefix = kept
        self._prefix_lengths.fill_(kept)

    def evict_suffix(self, budget: int, recent: int = 32) -> None:
        """Keep `budget` slots of every branch's own cache, in place: the
        `recent` newest tokens and those that were looked at most."""
        self._summed()
        kept = torch.empty_like(self._suffix_lengths)
        for i in range(self.config.layers):
            caches = (self._suffix_key[i], self._suffix_value[i], self.suffix_weights[i], self._suffix_positions[i])
            shared.cache_evict(*caches, self._suffix_lengths, budget, recent=min(recent, budget),
                               out=(*caches, kept))  # the next block still reads the old lengths
        self._suffix_lengths.copy_(kept)
        self.length = min(self.length, budget)
