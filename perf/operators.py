"""The shared-prefix serving operators as a user's program calls them, and their plain forms.

Three operators of a batch of sequences that continue one prompt:

* attention over the prompt's cache, held once for the whole batch, and over each sequence's own cache of what came
  after it ("attend");
* the same call with the weight that every cached key received added to running FP32 sums ("attend" with weights);
* eviction: the cache slots with the least accumulated weight are dropped and the rest compacted ("evict").

Definitions.  Row i of sequence b (rows = new tokens per sequence) attends prefix keys j < prefix_lengths[b] and suffix
keys j < suffix_lengths[b] - (rows - 1 - i); softmax of q.k / sqrt(width) over both; a row without keys gives zeros and a
log-sum-exp of -inf.  Query heads h use KV head h // (query_heads / kv_heads).

Eviction, per cache and KV head with n valid slots: a slot is protected when its position is below `first` or among the
`recent` newest positions; slots are ranked protected first, then by weight (largest first, NaN last), then lowest slot;
the best min(n, budget) stay.  Kept slots below that count stay where they are; the kept slots from there on move into
the vacated ones, in ascending order.
"""
import math

import torch

own = False


# ---------------------------------------------------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------------------------------------------------
def _attend(name, batch, rows, prefix, suffix, query_heads=32, kv_heads=8, width=128, ragged=False, branched=False,
            weights=False):
    c = {"op": "attend", "batch": batch, "rows": rows, "prefix": prefix, "suffix": suffix, "query_heads": query_heads,
         "kv_heads": kv_heads, "width": width, "ragged": ragged, "branched": branched, "weights": weights}
    return {"name": name, **c} if name else c


def _evict(name, caches, length, budget, first, recent, kv_heads=8, width=128, ragged=False):
    c = {"op": "evict", "caches": caches, "length": length, "budget": budget, "first": first, "recent": recent,
         "kv_heads": kv_heads, "width": width, "ragged": ragged}
    return {"name": name, **c} if name else c


def listed():
    return [
        # A steered and an unsteered continuation of one 256-token prompt, one decode step: latency.
        _attend("two branches, 256 keys", 2, 1, 256, 64),
        # Sixteen samples from a 64-token prefix, some way into their 128 tokens: latency, suffixes longer than the prefix.
        _attend("sixteen samples, 64 keys", 16, 1, 64, 128, ragged=True),
        # Batch 32 on an 8192-token prompt, answers of different lengths: the ordinary decode step.
        _attend("batch 32, 8192 keys", 32, 1, 8192, 256, ragged=True),
        # A long document answered at length for 64 users: the largest decode step.
        _attend("batch 64, 32768 keys", 64, 1, 32768, 2048, ragged=True),
        # Odd sizes, seven query heads per KV head, narrow heads, branches that leave the prompt at different tokens.
        _attend("five odd branches", 5, 1, 1999, 77, 28, 4, 64, ragged=True, branched=True),
        # The prompt is cached; every user's next turn of 48 tokens is read in one pass.
        _attend("turns of 48 tokens", 8, 48, 4096, 112, ragged=True),
        # Eight documents' own 512 tokens after a common 8192-token prompt: the largest pass over new tokens.
        _attend("eight tails of 512", 8, 512, 8192, 512),
        # The ordinary decode step of a server that will evict by accumulated weight.
        _attend("batch 32 with weights", 32, 1, 8192, 256, ragged=True, weights=True),
        # A prompt's last 64 tokens score its keys before the cache is cut.
        _attend("window of 64 with weights", 4, 64, 8192, 64, weights=True),
        # Two short caches trimmed by a quarter: latency.
        _evict("two caches 320 to 256", 2, 320, 256, 4, 32),
        # A batch of 32 caches over their budget by an eighth, of different lengths.
        _evict("batch 32, 2304 to 2048", 32, 2304, 2048, 4, 256, ragged=True),
        # A long prompt's cache cut to a quarter before the batch continues it.
        _evict("prompt 32768 to 8192", 1, 32768, 8192, 4, 512),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    most = [work(c) for c in listed()]
    most = {k: max(w[k] for w in most) for k in ("bytes", "flops")}
    while True:
        kind = rng.choice(("decode", "decode", "rows", "evict"))
        width = rng.choice((64, 128, 128, 128))
        kv_heads = rng.choice((1, 2, 4, 8, 8))
        if kind == "evict":
            length = _log_int(rng, 64, 32768)
            budget = max(16, int(length * rng.uniform(0.2, 0.95)))
            case = _evict(None, _log_int(rng, 1, 32), length, budget, rng.choice((0, 1, 4)),
                          rng.randint(0, budget // 4), kv_heads, width, rng.random() < 0.5)
        else:
            rows = 1 if kind == "decode" else _log_int(rng, 2, 512)
            prefix = _log_int(rng, 16, 32768)
            suffix = rows - 1 + _log_int(rng, 1, 2048 if kind == "decode" else 512)
            case = _attend(None, _log_int(rng, 1, 64), rows, prefix, suffix, kv_heads * rng.choice((1, 2, 4, 4, 5, 7, 8)),
                           kv_heads, width, rng.random() < 0.5, rng.random() < 0.3, rng.random() < 0.4)
        need = work(case)
        if all(need[k] <= most[k] for k in need):
            return case


def _lengths(case):
    """(prefix lengths, suffix lengths) or the caches' lengths: plain numbers of the case alone."""
    if case["op"] == "evict":
        n, top, low = case["caches"], case["length"], max(1, case["budget"] // 2)
        return [top - (b * 7919 % 97) * (top - low) // 97 if case["ragged"] else top for b in range(n)]
    n, rows, p, s = case["batch"], case["rows"], case["prefix"], case["suffix"]
    suffix = [s - (b * 7919 % 97) * (s - rows) // 97 if case["ragged"] else s for b in range(n)]
    prefix = [p - (b * 31 % 8) * p // 16 if case["branched"] else p for b in range(n)]
    return prefix, suffix


def work(case):
    if case["op"] == "evict":
        rows = sum(min(n, case["budget"]) for n in _lengths(case)) * case["kv_heads"]
        seen = sum(_lengths(case)) * case["kv_heads"]
        # Every weight and position read; the kept rows' keys, values, weights and positions written; their keys and
        # values read.
        return {"bytes": 8 * seen + 8 * rows + 2 * rows * 2 * 2 * case["width"], "flops": 0}
    prefix, suffix = _lengths(case)
    rows, hq, hkv, d = case["rows"], case["query_heads"], case["kv_heads"], case["width"]
    keys = max(prefix) + sum(suffix)
    pairs = sum(rows * (p + s) - rows * (rows - 1) // 2 for p, s in zip(prefix, suffix))
    tokens = case["batch"] * rows
    moved = 2 * keys * hkv * d * 2 + 2 * tokens * hq * d * 2 + 4 * tokens * hq
    if case["weights"]:
        moved += 8 * keys * hkv
    return {"bytes": moved, "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------------------------------------------------
def _normed(shape, gain, g):
    """Rows as QK-norm leaves them: unit mean square times a learned gain per feature."""
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.bfloat16)
    w = gain * torch.exp(0.3 * torch.randn(shape[-1], generator=g, device="cuda"))
    return x * w.to(torch.bfloat16)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    hkv, d = case["kv_heads"], case["width"]
    if case["op"] == "evict":
        n, top, budget = case["caches"], case["length"], case["budget"]
        lengths = torch.tensor(_lengths(case), device="cuda")
        heavy = torch.exp(2.5 * torch.randn((n, hkv, top), generator=g, device="cuda"))
        none = torch.rand((n, hkv, top), generator=g, device="cuda") < 0.1  # keys that nothing ever looked at
        order = torch.rand((n, hkv, top), generator=g, device="cuda")       # an earlier eviction moved some slots
        order = torch.where(torch.arange(top, device="cuda") < lengths[:, None, None], order, 2.0)
        return {"case": dict(case), "key": _normed((n, top, hkv, d), 1.0, g),
                "value": torch.randn((n, top, hkv, d), generator=g, device="cuda", dtype=torch.bfloat16),
                "weights": torch.where(none, 0.0, heavy), "positions": order.argsort(-1).argsort(-1).to(torch.int32),
                "lengths": lengths,
                "out": (torch.zeros((n, budget, hkv, d), device="cuda", dtype=torch.bfloat16),
                        torch.zeros((n, budget, hkv, d), device="cuda", dtype=torch.bfloat16),
                        torch.zeros((n, hkv, budget), device="cuda"),
                        torch.zeros((n, hkv, budget), device="cuda", dtype=torch.int32),
                        torch.zeros(n, device="cuda", dtype=torch.int64))}
    b, rows, p, s = case["batch"], case["rows"], case["prefix"], case["suffix"]
    prefix, suffix = _lengths(case)
    room_p, room_s = -(-p // 16) * 16, -(-s // 16) * 16  # caches have some room left
    state = {"case": dict(case), "query": _normed((b, rows, case["query_heads"], d), 1.5, g),
             "prefix_key": _normed((room_p, hkv, d), 1.0, g),
             "prefix_value": torch.randn((room_p, hkv, d), generator=g, device="cuda", dtype=torch.bfloat16),
             "suffix_key": _normed((b, room_s, hkv, d), 1.0, g),
             "suffix_value": torch.randn((b, room_s, hkv, d), generator=g, device="cuda", dtype=torch.bfloat16),
             "prefix_lengths": torch.tensor(prefix, device="cuda"), "suffix_lengths": torch.tensor(suffix, device="cuda"),
             "prefix_weights": None, "suffix_weights": None}
    if case["weights"]:
        share = rows * case["query_heads"] / (hkv * (p + s))  # sums of earlier steps
        state["prefix_weights"] = b * share * torch.rand((hkv, room_p), generator=g, device="cuda")
        state["suffix_weights"] = share * torch.rand((b, hkv, room_s), generator=g, device="cuda")
    return state


# ---------------------------------------------------------------------------------------------------------------------
# The passes
# ---------------------------------------------------------------------------------------------------------------------
def run(state):
    if state["case"]["op"] == "evict":
        if own:
            from dolittle_b200 import shared
            got = shared.cache_evict(state["key"], state["value"], state["weights"], state["positions"],
                                     state["lengths"], state["case"]["budget"], first=state["case"]["first"],
                                     recent=state["case"]["recent"], out=state["out"])
        else:
            got = _plain_evict(state)
        return dict(zip(("key", "value", "weights", "positions", "lengths"), got))
    if own:
        from dolittle_b200 import shared
        out, lse = shared.attention_shared(state["query"], state["prefix_key"], state["prefix_value"],
                                           state["suffix_key"], state["suffix_value"], state["prefix_lengths"],
                                           state["suffix_lengths"], prefix_weights=state["prefix_weights"],
                                           suffix_weights=state["suffix_weights"])
    else:
        out, lse = _plain_attend(state)
    got = {"out": out, "lse": lse}
    if state["case"]["weights"]:
        got.update(prefix_weights=state["prefix_weights"], suffix_weights=state["suffix_weights"])
    return got


def _plain_attend(state):
    q = state["query"].float()
    b, rows, hq, d = q.shape
    pk, pv, sk, sv = (state[n].float() for n in ("prefix_key", "prefix_value", "suffix_key", "suffix_value"))
    hkv, p, s = pk.shape[1], pk.shape[0], sk.shape[1]
    group = hq // hkv
    q = q.view(b, rows, hkv, group, d).permute(2, 0, 1, 3, 4)  # [Hkv][B][rows][group][d]
    one = q.reshape(hkv, b * rows * group, d) @ pk.permute(1, 2, 0)
    two = q.reshape(hkv, b, rows * group, d) @ sk.permute(2, 0, 3, 1)
    shape = (hkv, b, rows, group)
    scores = torch.cat((one.view(*shape, p), two.view(*shape, s)), -1) * (1.0 / math.sqrt(d))
    at = torch.arange(p + s, device="cuda")
    row = torch.arange(rows, device="cuda")
    seen_p = (at[:p] < state["prefix_lengths"][:, None])[:, None].expand(b, rows, p)
    seen_s = at[:s] < (state["suffix_lengths"][:, None] - (rows - 1 - row))[:, :, None]
    seen = torch.cat((seen_p, seen_s), -1)[None, :, :, None]  # [1][B][rows][1][keys]
    scores = torch.where(seen, scores, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0.0, top)
    weights = torch.exp(scores - top)
    total = weights.sum(-1, keepdim=True)
    lse = torch.log(total) + top
    weights = weights / torch.where(total == 0, 1.0, total)
    out = weights[..., :p].reshape(hkv, b * rows * group, p) @ pv.transpose(0, 1)
    out = out.view(hkv, b, rows * group, d) + weights[..., p:].reshape(hkv, b, rows * group, s) @ sv.permute(2, 0, 1, 3)
    if state["prefix_weights"] is not None:
        state["prefix_weights"] += weights[..., :p].sum((1, 2, 3))
        state["suffix_weights"] += weights[..., p:].sum((2, 3)).transpose(0, 1)
    out = out.view(*shape, d).permute(1, 2, 0, 3, 4).reshape(b, rows, hq, d)
    return out.to(torch.bfloat16), lse.view(shape).permute(1, 2, 0, 3).reshape(b, rows, hq)


def _plain_evict(state):
    case, weights, positions = state["case"], state["weights"], state["positions"]
    budget, top = case["budget"], weights.shape[-1]
    slot = torch.arange(top, device="cuda")
    count = state["lengths"][:, None, None]
    stays = torch.clamp(count, max=budget)
    valid = slot < count
    newest = torch.where(valid, positions, -1).amax(-1, keepdim=True)
    rank = valid.int() + (valid & ((positions < case["first"]) | (positions > newest - case["recent"]))).int()
    weight = torch.where(torch.isnan(weights), -math.inf, weights)
    order = torch.sort(weight, dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, torch.sort(rank.gather(-1, order), dim=-1, descending=True, stable=True).indices)
    kept = torch.zeros_like(valid.expand_as(rank)).scatter(-1, order, slot.expand_as(order) < stays)
    moved = torch.sort((kept & (slot >= stays)).int(), dim=-1, descending=True, stable=True).indices
    hole = ~kept & (slot < stays)
    source = torch.where(hole, moved.gather(-1, (hole.cumsum(-1) - 1).clamp(min=0)), slot)[..., :budget]
    there = (slot < stays)[..., :budget]
    key, value, weight_out, position_out, length_out = state["out"]
    at = source.transpose(1, 2)[..., None]
    live = there.transpose(1, 2)[..., None]
    key.copy_(torch.where(live, state["key"].gather(1, at.expand(*at.shape[:3], case["width"])), key))
    value.copy_(torch.where(live, state["value"].gather(1, at.expand(*at.shape[:3], case["width"])), value))
    weight_out.copy_(torch.where(there, weights.gather(-1, source), weight_out))
    position_out.copy_(torch.where(there, positions.gather(-1, source), position_out))
    length_out.copy_(stays[:, 0, 0])
    return state["out"]


# ---------------------------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    return _exact_evict(state) if case["op"] == "evict" else _exact_attend(state)


def _exact_attend(state):
    case = state["case"]
    prefix, suffix = _lengths(case)
    rows, d, hkv = case["rows"], case["width"], case["kv_heads"]
    group = case["query_heads"] // hkv
    out = torch.zeros(state["query"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(out.shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    sums = [state[n].double() if state[n] is not None else None for n in ("prefix_weights", "suffix_weights")]
    for b, (p, s) in enumerate(zip(prefix, suffix)):
        last = s - (rows - 1) + torch.arange(rows, device="cuda")  # suffix keys that each row sees
        hidden = torch.arange(s, device="cuda")[None, :] >= last[:, None]
        for h in range(hkv):
            k = torch.cat((state["prefix_key"][:p, h], state["suffix_key"][b, :s, h])).double()
            v = torch.cat((state["prefix_value"][:p, h], state["suffix_value"][b, :s, h])).double()
            for i in range(h * group, (h + 1) * group):
                x = state["query"][b, :, i].double() @ k.T / d ** 0.5
                x[:, p:].masked_fill_(hidden, -math.inf)
                lse[b, :, i] = torch.logsumexp(x, -1)
                w = torch.softmax(x, -1)
                out[b, :, i] = w @ v
                if sums[0] is not None:
                    sums[0][h, :p] += w[:, :p].sum(0)
                    sums[1][b, h, :s] += w[:, p:].sum(0)
    got = {"out": out, "lse": lse}
    if sums[0] is not None:
        got.update(prefix_weights=sums[0], suffix_weights=sums[1])
    return got


def _exact_evict(state):
    case = state["case"]
    key, value, weight_out, position_out, length_out = (x.double().cpu() if x.is_floating_point() else x.cpu()
                                                        for x in state["out"])
    weights, positions = state["weights"].cpu(), state["positions"].cpu()
    source_key, source_value = state["key"].cpu(), state["value"].cpu()
    for c, n in enumerate(_lengths(case)):
        stays = min(n, case["budget"])
        length_out[c] = stays
        for h in range(case["kv_heads"]):
            w, pos = weights[c, h, :n].tolist(), positions[c, h, :n].tolist()
            newest = max(pos)
            best = sorted(range(n), key=lambda j: (not (pos[j] < case["first"] or pos[j] > newest - case["recent"]),
                                                   -w[j], j))[:stays]
            kept = set(best)
            late = iter(sorted(j for j in best if j >= stays))
            source = torch.tensor([j if j in kept else next(late) for j in range(stays)])
            key[c, :stays, h] = source_key[c, source, h].double()
            value[c, :stays, h] = source_value[c, source, h].double()
            weight_out[c, h, :stays] = weights[c, h, source].double()
            position_out[c, h, :stays] = positions[c, h, source]
    return {"key": key, "value": value, "weights": weight_out, "positions": position_out, "lengths": length_out}
