"""Attention over a shared prefix and per-sequence suffixes, the sums of the
weight each key receives, and eviction by them, against the definitions in 64
bits.

Tolerances, all from the operation counts:
* output: one BF16 rounding of the result (2^-9 of it) and one of each softmax
  weight before the second product (2^-9 of sum w |v|, which bounds the
  result), 2 % on top for the FP32 steps;
* log-sum-exp: a score is d FP32 accumulations (d 2^-24 of sum |q k| scale,
  which also covers an accumulator that truncates), the sum of n exponentials
  random roundings (4 sqrt(n) 2^-24) of exponentials good to 2^-21;
* key weights: exp of the errors of score and log-sum-exp, and the roundings of
  a sum over the rows.
Eviction moves bits and is exact.
"""
import math

import pytest
import torch

from dolittle_b200 import _lib, shared

pytestmark = pytest.mark.gpu


def make(batch, rows, prefix, suffix, hq=32, hkv=8, d=128, seed=0, plens=None, slens=None, gain=1.5, room=5):
    """Inputs of one call; everything past the lengths is NaN or infinite."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def rand(*shape, k=1.0):
        return (k * torch.randn(shape, generator=g, device="cuda")).to(torch.bfloat16)

    t = {"query": rand(batch, rows, hq, d, k=gain)}
    for side, n, lead, lens in (("prefix", prefix, (), plens), ("suffix", suffix, (batch,), slens)):
        if n is None:
            t.update({f"{side}_key": None, f"{side}_value": None, f"{side}_lengths": None})
            continue
        lens = [n] * batch if lens is None else lens
        key, value = rand(*lead, n + room, hkv, d), rand(*lead, n + room, hkv, d)
        for b in range(batch if lead else 1):
            end = lens[b] if lead else max(lens)
            at = (b,) if lead else ()
            key[at][end:], value[at][end:] = math.nan, math.inf
        t.update({f"{side}_key": key, f"{side}_value": value,
                  f"{side}_lengths": torch.tensor(lens, dtype=torch.int64, device="cuda")})
    return t


def reference(t):
    """out, lse, key weights of prefix and suffix, and the tolerances' sums."""
    q = t["query"].double()
    batch, rows, hq, d = q.shape
    caches = [t[f"{s}_{k}"] for s in ("prefix", "suffix") for k in ("key", "value")]
    hkv = next(c for c in caches if c is not None).shape[-2]
    group = hq // hkv
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    lse = torch.full((batch, rows, hq), -math.inf, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(lse)
    pw = None if caches[0] is None else torch.zeros(hkv, caches[0].shape[0], dtype=torch.float64, device="cuda")
    sw = None if caches[2] is None else torch.zeros(batch, hkv, caches[2].shape[1], dtype=torch.float64, device="cuda")
    for b in range(batch):
        np_ = 0 if pw is None else int(t["prefix_lengths"][b])
        for i in range(rows):
            ns = 0 if sw is None else max(0, int(t["suffix_lengths"][b]) - (rows - 1 - i))
            if np_ + ns == 0:
                continue
            parts_k, parts_v = [], []
            if np_:
                parts_k.append(caches[0][:np_]), parts_v.append(caches[1][:np_])
            if ns:
                parts_k.append(caches[2][b, :ns]), parts_v.append(caches[3][b, :ns])
            k = torch.cat(parts_k).double().repeat_interleave(group, 1)
            v = torch.cat(parts_v).double().repeat_interleave(group, 1)
            s = torch.einsum("hd,nhd->hn", q[b, i], k) / math.sqrt(d)
            w = torch.softmax(s, -1)
            lse[b, i] = torch.logsumexp(s, -1)
            size[b, i] = (torch.einsum("hd,nhd->hn", q[b, i].abs(), k.abs()) / math.sqrt(d)).amax(-1)
            out[b, i] = torch.einsum("hn,nhd->hd", w, v)
            spread[b, i] = torch.einsum("hn,nhd->hd", w, v.abs())
            per_head = w.view(hkv, group, -1).sum(1)
            if np_:
                pw[:, :np_] += per_head[:, :np_]
            if ns:
                sw[b, :, :ns] += per_head[:, np_:]
    return out, lse, pw, sw, spread, size


def check_attention(t, weights=True, **kw):
    out, lse, pw, sw, spread, size = reference(t)
    batch, rows, hq, d = out.shape
    start = []
    for ref in (pw, sw):
        start.append(None if ref is None or not weights else torch.rand(ref.shape, device="cuda"))
    acc = [None if x is None else x.clone() for x in start]
    got, got_lse = shared.attention_shared(t["query"], t["prefix_key"], t["prefix_value"], t["suffix_key"],
                                           t["suffix_value"], t["prefix_lengths"], t["suffix_lengths"],
                                           prefix_weights=acc[0], suffix_weights=acc[1], **kw)
    torch.cuda.synchronize()
    keys = sum(0 if t[f"{s}_key"] is None else int(t[f"{s}_lengths"].max()) for s in ("prefix", "suffix"))
    lse_tol = d * 2.0 ** -24 * size + 4 * math.sqrt(keys + 1) * 2.0 ** -24 + 2.0 ** -21
    empty = torch.isinf(lse)
    assert torch.equal(torch.isinf(got_lse), empty) and bool((got_lse[empty] < 0).all())
    assert bool((got[empty] == 0).all())
    err = (got_lse.double() - lse).abs()[~empty]
    assert bool((err <= lse_tol[~empty]).all()), (err.max().item(), lse_tol.min().item())
    err = (got.double() - out).abs()
    tol = 1.02 * 2.0 ** -8 * spread
    assert bool((err <= tol).all()), ((err - tol).max().item(), err.max().item())
    for ref, a, x in ((pw, acc[0], start[0]), (sw, acc[1], start[1])):
        if x is None:
            continue
        added = 2 * lse_tol.max() + 2.0 ** -21 + 4 * math.sqrt(batch * rows * hq) * 2.0 ** -24
        err = (a.double() - (x.double() + ref)).abs()
        tol = added * ref + 2.0 ** -23 * (ref + x)
        assert bool((err <= tol).all()), ((err - tol).max().item(), err.max().item())
        assert torch.equal(a[ref == 0], x[ref == 0])  # keys no row saw stay as they were
    return got, got_lse, acc


SHAPES = [
    # batch, rows, prefix, suffix, hq, hkv, d, plens, slens
    (2, 1, 256, 64, 32, 8, 128, None, None),
    (16, 1, 64, 128, 32, 8, 128, None, [1, 2, 15, 16, 17, 63, 64, 65, 100, 127, 128, 31, 32, 33, 48, 5]),
    (32, 1, 700, 40, 32, 8, 128, None, None),
    (33, 1, 1025, 9, 32, 8, 128, None, None),                   # one token past a tile of rows
    (70, 1, 300, 70, 16, 4, 128, None, None),
    (1, 1, 1, None, 8, 8, 128, None, None),                     # one key
    (3, 1, None, 5, 8, 2, 128, None, [5, 1, 0]),                # no prefix, one empty row
    (4, 1, 130, 3, 28, 4, 64, [130, 0, 1, 129], [3, 0, 0, 2]),  # an empty sequence, ends inside a tile
    (5, 1, 127, 1, 5, 5, 64, [127, 126, 64, 63, 1], None),
    (3, 1, 257, 30, 64, 1, 128, None, None),                    # 64 query heads on one KV head
    (2, 1, 4000, 2100, 8, 2, 128, None, [2100, 1999]),          # few units, long ranges
    (1, 1, 9000, 1, 4, 1, 128, None, None),
    (6, 1, 500, 200, 40, 8, 128, [500, 480, 470, 500, 33, 128], None),
    (3, 2, 100, 20, 32, 8, 128, None, None),
    (4, 8, 200, 30, 32, 8, 128, None, [30, 8, 7, 1]),           # fewer suffix keys than rows
    (5, 9, 131, 40, 28, 4, 64, [131, 0, 128, 5, 130], [40, 9, 3, 0, 20]),
    (3, 33, 300, 65, 32, 8, 128, None, [65, 33, 50]),
    (2, 40, 260, 300, 28, 4, 128, [260, 100], [300, 41]),
    (2, 100, 129, 100, 8, 8, 64, None, None),
    (1, 150, None, 150, 32, 8, 128, None, None),                # a prompt alone
    (1, 257, 64, 300, 16, 2, 128, None, None),
    (2, 20, 500, None, 64, 1, 64, None, None),
    (40, 3, 90, 12, 12, 4, 128, None, None),
]


@pytest.mark.parametrize("batch,rows,prefix,suffix,hq,hkv,d,plens,slens", SHAPES)
def test_attention_matches_definition(batch, rows, prefix, suffix, hq, hkv, d, plens, slens):
    t = make(batch, rows, prefix, suffix, hq, hkv, d, seed=batch * 31 + rows, plens=plens, slens=slens)
    got, lse, acc = check_attention(t)
    # The weights are a by-product: the attention is the same without them.
    got2, lse2, _ = check_attention(t, weights=False)
    assert torch.equal(got, got2) and torch.equal(lse, lse2)


# Sizes around the limits between the plans: rows of a sequence and KV head in
# one or two blocks of 16, one or four warps per joined row, one or more chunks
# of suffix keys, key ranges of one and of two row tiles.
PLANS = [
    (64, 4, 300, 20, 32, 8, 128, None, [4 + 7919 * b % 17 for b in range(64)]),
    (20, 7, 600, 30, 32, 8, 128, [600 - 30 * b for b in range(20)], None),
    (6, 8, 900, 700, 32, 8, 128, None, [700, 8, 513, 512, 511, 7]),
    (2, 5, 200, 1100, 20, 4, 64, None, [1100, 1]),
    (3, 1, 3000, 1300, 16, 1, 128, [3000, 2999, 1], [1300, 1025, 0]),
    (3, 2, 900, 530, 32, 2, 64, None, None),
    (60, 1, 1500, 40, 28, 4, 64, None, None),
    (9, 1, 2600, 600, 32, 1, 128, None, None),
    (4, 48, 1300, 60, 32, 8, 128, None, [60, 48, 49, 50]),
    (9, 64, 500, 64, 32, 8, 64, None, None),
    (1, 200, 2000, 200, 16, 4, 128, None, None),
    (1, 88, 291, 91, 8, 4, 128, None, None),
    (2, 8, 512, 64, 32, 8, 128, [512, 300], [64, 9]),
    (3, 40, 300, 40, 28, 4, 64, [300, 0, 299], [40, 20, 3]),
    (2, 64, None, 64, 4, 1, 128, None, None),
    (13, 90, 71, 91, 4, 2, 64, [71, 0, 70] + [5 * b for b in range(10)], [91, 90, 60] + [91] * 10),
    (1, 700, 40, 700, 2, 1, 64, None, None),
    (3, 400, None, 600, 2, 1, 128, None, [600, 400, 3]),
]


@pytest.mark.parametrize("batch,rows,prefix,suffix,hq,hkv,d,plens,slens", PLANS)
def test_plans_match_definition_and_repeat(batch, rows, prefix, suffix, hq, hkv, d, plens, slens):
    t = make(batch, rows, prefix, suffix, hq, hkv, d, seed=batch * 37 + rows, plens=plens, slens=slens)
    got, lse, _ = check_attention(t)
    again, lse2, _ = check_attention(t, weights=False)
    assert torch.equal(got, again) and torch.equal(lse, lse2)


@pytest.mark.parametrize("rows", [1, 70])
def test_growing_and_huge_scores(rows):
    """Every block of keys raises the running maximum; scores up to several hundred."""
    t = make(3, rows, 700, 150, seed=5, gain=1.0, slens=[150, 149, 70])
    t["prefix_key"][:700] *= torch.linspace(0.1, 12, 700, device="cuda").to(torch.bfloat16)[:, None, None]
    t["suffix_key"][0, :150] *= 15
    t["query"] *= 4
    check_attention(t)


@pytest.mark.parametrize("rows", [1, 40])
def test_one_key_takes_everything(rows):
    """A score far above the rest: all other weights vanish, their sums stay exact zeros or tiny."""
    t = make(2, rows, 300, 60, seed=6)
    t["prefix_key"][7] = 100 * t["query"][0, 0, ::4]
    check_attention(t)


@pytest.mark.parametrize("rows,group", [(1, 4), (6, 4), (50, 8)])
def test_strides_and_views(rows, group):
    """Queries inside a fused qkv row, a prefix inside an engine-like arena with
    rows further apart, suffix keys and values interleaved per position."""
    batch, hkv, d = 3, 4, 128
    hq = hkv * group
    t = make(batch, rows, 200, 90, hq, hkv, d, seed=9, room=0)
    fused = torch.full((batch, rows, hq + 2 * hkv, d), math.nan, device="cuda", dtype=torch.bfloat16)
    fused[:, :, :hq] = t["query"]
    t["query"] = fused[:, :, :hq]
    wide = torch.full((230, 2, hkv + 1, d), math.nan, device="cuda", dtype=torch.bfloat16)
    wide[30:, 0, 1:], wide[30:, 1, 1:] = t["prefix_key"], t["prefix_value"]
    t["prefix_key"], t["prefix_value"] = wide[30:, 0, 1:], wide[30:, 1, 1:]
    both = torch.full((batch, 97, 2, hkv, d), math.nan, device="cuda", dtype=torch.bfloat16)
    both[:, 7:, 0], both[:, 7:, 1] = t["suffix_key"], t["suffix_value"]
    t["suffix_key"], t["suffix_value"] = both[:, 7:, 0], both[:, 7:, 1]
    check_attention(t)


@pytest.mark.parametrize("rows", [1, 40])
def test_offsets_past_32_bits(rows):
    """Sequences 1.2e9 elements apart: the third starts past 2^31."""
    apart, n, hkv, d = 1_200_000_000, 40, 2, 128
    arena = torch.empty(2 * apart + 2 * n * hkv * d, device="cuda", dtype=torch.bfloat16)
    t = make(3, rows, 50, n, 8, hkv, d, seed=11, room=0)
    shape, stride = (3, n, hkv, d), (apart, hkv * d, d, 1)
    key = torch.as_strided(arena, shape, stride, 0)
    value = torch.as_strided(arena, shape, stride, n * hkv * d)
    key.copy_(t["suffix_key"]), value.copy_(t["suffix_value"])
    t["suffix_key"], t["suffix_value"] = key, value
    check_attention(t)


@pytest.mark.parametrize("batch,rows,prefix,suffix", [(32, 1, 3000, 100), (2, 1, 200, 500), (3, 90, 700, 90)])
def test_repeats_bit_for_bit_and_on_other_streams(batch, rows, prefix, suffix):
    t = make(batch, rows, prefix, suffix, seed=13)
    args = [t[k] for k in ("query", "prefix_key", "prefix_value", "suffix_key", "suffix_value", "prefix_lengths",
                           "suffix_lengths")]

    def call():
        w = [torch.zeros(8, prefix + 5, device="cuda"), torch.zeros(batch, 8, suffix + 5, device="cuda")]
        return [*shared.attention_shared(*args, prefix_weights=w[0], suffix_weights=w[1]), *w]

    first = call()
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(first, call()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = call()
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(first, again))


@pytest.mark.parametrize("rows", [1, 30])
def test_captured_graph_follows_lengths(rows):
    """The lengths are device data: a captured call replays with the new ones."""
    t = make(4, rows, 300, 80, seed=17, plens=[200] * 4, slens=[40] * 4)
    out, lse = torch.zeros_like(t["query"]), torch.zeros(4, rows, 32, device="cuda")
    args = [t[k] for k in ("query", "prefix_key", "prefix_value", "suffix_key", "suffix_value", "prefix_lengths",
                           "suffix_lengths")]
    shared.attention_shared(*args, out=out, lse=lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        shared.attention_shared(*args, out=out, lse=lse)
    for name, n in (("prefix", 300), ("suffix", 80)):
        for part in ("key", "value"):
            t[f"{name}_{part}"].copy_(torch.randn_like(t[f"{name}_{part}"]))
    t["prefix_lengths"].copy_(torch.tensor([300, 1, 128, 0], device="cuda"))
    t["suffix_lengths"].copy_(torch.tensor([80, 30, 31, 0], device="cuda"))
    graph.replay()
    torch.cuda.synchronize()
    ref, ref_lse, _, _, spread, _ = reference(t)
    assert bool(((out.double() - ref).abs() <= 1.02 * 2.0 ** -8 * spread).all())
    assert torch.equal(torch.isinf(lse), torch.isinf(ref_lse))


def test_lengths_outside_the_caches_are_clamped():
    t = make(3, 1, 100, 20, seed=19, room=0)
    t["prefix_lengths"].copy_(torch.tensor([1 << 40, -3, 100], device="cuda"))
    t["suffix_lengths"].copy_(torch.tensor([20, -(1 << 33), 1 << 35], device="cuda"))
    args = [t[k] for k in ("query", "prefix_key", "prefix_value", "suffix_key", "suffix_value", "prefix_lengths",
                           "suffix_lengths")]
    out, lse = shared.attention_shared(*args)
    t["prefix_lengths"].copy_(torch.tensor([100, 0, 100], device="cuda"))
    t["suffix_lengths"].copy_(torch.tensor([20, 0, 20], device="cuda"))
    want, want_lse = shared.attention_shared(*args)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    assert bool((out[1] == 0).all()) and bool(torch.isinf(lse[1]).all())


def test_attention_refusals():
    t = make(2, 1, 64, 16, seed=1)
    args = [t[k] for k in ("query", "prefix_key", "prefix_value", "suffix_key", "suffix_value", "prefix_lengths",
                           "suffix_lengths")]

    def refused(error, **change):
        names = ("query", "prefix_key", "prefix_value", "suffix_key", "suffix_value", "prefix_lengths",
                 "suffix_lengths")
        kw = {k: v for k, v in change.items() if k not in names}
        with pytest.raises(error):
            shared.attention_shared(*[change.get(n, a) for n, a in zip(names, args)], **kw)

    refused(ValueError, query=t["query"].float())
    refused(ValueError, query=t["query"][..., ::2])
    refused(ValueError, prefix_value=t["prefix_value"][:-1])
    refused(ValueError, prefix_key=t["prefix_key"].cpu())
    refused(ValueError, suffix_key=t["suffix_key"][:1], suffix_value=t["suffix_value"][:1])
    refused(ValueError, prefix_lengths=t["prefix_lengths"].int())
    refused(ValueError, suffix_lengths=t["suffix_lengths"][:1])
    refused(ValueError, prefix_weights=torch.zeros(8, 64, device="cuda"))  # the capacity is 69
    refused(ValueError, suffix_weights=torch.zeros(2, 8, 21, device="cuda", dtype=torch.float64))
    refused(ValueError, out=torch.zeros(2, 1, 32, 64, device="cuda", dtype=torch.bfloat16))
    refused(_lib.DolittleError, query=t["query"][:, :, :30])  # 30 heads on 8
    narrow = {k: (v[..., :96].contiguous() if "len" not in k else v) for k, v in t.items()}
    with pytest.raises(_lib.DolittleError):
        shared.attention_shared(*[narrow[k] for k in ("query", "prefix_key", "prefix_value", "suffix_key",
                                                      "suffix_value", "prefix_lengths", "suffix_lengths")])


# ---------------------------------------------------------------------------
# Eviction
# ---------------------------------------------------------------------------
def make_caches(n, capacity, hkv=2, d=64, seed=0, lengths=None, shuffled=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    lengths = torch.tensor([capacity] * n if lengths is None else lengths, dtype=torch.int64, device="cuda")
    order = torch.rand((n, hkv, capacity), generator=g, device="cuda")
    order = torch.where(torch.arange(capacity, device="cuda") < lengths[:, None, None], order, 2.0)
    positions = (order.argsort(-1).argsort(-1) if shuffled else
                 torch.arange(capacity, device="cuda").expand(n, hkv, capacity)).to(torch.int32).contiguous()
    return {"key": torch.randn((n, capacity, hkv, d), generator=g, device="cuda").to(torch.bfloat16),
            "value": torch.randn((n, capacity, hkv, d), generator=g, device="cuda").to(torch.bfloat16),
            "weights": torch.rand((n, hkv, capacity), generator=g, device="cuda"),
            "positions": positions, "lengths": lengths}


def kept_slots(weights, positions, n, budget, first, recent):
    """The slot that ends up in each place, by the definition, in Python."""
    stays = min(n, budget)
    if n == 0:
        return []
    newest = max(positions[:n])

    def rank(j):
        w = weights[j]
        guarded = positions[j] < first or positions[j] > newest - recent
        return (not guarded, 0 if w == w else 1, -w if w == w else 0.0, j)

    def key(j):
        r = rank(j)
        return (r[0], 0, 0.0, j) if not r[0] else r

    best = sorted(range(n), key=key)[:stays]
    kept, late = set(best), iter(sorted(j for j in best if j >= stays))
    return [j if j in kept else next(late) for j in range(stays)]


def check_eviction(c, budget, first, recent, in_place, out_room=0):
    n, capacity, hkv, d = c["key"].shape
    names = ("key", "value", "weights", "positions", "lengths")
    before = {k: c[k].clone() for k in names}
    room = min(budget, capacity) + out_room
    if in_place:
        out = None
        want = {k: c[k].clone() for k in names}
    else:
        out = [torch.full((n, room, hkv, d), 3.0, device="cuda", dtype=torch.bfloat16) for _ in range(2)]
        out += [torch.full((n, hkv, room), 3.0, device="cuda"),
                torch.full((n, hkv, room), 3, device="cuda", dtype=torch.int32),
                torch.full((n,), 3, device="cuda", dtype=torch.int64)]
        want = {k: x.clone() for k, x in zip(names, out)}
    for i in range(n):
        length = max(0, min(capacity, int(before["lengths"][i])))
        want["lengths"][i] = min(length, budget)
        for h in range(hkv):
            source = kept_slots(before["weights"][i, h].tolist(), before["positions"][i, h].tolist(), length, budget,
                                first, recent)
            at, to = torch.tensor(source, dtype=torch.long, device="cuda"), len(source)
            for k in ("key", "value"):
                want[k][i, :to, h] = before[k][i, at, h]
            for k in ("weights", "positions"):
                want[k][i, h, :to] = before[k][i, h, at]
    got = shared.cache_evict(*[c[k] for k in names], budget, first=first, recent=recent, out=out)
    torch.cuda.synchronize()
    for k, x in zip(names, got):
        same = x.view(torch.int32) if x.dtype == torch.float32 else x
        ref = want[k].view(torch.int32) if x.dtype == torch.float32 else want[k]
        assert torch.equal(same, ref), k
        if not in_place:
            assert torch.equal(c[k], before[k]) or x.dtype == torch.float32  # the inputs are only read
    return got


EVICTIONS = [
    # caches, capacity, lengths, budget, first, recent, hkv, d
    (2, 320, None, 256, 4, 32, 8, 128),
    (3, 50, [50, 1, 0], 20, 0, 0, 2, 64),
    (1, 1, None, 1, 0, 1, 1, 64),
    (4, 33, [33, 32, 31, 5], 32, 1, 31, 2, 128),
    (2, 2048, [2048, 1500], 1024, 4, 100, 2, 64),
    (1, 5000, None, 4999, 4, 16, 3, 64),
    (2, 9001, [9001, 8193], 3000, 0, 64, 1, 64),
    (1, 40000, None, 7000, 4, 512, 1, 64),
    (3, 100, None, 200, 2, 2, 2, 64),        # a budget above the capacity evicts nothing
    (2, 64, None, 7, 0, 7, 2, 24),           # every kept slot protected, an unusual width
    (2, 130, [1 << 40, -5], 100, 3, 10, 2, 64),
    (1, 9000, [4097], 2048, 0, 0, 2, 8),     # a cluster whose last blocks hold few slots
    (1, 70000, None, 30000, 2, 3, 1, 8),
    (1, 200000, [150001], 66000, 0, 9, 1, 8),
]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("n,capacity,lengths,budget,first,recent,hkv,d", EVICTIONS)
def test_eviction_matches_definition(n, capacity, lengths, budget, first, recent, hkv, d, in_place):
    c = make_caches(n, capacity, hkv, d, seed=capacity + budget, lengths=lengths)
    check_eviction(c, budget, first, recent, in_place, out_room=3)


@pytest.mark.parametrize("in_place", [True, False])
def test_eviction_of_ties_and_special_weights(in_place):
    """Equal weights (ties to the lowest slot), both zeros, infinities, NaN, negatives, subnormals."""
    c = make_caches(3, 700, 2, 64, seed=3, lengths=[700, 699, 350])
    c["weights"][0] = 1.0
    w = c["weights"][1]
    w[:, ::7], w[:, 1::7], w[:, 2::7], w[:, 3::7] = 0.0, -0.0, math.inf, math.nan
    w[:, 4::7], w[:, 5::7], w[:, 6::7] = -math.inf, 1e-40, -2.5
    c["weights"][2] = torch.randint(0, 4, (2, 700), device="cuda").float()
    check_eviction(c, 300, 5, 40, in_place)


@pytest.mark.parametrize("n,capacity,budget", [(2, 1000, 600), (1, 4000, 999), (1, 20000, 12345), (1, 80000, 40001),
                                               (1, 140000, 70001)])
def test_eviction_of_equal_weights(n, capacity, budget):
    """More equal keys than are ranked one by one: the lowest slots stay."""
    c = make_caches(n, capacity, 1, 8, seed=capacity)
    c["weights"][:] = 0.5
    c["weights"][:, :, capacity // 2::3] = 0.25
    check_eviction(c, budget, 0, 17, True)


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("n,capacity,hkv,d", [(20, 300, 8, 64), (36, 600, 8, 64), (40, 200, 8, 128), (5, 5000, 3, 64),
                                                  (10, 16000, 4, 8), (3, 7000, 1, 8), (80, 4200, 1, 8)])
def test_eviction_with_few_and_many_heads(n, capacity, hkv, d, in_place):
    lengths = [capacity - 13 * b % capacity for b in range(n)]
    check_eviction(make_caches(n, capacity, hkv, d, seed=n, lengths=lengths), capacity * 2 // 3, 4, 20, in_place)


def test_eviction_in_place_with_lengths_of_its_own():
    """In place for the caches, the new lengths elsewhere; then both out of place."""
    for in_place in (True, False):
        c = make_caches(3, 300, 4, 64, seed=8, lengths=[300, 200, 129])
        d = {k: v.clone() for k, v in c.items()}
        want = shared.cache_evict(*[d[k] for k in ("key", "value", "weights", "positions", "lengths")], 128, recent=9)
        fresh = torch.zeros_like(c["lengths"])
        args = [c[k] for k in ("key", "value", "weights", "positions")]
        out = [x if in_place else torch.zeros_like(x) for x in args]
        got = shared.cache_evict(*args, c["lengths"], 128, recent=9, out=[*out, fresh])
        assert c["lengths"].tolist() == [300, 200, 129] and fresh.tolist() == [128, 128, 128]
        for x, y in zip(got[:2], want[:2]):
            assert torch.equal(x[:, :128], y[:, :128])
        for x, y in zip(got[2:4], want[2:4]):
            assert torch.equal(x[..., :128], y[..., :128])


def test_eviction_drops_nan_only_when_it_must():
    c = make_caches(1, 100, 1, 64, seed=4)
    c["weights"][0, 0, 10:90] = math.nan
    check_eviction(c, 50, 0, 0, True)


def test_eviction_in_long_caches_past_32_bits():
    apart, n, hkv, d = 1_200_000_000, 300, 2, 64
    arena = torch.empty(2 * apart + 2 * n * hkv * d, device="cuda", dtype=torch.bfloat16)
    c = make_caches(3, n, hkv, d, seed=5)
    shape, stride = (3, n, hkv, d), (apart, hkv * d, d, 1)
    for i, k in enumerate(("key", "value")):
        x = torch.as_strided(arena, shape, stride, i * n * hkv * d)
        x.copy_(c[k])
        c[k] = x
    small = {k: (v if k not in ("key", "value") else v.contiguous()) for k, v in c.items()}
    want = shared.cache_evict(*[small[k].clone() for k in ("key", "value", "weights", "positions", "lengths")], 100)
    got = shared.cache_evict(*[c[k] for k in ("key", "value", "weights", "positions", "lengths")], 100)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_eviction_refusals():
    c = make_caches(2, 64)
    args = [c[k] for k in ("key", "value", "weights", "positions", "lengths")]
    with pytest.raises(_lib.DolittleError):
        shared.cache_evict(*args, 0)
    with pytest.raises(_lib.DolittleError):
        shared.cache_evict(*args, 16, first=10, recent=7)
    with pytest.raises(ValueError):
        shared.cache_evict(*args[:3], c["positions"].long(), c["lengths"], 16)
    with pytest.raises(ValueError):
        shared.cache_evict(*args[:4], c["lengths"][:1], 16)
    with pytest.raises(_lib.DolittleError):  # some outputs are inputs, others are not
        shared.cache_evict(*args, 16, out=(c["key"], c["value"], torch.zeros_like(c["weights"]), c["positions"],
                                           c["lengths"]))
    small = make_caches(2, 8)
    with pytest.raises(_lib.DolittleError):  # no room for the budget
        shared.cache_evict(*args, 16, out=[small[k] for k in ("key", "value", "weights", "positions", "lengths")])
    odd = torch.zeros((2, 64, 2, 12), device="cuda", dtype=torch.bfloat16)
    with pytest.raises(_lib.DolittleError):
        shared.cache_evict(odd, odd.clone(), *args[2:], 16)


def test_weights_then_eviction_keep_the_attended_keys():
    """The two together: eviction by the sums that attention left keeps each
    head's most attended keys beside the protected ones."""
    t = make(4, 1, 1000, None, seed=21, room=0, gain=1.0)
    weights = torch.zeros(8, 1000, device="cuda")
    shared.attention_shared(t["query"], t["prefix_key"], t["prefix_value"], None, None, t["prefix_lengths"], None,
                            prefix_weights=weights)
    total = weights.sum(-1)
    assert torch.allclose(total, torch.full_like(total, 16.0), rtol=1e-4)  # 4 sequences x 4 heads, 1 each
    positions = torch.arange(1000, dtype=torch.int32, device="cuda").expand(1, 8, 1000).contiguous()
    lengths = torch.tensor([1000], device="cuda")
    before = weights.clone()
    _, _, w, p, n = shared.cache_evict(t["prefix_key"][None], t["prefix_value"][None], weights[None], positions,
                                       lengths, 64, first=4, recent=8)
    assert int(n[0]) == 64
    for h in range(8):
        best = before[h, 4:992].topk(52).indices + 4
        want = set(range(4)) | set(range(992, 1000)) | set(best.tolist())
        assert set(p[0, h, :64].tolist()) == want
        assert torch.equal(w[0, h, :64], before[h, p[0, h, :64].long()])
