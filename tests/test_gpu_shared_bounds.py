"""Shared-prefix operators at the bounds of what their arguments may be."""
import pytest
import torch

from dolittle_b200 import _lib, shared
from tests.attention_bounds import output_bound
from tests.test_gpu_shared import check_attention, make, make_caches, reference
from tests.test_shared_guards import MadeOnAccess

pytestmark = pytest.mark.gpu

NAMES = ("key", "value", "weights", "positions", "lengths")


def test_eviction_into_outputs_that_a_sequence_makes_on_access():
    c = make_caches(2, 64, lengths=[64, 40])
    args = [c[k] for k in NAMES]
    out = MadeOnAccess(*[lambda x=x: torch.zeros_like(x) for x in args])
    got = shared.cache_evict(*args, 16, recent=3, out=out)
    want = shared.cache_evict(*[x.clone() for x in args], 16, recent=3)
    assert out.lost == 0 and got[4].tolist() == [16, 16]
    assert all(torch.equal(x[:, :16], y[:, :16]) for x, y in zip(got[:2], want[:2]))
    assert all(torch.equal(x[..., :16], y[..., :16]) for x, y in zip(got[2:4], want[2:4]))


@pytest.mark.parametrize("batch,rows,prefix,suffix,hq,hkv,d,slens", [
    (5, 1, 300, 70, 32, 8, 128, [70, 69, 1, 0, 33]),   # the few-row kernel alone
    (20, 1, 3000, 200, 32, 8, 128, None),              # beside tiles over the prefix
    (3, 40, 260, 300, 28, 4, 64, [300, 40, 211]),      # tiles over both
    (2, 129, None, 400, 8, 8, 128, [400, 333]),
])
def test_one_suffix_cache_expanded_over_the_sequences(batch, rows, prefix, suffix, hq, hkv, d, slens):
    """Every sequence reads the same suffix rows (a sequence stride of 0), as far as its own length goes."""
    t = make(batch, rows, prefix, suffix, hq, hkv, d, seed=batch, slens=slens)
    for part in ("key", "value"):
        longest = max(range(batch), key=lambda b: int(t["suffix_lengths"][b]))
        t[f"suffix_{part}"] = t[f"suffix_{part}"][longest:longest + 1].expand(batch, -1, -1, -1)
        assert t[f"suffix_{part}"].stride(0) == 0
    check_attention(t)


def test_refusals_carry_the_library_s_status():
    """What is unsupported is told from what is invalid, as the C ABI does."""
    key = torch.zeros(16, 8, 96, device="cuda", dtype=torch.bfloat16)
    lengths = torch.full((2,), 16, device="cuda")

    def status(call, *args, **kw):
        with pytest.raises(_lib.DolittleError) as e:
            call(*args, **kw)
        return e.value.status, str(e.value)

    q = torch.zeros(2, 1, 32, 96, device="cuda", dtype=torch.bfloat16)
    got = status(shared.attention_shared, q, key, key, None, None, lengths, None)
    assert got[0] == _lib.DL_UNSUPPORTED and "head width" in got[1]
    got = status(shared.attention_shared, q[:, :0], key, key, None, None, lengths, None)
    assert got[0] == _lib.DL_INVALID_ARGUMENT and "empty" in got[1]
    c = make_caches(2, 64)
    args = [c[k] for k in NAMES]
    got = status(shared.cache_evict, *args, 0)
    assert got[0] == _lib.DL_INVALID_ARGUMENT and "empty" in got[1]
    odd = torch.zeros((2, 64, 2, 12), device="cuda", dtype=torch.bfloat16)
    got = status(shared.cache_evict, odd, odd.clone(), *args[2:], 16)
    assert got[0] == _lib.DL_UNSUPPORTED and "multiples of 8" in got[1]


@pytest.mark.parametrize("batch,rows,prefix,suffix,hq,hkv,d,gain", [
    (3, 1, 2, 3, 32, 8, 128, 1.0),        # the few-row kernel alone, a handful of keys
    (4, 2, 3, None, 28, 4, 64, 1.0),
    (2, 1, 256, 64, 32, 8, 128, 1.5),
    (16, 1, 2048, 64, 32, 8, 128, 6.0),   # beside pooled tiles; a few keys take nearly everything
    (32, 1, 1500, 200, 32, 8, 128, 1.5),
    (3, 60, 2, 63, 32, 8, 128, 1.0),      # tiles per sequence
    (2, 64, 1000, 64, 32, 8, 128, 6.0),
    (8, 150, 300, 200, 16, 4, 64, 1.5),
])
def test_output_keeps_fp32_weights(batch, rows, prefix, suffix, hq, hkv, d, gain):
    t = make(batch, rows, prefix, suffix, hq, hkv, d, seed=batch + rows, gain=gain)
    out, _, _, _, spread, size = reference(t)
    got, _ = shared.attention_shared(*[t[k] for k in ("query", "prefix_key", "prefix_value", "suffix_key", "suffix_value",
                                                      "prefix_lengths", "suffix_lengths")])
    off = (got.double() - out).abs() / output_bound(out, spread, size, prefix + (suffix or 0), d)
    assert bool((off <= 1).all()), off.max().item()


@pytest.mark.parametrize("room", [2000, 8000])
@pytest.mark.parametrize("batch,rows,prefix,suffix,hq,hkv,d,plens,slens", [
    (2, 1, 256, 64, 32, 8, 128, None, [64, 1]),
    (16, 1, 64, 50, 32, 8, 128, None, [50] * 15 + [0]),
    (32, 1, 2500, 60, 32, 8, 128, None, None),
    (5, 1, 700, 30, 28, 4, 64, [700, 0, 1, 129, 699], None),
    (4, 8, 500, 40, 32, 8, 128, None, [40, 8, 7, 1]),
    (3, 48, 600, 60, 32, 8, 128, None, [60, 48, 49]),
    (2, 130, 129, 130, 8, 2, 64, None, None),
])
def test_caches_with_room_to_grow(batch, rows, prefix, suffix, hq, hkv, d, plens, slens, room):
    """Plans are made from capacities; lengths far below them change the answer no more than anything else."""
    check_attention(make(batch, rows, prefix, suffix, hq, hkv, d, seed=batch, plens=plens, slens=slens, room=room))


@pytest.mark.parametrize("batch,rows,hq,hkv,d", [(2, 1, 32, 8, 128), (70, 3, 28, 4, 64), (3, 100, 8, 8, 128),
                                                 (40, 300, 16, 2, 128)])
def test_caches_without_any_position(batch, rows, hq, hkv, d):
    """Both sides of capacity 0: every row is empty."""
    q = torch.randn(batch, rows, hq, d, device="cuda").to(torch.bfloat16)
    prefix = torch.empty(0, hkv, d, device="cuda", dtype=torch.bfloat16)
    suffix = torch.empty(batch, 0, hkv, d, device="cuda", dtype=torch.bfloat16)
    lengths = torch.full((batch,), 9, device="cuda")
    for p, s in ((prefix, suffix), (prefix, None), (None, suffix)):
        out, lse = shared.attention_shared(q, p, p, s, s, None if p is None else lengths, None if s is None else lengths)
        assert bool((out == 0).all()) and bool((lse == -torch.inf).all())


@pytest.mark.parametrize("n,capacity,budget", [(2, 320, 256), (40, 300, 200), (1, 20000, 9000)])
def test_inputs_of_an_eviction_into_other_buffers_are_only_read(n, capacity, budget):
    c = make_caches(n, capacity, lengths=[capacity - b for b in range(n)])
    c["weights"][:, :, ::5] = torch.nan
    args = [c[k] for k in NAMES]
    before = [x.clone() for x in args]
    shared.cache_evict(*args, budget, first=2, recent=9, out=[torch.empty_like(x) for x in args])
    for k, x, y in zip(NAMES, args, before):
        x, y = (z.view(torch.int32) if z.dtype == torch.float32 else z for z in (x, y))
        assert torch.equal(x, y), k


def test_caches_expanded_from_one_are_evicted_into_others_only():
    """Read from one place into three: right; in place: refused, and nothing is written."""
    c = make_caches(1, 90, lengths=[90])
    args = [c["key"].expand(3, -1, -1, -1), c["value"].expand(3, -1, -1, -1), torch.rand(3, 2, 90, device="cuda"),
            c["positions"].expand(3, -1, -1).contiguous(), torch.tensor([90, 50, 0], device="cuda")]
    key = c["key"].clone()
    with pytest.raises(_lib.DolittleError, match="overlap"):
        shared.cache_evict(*args, 30)
    assert torch.equal(c["key"], key)
    got = shared.cache_evict(*args, 30, out=[torch.zeros_like(x.contiguous()) for x in args])
    want = shared.cache_evict(*[x.clone(memory_format=torch.contiguous_format) for x in args], 30)
    for i, n in enumerate((30, 30, 0)):
        assert all(torch.equal(x[i, :n], y[i, :n]) for x, y in zip(got[:2], want[:2]))
        assert all(torch.equal(x[i, :, :n], y[i, :, :n]) for x, y in zip(got[2:4], want[2:4]))
    assert got[4].tolist() == want[4].tolist() == [30, 30, 0]


def test_queries_and_outputs_that_share_memory_are_refused():
    t = make(2, 3, 40, 10, seed=4)
    args = [t[k] for k in ("query", "prefix_key", "prefix_value", "suffix_key", "suffix_value", "prefix_lengths",
                           "suffix_lengths")]
    with pytest.raises(_lib.DolittleError, match="overlaps the query"):
        shared.attention_shared(*args, out=t["query"])
    one = t["query"][:1, :1].expand(2, 3, 32, 128)
    with pytest.raises(ValueError, match="stride"):
        shared.attention_shared(one, *args[1:])
    got, _ = shared.attention_shared(one.contiguous(), *args[1:])
    want, _, _, _, spread, size = reference({**t, "query": one})
    assert bool(((got.double() - want).abs() <= output_bound(want, spread, size, 50, 128)).all())
