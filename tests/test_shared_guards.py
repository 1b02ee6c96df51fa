"""Calls of the shared-prefix operators that would read or write memory that is
not theirs: refused on the host, before any device is touched."""
import ctypes as C
import weakref

import pytest
import torch

import dolittle_b200 as dl
from dolittle_b200 import _lib, shared


def cache(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


@pytest.mark.parametrize("batch,rows", [(3, 1), (1, 3), (3, 2)])
def test_one_query_expanded_over_the_tokens_is_refused(batch, rows):
    """All tokens at one address: a token stride of 0, which the C ABI takes for dense rows."""
    q = cache(1, 1, 8, 128).expand(batch, rows, 8, 128)
    key = cache(20, 2, 128)
    lengths = torch.full((batch,), 20)
    with pytest.raises(ValueError, match="stride"):
        shared.attention_shared(q, key, key, None, None, lengths, None)


def test_queries_that_overlap_one_another_are_refused():
    q = torch.as_strided(cache(4096), (3, 1, 8, 128), (512, 512, 128, 1))
    key = cache(20, 2, 128)
    with pytest.raises(ValueError, match="stride"):
        shared.attention_shared(q, key, key, None, None, torch.full((3,), 20), None)


def test_one_token_may_have_any_strides():
    """Strides of dimensions of size 1 are not used: the device is what is refused here."""
    q = torch.as_strided(cache(1024), (1, 1, 8, 128), (0, 0, 128, 1))
    key = cache(20, 2, 128)
    with pytest.raises(ValueError, match="CUDA"):
        shared.attention_shared(q, key, key, None, None, torch.full((1,), 20), None)


# ---------------------------------------------------------------------------
# Eviction through the C ABI; the addresses are never read.
# ---------------------------------------------------------------------------
P = 1 << 30


def eviction(apart, **change):
    """Three caches of 100 slots, 2 heads of 64; values `apart` elements after the keys, all in place."""
    e = _lib.CacheEviction(3, 2, 64, 100, 50, 0, 0, P, P + 2 * apart, 128, 12800, 2 * P, 3 * P, 4 * P, P, P + 2 * apart,
                           100, 128, 12800, 2 * P, 3 * P, 4 * P)
    for k, v in change.items():
        setattr(e, k, v)
    return e


FRESH = dict(weights_out=6 * P, positions_out=7 * P, lengths_out=8 * P)


@pytest.mark.parametrize("apart,change", [
    # in place: every cache at one address, or a slot of one where another's lies
    (1 << 20, dict(out_cache_stride=0)),
    (1 << 20, dict(out_cache_stride=64)),
    (1 << 20, dict(out_cache_stride=99 * 128)),
    (64, dict(out_row_stride=256, out_cache_stride=25600)),
    (12800, {}),  # the values are the next cache's keys
    # into other buffers (50 slots): the same, and values over keys
    (1 << 20, dict(key_out=9 * P, value_out=10 * P, out_cache_stride=0, **FRESH)),
    (1 << 20, dict(key_out=9 * P, value_out=10 * P, out_cache_stride=49 * 128, **FRESH)),
    (1 << 20, dict(key_out=9 * P, value_out=9 * P, **FRESH)),
    (1 << 20, dict(key_out=9 * P, value_out=9 * P + 2 * 49 * 128, **FRESH)),
    (1 << 20, dict(key_out=9 * P + 2 * 12800, value_out=9 * P, **FRESH)),
])
def test_evictions_whose_output_rows_overlap_are_refused(apart, change):
    e = eviction(apart, **change)
    if e.key_out == e.key:
        e.row_stride, e.cache_stride = e.out_row_stride, e.out_cache_stride
    L = dl.lib()
    assert L.dl_cache_evict(C.byref(e), P, None) == _lib.DL_INVALID_ARGUMENT
    assert b"rows overlap" in L.dl_last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the calls would be made")
@pytest.mark.parametrize("apart,change", [
    (1 << 20, {}),
    (0, {}),                                                        # keys that are the values
    (128, dict(out_row_stride=256, out_cache_stride=25600)),        # keys and values of a position side by side
    (1 << 20, dict(out_row_stride=3 * 128, out_cache_stride=128)),  # the caches' slots side by side
    (3 * 128, dict(out_row_stride=6 * 128, out_cache_stride=128)),  # both
    (1 << 20, dict(caches=1, out_cache_stride=0)),
    (1 << 20, dict(key_out=9 * P, value_out=9 * P + 2 * 128, out_row_stride=256, out_cache_stride=25600, **FRESH)),
    (1 << 20, dict(key_out=9 * P, value_out=10 * P, out_cache_stride=49 * 128 + 128, **FRESH)),
    (1 << 20, dict(key_out=9 * P, value_out=9 * P + 2 * 50 * 128, **FRESH)),  # in each other's free slots
])
def test_evictions_into_rows_of_their_own_are_not_refused(apart, change):
    """Without a device they come as far as the launch."""
    e = eviction(apart, **change)
    if e.key_out == e.key:
        e.row_stride, e.cache_stride = e.out_row_stride, e.out_cache_stride
    L = dl.lib()
    assert L.dl_cache_evict(C.byref(e), P, None) == _lib.DL_CUDA_ERROR, L.dl_last_error()


@pytest.mark.parametrize("change", [
    dict(lengths_out=4 * P + 8),            # moved by one cache: a block may still read what another writes
    dict(lengths_out=2 * P),                # the weights'
    dict(lengths_out=3 * P + 4 * 599),      # the last position
    dict(weights_out=6 * P, positions_out=6 * P, key_out=9 * P, value_out=10 * P),
    dict(weights_out=3 * P + 2000, positions_out=7 * P, key_out=9 * P, value_out=10 * P),
    dict(weights_out=4 * P, positions_out=7 * P, key_out=9 * P, value_out=10 * P),
])
def test_sums_positions_and_lengths_that_overlap_are_refused(change):
    L = dl.lib()
    assert L.dl_cache_evict(C.byref(eviction(1 << 20, **change)), P, None) == _lib.DL_INVALID_ARGUMENT
    assert b"overlap" in L.dl_last_error()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the calls would be made")
@pytest.mark.parametrize("change", [
    dict(lengths_out=4 * P + 24),  # right behind the lengths
    dict(key_out=9 * P, value_out=10 * P, weights_out=6 * P, positions_out=7 * P, lengths_out=4 * P),
])
def test_lengths_beside_or_in_place_are_not_refused(change):
    L = dl.lib()
    assert L.dl_cache_evict(C.byref(eviction(1 << 20, **change)), P, None) == _lib.DL_CUDA_ERROR, L.dl_last_error()


# ---------------------------------------------------------------------------
# Attention through the C ABI; the addresses are never read.
# ---------------------------------------------------------------------------
def attention(output, query_stride=0, output_stride=0):
    """Three sequences of two tokens, 4 heads of 64 (256 elements a token), query at P."""
    a = _lib.SharedAttention(3, 2, 4, 2, 64, query_stride, output_stride, 2 * P, 3 * P, 100, 128, 4 * P, 5 * P, 6 * P, 50,
                             128, 6400, 7 * P)
    L = dl.lib()
    return L.dl_attention_shared(C.byref(a), P, output, None, None, None, 8 * P, None), L.dl_last_error()


@pytest.mark.parametrize("output,strides", [
    (P, (0, 0)),                        # in place
    (P + 2 * 256, (0, 0)),              # over the next token
    (P + 2 * (6 * 256 - 8), (0, 0)),    # the last token's end
    (P - 2 * 248, (0, 0)),
    (P + 2 * 256, (504, 504)),          # between the tokens of a fused row, eight elements too far
    (P, (512, 256)),                    # dense over the tokens of a fused row
    (P + 2 * 5 * 512, (512, 0)),
])
def test_outputs_over_the_query_are_refused(output, strides):
    status, reason = attention(output, *strides)
    assert status == _lib.DL_INVALID_ARGUMENT and b"overlaps the query" in reason


@pytest.mark.skipif(torch.cuda.is_available(), reason="the calls would be made")
@pytest.mark.parametrize("output,strides", [
    (P + 2 * 6 * 256, (0, 0)),       # right behind the query
    (P + 2 * 256, (512, 512)),       # the other half of each fused row
    (P - 2 * 256, (512, 512)),
    (P + 2 * (5 * 512 + 256), (512, 0)),
])
def test_outputs_beside_the_query_are_not_refused(output, strides):
    assert attention(output, *strides)[0] == _lib.DL_CUDA_ERROR


# ---------------------------------------------------------------------------
# Output sequences that keep nothing
# ---------------------------------------------------------------------------
class MadeOnAccess:
    """Five elements, each made when it is asked for; counts those that went away before the call was over."""

    def __init__(self, *make):
        self.make, self.alive, self.lost = make, [], 0

    def __len__(self):
        return len(self.make)

    def __getitem__(self, i):
        self.lost += sum(r() is None for r in self.alive)
        x = self.make[i]()
        self.alive.append(weakref.ref(x))
        return x


def test_outputs_of_an_eviction_are_held_until_it_returns():
    """The call comes as far as the device's check here; every element made so far is alive until then."""
    t = cache(1, 8, 2, 64)
    out = MadeOnAccess(*[lambda: cache(1, 4, 2, 64)] * 5)
    with pytest.raises(ValueError, match="CUDA"):
        shared.cache_evict(t, t.clone(), None, None, None, 4, out=out)
    assert len(out.alive) == 5 and out.lost == 0
    assert all(r() is None for r in out.alive)  # and given back afterwards
