"""Shared-prefix operators at the bounds of what their arguments may be."""
import pytest
import torch

from dolittle_b200 import _lib, shared
from tests.test_gpu_shared import check_attention, make, make_caches
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
