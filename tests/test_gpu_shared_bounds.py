"""Shared-prefix operators at the bounds of what their arguments may be."""
import pytest
import torch

from dolittle_b200 import shared
from tests.test_gpu_shared import make_caches
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
