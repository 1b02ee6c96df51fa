"""Calls of the shared-prefix operators that would read or write memory that is
not theirs: refused on the host, before any device is touched."""
import pytest
import torch

from dolittle_b200 import shared


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
