"""The bound on attention outputs tells FP32 weights from weights stored in one BF16 number."""
import math

import pytest
import torch

from tests.attention_bounds import output_bound


@pytest.mark.parametrize("keys,gain", [(2, 1.0), (5, 1.0), (300, 1.5), (2100, 6.0)])
def test_the_bound_admits_fp32_weights_and_rejects_one_bf16_number(keys, gain):
    g = torch.Generator().manual_seed(keys)
    d, heads = 128, 64

    def rand(*shape, k=1.0):
        return (k * torch.randn(shape, generator=g)).bfloat16().double()

    q, k, v = rand(heads, d, k=gain), rand(heads, keys, d), rand(heads, keys, d)
    s = torch.einsum("hd,hnd->hn", q, k) / math.sqrt(d)
    w = torch.softmax(s, -1)
    out, spread = torch.einsum("hn,hnd->hd", w, v), torch.einsum("hn,hnd->hd", w, v.abs())
    size = (torch.einsum("hd,hnd->hn", q.abs(), k.abs()) / math.sqrt(d)).amax(-1)
    bound = output_bound(out, spread, size, keys, d)

    def off(weights):
        return (torch.einsum("hn,hnd->hd", weights, v).bfloat16().double() - out).abs() / bound

    e = torch.exp(s - s.amax(-1, keepdim=True))
    total = e.sum(-1, keepdim=True)
    hi = (e.float().view(torch.int32) & -65536).view(torch.float32)
    lo = ((e.float() - hi).view(torch.int32) & -65536).view(torch.float32)
    assert off(w.float().double()).max() <= 1
    assert off((hi + lo).double() / total).max() <= 1    # two BF16 numbers, both cut off
    assert off(e.bfloat16().double() / total).max() > 1  # one, rounded to nearest
    assert off(hi.double() / total).max() > 1            # one, cut off
