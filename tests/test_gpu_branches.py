"""Branches of one prompt against an engine that runs each branch by itself,
and caches cut by accumulated weight against what the definition keeps."""
import numpy as np
import pytest
import torch

import dolittle_b200 as dl
from dolittle_b200.branches import Branches
from tests import numerics as nm

pytestmark = pytest.mark.gpu

CONFIG = dl.Qwen3Config(hidden=512, query_heads=8, kv_heads=2, head_width=128, mlp_width=1024, vocabulary=1024, layers=3,
                        theta=1e6)


def engine(capacity=512):
    e = dl.Engine(CONFIG, capacity=capacity, max_rows=64)
    e.init_random(3, 0.05)
    return e


def close(got, bits, what):
    """BF16 logits within the tolerance that the fast paths are held to elsewhere."""
    ours = got.float().cpu().numpy()
    theirs = nm.bf16_bits_to_f32(bits)
    peak = float(np.max(np.abs(theirs)))
    r = nm.compare_values(theirs, ours, max(1e-4, 0.0625 * peak), 0.03)
    assert r["passed"] and nm.cosine(theirs, ours) > 0.999, (what, r)


@pytest.mark.parametrize("batch,prompt,turns", [(1, 40, [1, 1]), (3, 150, [1, 5, 1]), (16, 64, [1] * 6), (2, 300, [40, 1])])
def test_branches_match_separate_sequences(batch, prompt, turns):
    rng = np.random.default_rng(batch)
    ids = rng.integers(0, CONFIG.vocabulary, prompt)
    e, alone = engine(), engine()
    e.consume_view(ids)
    b = Branches(e, batch, sum(turns) + 3, weights=batch == 3)
    new = rng.integers(0, CONFIG.vocabulary, (batch, sum(turns)))
    at = 0
    for rows in turns:
        logits = b.step(torch.from_numpy(new[:, at:at + rows]).cuda())
        at += rows
        for s in range(batch):
            alone.reset()
            close(logits[s], alone.consume_view(np.concatenate([ids, new[s, :at]])), (at, s))
    if batch == 3:  # every row's weights sum to one
        total = sum(w.sum().item() for w in b.prefix_weights) + b.suffix_weights.sum().item()
        assert abs(total - CONFIG.layers * batch * at * CONFIG.query_heads) < 1e-3 * total


def test_evicted_branches_attend_what_is_left():
    """A cut of the prompt and of the branches' own caches keeps exactly the
    slots the definition names, and steps go on over what is left."""
    rng = np.random.default_rng(1)
    batch, prompt = 4, 200
    ids = rng.integers(0, CONFIG.vocabulary, prompt)
    e = engine()
    e.consume_view(ids)
    b = Branches(e, batch, 64, weights=True)
    for _ in range(24):
        b.step(torch.from_numpy(rng.integers(0, CONFIG.vocabulary, batch)).cuda())
    sums = [w.clone() for w in b.prefix_weights]
    own = b.suffix_weights.clone()
    keys = [(k.clone(), v.clone()) for k, v in b._prefix]
    b.evict_prefix(64, first=4, recent=16)
    b.evict_suffix(12, recent=4)
    assert b.prefix == 64 and b.length == 12 and b.position == prompt + 24
    assert b._suffix_lengths.tolist() == [12] * batch
    for layer in range(CONFIG.layers):
        for h in range(CONFIG.kv_heads):
            held = b._prefix_positions[layer][0, h].long()
            middle = sums[layer][h, 4:184].topk(64 - 20).indices + 4
            assert set(held.tolist()) == set(range(4)) | set(range(184, 200)) | set(middle.tolist())
            assert torch.equal(b._prefix[layer][0][:, h], keys[layer][0][held, h])
            assert torch.equal(b._prefix[layer][1][:, h], keys[layer][1][held, h])
            for s in range(batch):
                held = b._suffix_positions[layer, s, h, :12].long() - prompt
                best = own[layer, s, h, :20].topk(8).indices
                assert set(held.tolist()) == set(range(20, 24)) | set(best.tolist()), (layer, h, s)
    logits = b.step(torch.from_numpy(rng.integers(0, CONFIG.vocabulary, batch)).cuda())
    assert bool(torch.isfinite(logits.float()).all()) and b.length == 13
    # The prompt's cut is the branches' own copy: the engine's cache is untouched.
    again = Branches(e, 1, 4)
    assert all(torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]) for x, y in zip(again._prefix, keys))


def test_refusals():
    e = engine(64)
    with pytest.raises(ValueError):
        Branches(e, 2, 8)  # nothing consumed yet
    e.consume_view([1, 2, 3])
    b = Branches(e, 2, 2)
    with pytest.raises(ValueError):
        b.step(torch.zeros(3, 1, dtype=torch.int64).cuda())
    with pytest.raises(ValueError):
        b.step(torch.zeros(2, 3, dtype=torch.int64).cuda())
    with pytest.raises(ValueError):
        b.evict_prefix(2)  # no weights were summed
    with pytest.raises(dl.DolittleError):
        e.kv_device(99, False)


@pytest.mark.parametrize("prompt,budget,first,recent", [(200, 256, 4, 200), (3, 64, 4, 0), (40, 40, 4, 36), (5, 1 << 40, 0, 9)])
def test_a_budget_at_or_above_the_prompt_keeps_it(prompt, budget, first, recent):
    """Everything fits the budget: all slots stay, whatever is protected."""
    rng = np.random.default_rng(prompt)
    e = engine()
    e.consume_view(rng.integers(0, CONFIG.vocabulary, prompt))
    b = Branches(e, 2, 8, weights=True)
    ids = torch.from_numpy(rng.integers(0, CONFIG.vocabulary, (2, 3))).cuda()
    b.step(ids[:, 0])
    keys = [(k.clone(), v.clone()) for k, v in b._prefix]
    sums = [w.clone() for w in b.prefix_weights]
    b.evict_prefix(budget, first=first, recent=recent)
    assert b.prefix == prompt and b._prefix_lengths.tolist() == [prompt] * 2
    assert all(torch.equal(x[0], y[0]) and torch.equal(x[1], y[1]) for x, y in zip(b._prefix, keys))
    assert all(torch.equal(x, y) for x, y in zip(b.prefix_weights, sums))
    again = Branches(e, 2, 8)
    again.step(ids[:, 0])
    assert torch.equal(b.step(ids[:, 1]), again.step(ids[:, 1]))


@pytest.mark.parametrize("bad", [-1, CONFIG.vocabulary, (1 << 32) + 5, -(1 << 31), 1 << 40])
def test_ids_outside_the_vocabulary(bad):
    """Refused where the host has them; on the device their branch turns NaN and no other branch changes."""
    rng = np.random.default_rng(2)
    e = engine()
    e.consume_view(rng.integers(0, CONFIG.vocabulary, 30))
    ids = torch.from_numpy(rng.integers(0, CONFIG.vocabulary, (3, 4)))
    wrong = ids.clone()
    wrong[1, 1] = bad
    a, b = Branches(e, 3, 8, weights=True), Branches(e, 3, 8, weights=True)
    with pytest.raises(ValueError, match="vocabulary"):
        b.step(wrong)
    assert b.length == 0 and b.position == 30
    for at, rows in ((0, 1), (1, 2), (3, 1)):
        right = a.step(ids[:, at:at + rows].cuda())
        got = b.step(wrong[:, at:at + rows].cuda())
        assert bool(torch.isfinite(right.float()).all())
        assert torch.equal(got[0::2], right[0::2])
        assert bool(torch.isnan(got[1]).all()) == (at >= 1) and (at >= 1 or torch.equal(got[1], right[1]))
    assert all(bool(torch.isfinite(w).all()) for w in b.prefix_weights)


def test_ids_may_come_from_the_host():
    rng = np.random.default_rng(3)
    e = engine()
    e.consume_view(rng.integers(0, CONFIG.vocabulary, 30))
    ids = rng.integers(0, CONFIG.vocabulary, (2, 3))
    a, b = Branches(e, 2, 8), Branches(e, 2, 8)
    assert torch.equal(a.step(torch.from_numpy(ids).cuda()), b.step(ids))
    assert torch.equal(a.step(torch.from_numpy(ids[:, 0]).int().cuda()), b.step(ids[:, 0].tolist()))


def test_a_closed_engine_is_refused():
    e = engine(64)
    e.consume_view([1, 2, 3])
    b = Branches(e, 2, 4, weights=True)
    b.step([1, 2])
    torch.cuda.synchronize()
    e.close()
    with pytest.raises(ValueError, match="closed"):
        b.step([1, 2])
    with pytest.raises(ValueError, match="closed"):
        b.evict_prefix(8)
    assert b.length == 1
    b.evict_suffix(1, recent=1)  # the branches' own
    assert b.length == 1


def test_branches_are_on_their_engine_s_device(monkeypatch):
    """Wherever the current device points, which here is one that need not exist."""
    e = engine(64)
    e.consume_view([1, 2, 3])
    want = Branches(e, 2, 4).step([1, 2])
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "current_device", lambda: 1)
        b = Branches(e, 2, 4)
    assert b._device == want.device and all(k.device == want.device for k, _ in b._prefix)
    assert torch.equal(b.step([1, 2]), want)
