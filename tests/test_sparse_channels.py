"""What rounding the bounds and the query costs a selection, by the definitions in 64 bits (sparse_ref.py; the
kernels follow them exactly), and what channels give back. Without a GPU."""
import math

import numpy as np
import pytest
import torch

import sparse_ref as ref
import tileinfer_hip as ti

PAGES, P, D, G, KEEP = 512, 64, 128, 4, 64


def powers(channel):
    return 2.0 ** np.clip(np.round(np.log2(channel)), -30, 30)


def kept_by(q, keys, channel):
    """Pages by rounded and by unrounded scores, and what either kind of score holds: q [G][D], keys [pages][P][D]."""
    c = np.ones(D) if channel is None else powers(channel)
    bounds, scale = np.zeros((PAGES, 1, 2, D)), np.zeros((PAGES, 1))
    for i in range(PAGES):
        bounds[i, 0, 0], bounds[i, 0, 1], scale[i, 0] = ref.page_bounds(keys[i] / c)
    table, _ = ref.select(q * c, bounds, scale, np.arange(1, PAGES + 1), PAGES * P - 1, P, KEEP, 0, 1)
    hi, lo = keys.max(1), keys.min(1)
    true = np.maximum(q[:, None] * hi, q[:, None] * lo).sum(2)           # [G][pages]
    order = np.argsort(-true.max(0)[:-1], kind="stable")[:KEEP - 1]      # the last page is kept by either
    return set(table[0].tolist()), set((order + 1).tolist()) | {PAGES}, true, (bounds[:, 0], scale[:, 0], c)


def sample(kind, amp, seed):
    g = np.random.default_rng(seed)
    keys = 0.5 * g.standard_normal((PAGES, 1, D)) + g.standard_normal((PAGES, P, D))
    large = [5, 77]
    if kind == "times":
        keys[:, :, large] *= amp
    else:
        keys[:, :, large] += amp
    return keys, g.standard_normal((8, G, D))


@pytest.mark.parametrize("kind,amp", [("times", 1), ("times", 5), ("times", 10), ("plus", 30), ("plus", 100)])
def test_pages_that_rounding_loses(kind, amp):
    """The pages of the unrounded score that are kept. Few are lost where keys are alike; two large dimensions of 128
    cost up to a third, and channels of the keys' largest magnitudes give most of them back."""
    keys, queries = sample(kind, amp, 3)
    channel = np.abs(keys).max((0, 1))
    share = {}
    for name, c in (("none", None), ("channel", channel)):
        got = [kept_by(q, keys, c)[:2] for q in queries]
        share[name] = np.mean([len(a & b) / KEEP for a, b in got])
    print(kind, amp, share)
    assert share["channel"] >= 0.85
    if amp == 1:
        assert share["none"] >= 0.95
    else:
        assert share["none"] <= 0.9 and share["channel"] >= share["none"] + 0.05


@pytest.mark.parametrize("with_channel", [False, True])
@pytest.mark.parametrize("kind,amp", [("times", 1), ("times", 10), ("plus", 100)])
def test_scores_are_within_the_stated_distances(kind, amp, with_channel):
    """A score is at least the unrounded one less 2^(e - 1) scale sum max |bounds|, at most it and that and
    2^e scale sum |w| more."""
    keys, queries = sample(kind, amp, 4)
    for q in queries[:3]:
        _, _, true, (b, s, c) = kept_by(q, keys, np.abs(keys).max((0, 1)) if with_channel else None)
        for g in range(G):
            e = ref.least_power(np.abs(q[g] * c).max())
            w = np.rint(q[g] * c / e)
            score = np.where(w > 0, w * b[:, 0], w * b[:, 1]).sum(1) * e * s
            near = e / 2 * s * np.maximum(np.abs(b[:, 0]), np.abs(b[:, 1])).sum(1)
            wide = e * s * np.abs(w).sum()
            assert (score >= true[g] - near - 1e-9).all() and (score <= true[g] + near + wide + 1e-9).all()


def test_channel_of_key_bounds():
    """Rounded to powers of two by ratio, spread over the heads; refused where it is not a size."""
    make = lambda c: ti.key_bounds(64, 16, 3, 10, device="cpu", channel=c)
    assert make(None).channel is None
    c = torch.ones(64)
    c[:8] = torch.tensor([1.41, 1.42, 0.5, 0.71, 0.7, 3.0, 1e30, 1e-30])
    kb = make(c)
    assert kb.channel.shape == (3, 64) and kb.channel.dtype == torch.float32 and kb.channel.is_contiguous()
    assert kb.channel[2, :8].tolist() == [1, 2, 0.5, 1, 0.5, 4, 2.0 ** 30, 2.0 ** -30]
    per_head = torch.rand((3, 64)) + 0.01
    assert np.array_equal(make(per_head).channel.numpy(), powers(per_head.double().numpy()))
    for bad in (torch.ones(63), torch.ones((2, 64)), torch.zeros(64), -torch.ones(64), torch.full((64,), math.nan), torch.full((64,), math.inf)):
        with pytest.raises(ti.ArgumentError):
            make(bad)
    cache = ti.PagedKVCache(2, 64, 3, 10, page_size=16, device="cpu", bounds=True, bounds_channel=[c, per_head])
    assert torch.equal(cache.bounds[0].channel, kb.channel) and cache.bounds[1].channel.shape == (3, 64)
