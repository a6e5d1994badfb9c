"""Bounds and selection with channels against their definitions in 64 bits, exactly."""
import math

import numpy as np
import pytest
import torch

import sparse_ref as ref
import tileinfer_hip as ti
from test_gpu_sparse import T, Cache, i32, offsets, positions, random_bounds, tables_for

pytestmark = pytest.mark.gpu
BE = ti.HipBackend()


def channel_of(H, D, seed, per_head=True):
    g = torch.Generator().manual_seed(seed)
    c = torch.exp2(torch.randint(-4, 5, (H, D), generator=g).float())
    c[:, 3], c[:, D - 1] = 2.0 ** 12, 2.0 ** -9
    return c if per_head else c[0]


@pytest.mark.parametrize("kv", ["bf16", "fp32", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("P", [5, 16, 64])
def test_bounds(gpu, kv, D, P):
    """Each key divided by its channel, a key that is not finite among them; a step that begins inside a page."""
    starts, counts = [0, 3, 64, 130], [1, 70, 33, 9]
    c = Cache(kv, D, 3, P, [s + n for s, n in zip(starts, counts)], seed=P + D)
    channel = channel_of(3, D, P)
    if kv != "int8":
        c.k[c.rows[2][70 // P] - 1, 1, 70 % P, 5] = math.inf
        c.hk[c.rows[2][70 // P] - 1, 1, 70 % P, 5] = math.inf
    kb = ti.key_bounds(D, P, 3, c.pages, channel=channel)
    ti.update_key_bounds_(BE, kb, c.k, c.v, c.tables, positions(starts, counts), offsets(counts), max(counts))
    bounds, scale = np.zeros((c.pages, 3, 2, D)), np.zeros((c.pages, 3))
    part = channel.double().numpy()
    for b, (s, n) in enumerate(zip(starts, counts)):
        ref.update_bounds(bounds, scale, lambda i, h, m: c.key_at(i, h, m) / part[h], c.tables[b].tolist(), s, n, P, 3, c.pages)
    assert np.array_equal(kb.bounds.cpu().numpy(), bounds)
    assert np.array_equal(kb.scale.cpu().numpy().astype(np.float64), scale)


@pytest.mark.parametrize("G", [1, 3, 4, 16, 24])
@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp32", 64)])
@pytest.mark.parametrize("per_head", [True, False])
def test_selection(gpu, G, dtype, D, per_head):
    """Each query times its head's channel; heads whose product is not finite count for nothing."""
    starts, counts, P, H, pages = [0, 1000, 37, 500], [9, 1, 21, 5], 16, 2, 90
    tables = tables_for([s + n for s, n in zip(starts, counts)], P, pages, G)
    plain, channel = random_bounds(pages, H, D, P, G), channel_of(H, D, G, per_head)
    kb = ti.KeyBounds(plain.bounds, plain.scale, P, channel)
    torch.manual_seed(G)
    q = torch.randn((sum(counts), H * G, D), device="cuda", dtype=T[dtype])
    q[4, 0, 3] = 2e38                                   # finite, times 2^12 not
    q[5] *= 1e30
    pos = positions(starts, counts)
    out, lengths = ti.select_pages(BE, q, kb, tables, pos, 12, 1, 2, True, offsets(counts), max(counts))
    c = channel.double().expand(H, D).repeat_interleave(G, 0).numpy()
    x = q.double().cpu().numpy() * c
    x[np.abs(x) > np.finfo(np.float32).max] = np.inf
    b, s = kb.bounds.cpu().numpy(), kb.scale.cpu().numpy()
    row = 0
    for i, (start, n) in enumerate(zip(starts, counts)):
        for t in range(n):
            want, want_len = ref.select(x[row], b, s, tables[i].tolist(), start + t, P, 12, 1, 2)
            assert np.array_equal(out[row].cpu().numpy(), want) and np.array_equal(lengths[row].cpu().numpy(), want_len), row
            row += 1
    # ones are none
    ones = ti.KeyBounds(plain.bounds, plain.scale, P, torch.ones(D))
    for a, b in zip(ti.select_pages(BE, q, plain, tables, pos, 12, 1, 2, True, offsets(counts), max(counts)),
                    ti.select_pages(BE, q, ones, tables, pos, 12, 1, 2, True, offsets(counts), max(counts))):
        assert torch.equal(a, b)


def test_large_dimensions_keep_their_pages(gpu):
    """Keys of which two dimensions are ten times as large, through the cache: with channels of the keys' largest
    magnitudes most pages of the unrounded score are kept, without them more are lost."""
    P, H, D, pages, keep = 64, 2, 128, 256, 32
    c = Cache("bf16", D, H, P, [pages * P], seed=61, spare=0)
    torch.manual_seed(61)
    c.k.add_(0.5 * torch.randn((pages, H, 1, D), device="cuda"))
    c.k[..., [5, 77]] *= 10
    q = torch.randn((16, H * 4, D), device="cuda", dtype=torch.bfloat16)
    pos = i32([pages * P - 1] * 16)
    k = c.k.double()
    qd = q.double().view(16, H, 4, 1, D)
    hi, lo = k.amax(2).transpose(0, 1)[:, None], k.amin(2).transpose(0, 1)[:, None]
    true = torch.maximum(qd * hi, qd * lo).sum(-1).amax(2)                    # [tokens][H][pages]
    true[:, :, c.rows[0][-1] - 1] = math.inf                                 # kept by either
    want = true.topk(keep, 2).indices.sort(2).values + 1
    share = {}
    for name, channel in (("none", None), ("channel", k.abs().amax((0, 2)))):
        kb = ti.key_bounds(D, P, H, pages, channel=channel)
        ti.update_key_bounds_(BE, kb, c.k, c.v, c.tables, positions([0], [pages * P]), max_query_len=pages * P)
        got, _ = ti.select_pages(BE, q, kb, c.tables.expand(16, -1).contiguous(), pos, keep, 0, 1)
        share[name] = (got[..., None] == want[:, :, None]).any(-1).float().mean().item()
    assert share["channel"] >= 0.85 and share["channel"] >= share["none"] + 0.05, share


def test_refusals(gpu):
    kb = ti.key_bounds(64, 16, 2, 20, channel=torch.full((64,), 4.0))
    k = torch.zeros((20, 2, 16, 64), device="cuda", dtype=torch.bfloat16)
    q, tables, pos = torch.zeros((1, 2, 64), device="cuda", dtype=torch.bfloat16), i32([[1, 2]]), i32([20])
    ti.update_key_bounds_(BE, kb, k, k, tables, pos)
    ti.select_pages(BE, q, kb, tables, pos, 4)
    good = kb.channel
    for bad in (good[:1], good.double(), good.cpu(), good.t().contiguous(), good.t()):
        kb.channel = bad
        with pytest.raises(ti.ArgumentError):
            ti.update_key_bounds_(BE, kb, k, k, tables, pos)
        with pytest.raises(ti.ArgumentError):
            ti.select_pages(BE, q, kb, tables, pos, 4)
