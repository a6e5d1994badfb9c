"""Edges of the chosen-page operators over steps of several tokens: lengths at the ends of their type, tokens
without keys, garbage in whatever a table does not name."""
import math

import numpy as np
import pytest
import torch

import sparse_ref as ref
import tileinfer_hip as ti
from test_gpu_sparse import Cache, T, check_attend, i32, offsets, positions, random_bounds, shared

pytestmark = pytest.mark.gpu
BE = ti.HipBackend()


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp32"])
@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("width", [7, 24])
def test_lengths_at_the_ends_of_their_type(gpu, kv, rows, width):
    """Negative lengths down to the lowest are none, longer than the table is all of it: token by token and in
    groups, in launches whose keys one work-group takes (7 pages) and several share (24)."""
    c = Cache(kv, 128, 8, 16, [900], seed=51)
    torch.manual_seed(51)
    q = torch.randn((rows, 32, 128), device="cuda", dtype=T[kv])
    tables, lengths = shared(c, rows, width, seed=51)
    lengths[0] = i32([-1, -2 ** 31, -2 ** 31 + 1, -2 ** 31 + 16, 2 ** 31 - 1, -2 ** 31 + 16 * width, -2 ** 30, 0])
    lengths[rows // 2, :3] = i32([-2 ** 31, 2 ** 31 - 1, -2 ** 31 + 17])
    for n in (1, rows):
        check_attend(c, q, tables, lengths, n=n)
    lengths.fill_(-2 ** 31)
    for n in (1, rows):
        assert (check_attend(c, q, tables, lengths, n=n) == 0).all()


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp32"])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("rows,heads,width", [(6, 2, 7), (6, 2, 8), (300, 8, 7)])
def test_tokens_without_keys_whose_queries_are_not_finite(gpu, kv, value, rows, heads, width):
    """Rows that pad a batch: no keys and whatever their memory holds as queries, beside tokens with keys. They
    get zeros, the others what they get beside queries of zeros."""
    c = Cache(kv, 128, heads, 16, [60 * 16], seed=52)
    torch.manual_seed(52)
    q = torch.randn((rows, heads * 4, 128), device="cuda", dtype=T[kv])
    tables, lengths = shared(c, rows, width, seed=52)
    lengths[:] = width * 16                    # whole pages: no tile is masked for the others' sake
    pad = torch.arange(rows, device="cuda") % 5 == 3
    lengths[pad] = 0
    q[pad] = 0
    want = ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.09, None, rows)
    q[pad, :, 17] = value
    got = ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.09, None, rows)
    assert (got[pad] == 0).all()
    if kv == "int8":                           # the same operations on the same numbers
        assert torch.equal(got[~pad], want[~pad])
    else:                                      # weights rounded or not (2^-8 each, their sum too), the output (2^-8)
        tol = 2 * 3 * 2.0 ** -8 * c.v.float().abs().max()
        assert ((got[~pad] - want[~pad]).float().abs() <= tol).all()
    if rows == 6:
        check_attend(c, q, tables, lengths, n=rows)


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp32"])
def test_one_workspace_for_all_batches(gpu, kv):
    """Made for the largest batch and block, used by every smaller call, whatever they split."""
    c = Cache(kv, 128, 8, 16, [40 * 16], seed=54)
    torch.manual_seed(54)
    q = torch.randn((48, 32, 128), device="cuda", dtype=T[kv])
    tables, lengths = shared(c, 48, 30, seed=54)
    ws = ti.sparse_attention_workspace(BE, q, c.k, tables, 16)
    for rows in (48, 33, 32, 31, 16, 15, 4, 1):
        for n in (1, 4, 16):
            for width in (30, 9):
                if rows % n:
                    continue
                t, m = tables[:rows, :, :width].contiguous(), lengths[:rows].clamp(max=16 * width)
                out = torch.empty_like(q[:rows])
                ti.sparse_attention_(BE, out, ws, q[:rows], c.k, c.v, t, m, 0.09, None, n)
                assert torch.equal(out, ti.sparse_attention(BE, q[:rows], c.k, c.v, t, m, 0.09, None, n))


@pytest.mark.parametrize("G,D", [(4, 64), (20, 64)])
def test_selection_in_parts(gpu, G, D):
    """Tables wider than LDS holds and more tokens than the workspace: worked on in parts, which begin inside a
    tile and a sequence; each sequence alone (one part) gives the same."""
    P, pages, H, width = 1, 3000, 8, 34000
    counts, starts = [67, 1, 0, 70, 5, 66, 130], [33000, 20, 0, 30000, 33990, 100, 33500]
    total, spare = sum(counts), 3
    g = torch.Generator().manual_seed(55)
    tables = torch.randint(1, pages + 1, (len(counts), width), generator=g, dtype=torch.int32).cuda()
    kb = random_bounds(pages, H, D, P, 55)
    torch.manual_seed(55)
    q = torch.randn((total + spare, H * G, D), device="cuda", dtype=torch.bfloat16)
    pos = torch.cat([positions(starts, counts), i32([0] * spare)])
    out = torch.full((total + spare, H, 40), -5, dtype=torch.int32, device="cuda")
    lengths = torch.full((total + spare, H), -5, dtype=torch.int32, device="cuda")
    ws = ti.select_pages_workspace(BE, q, kb, tables)
    assert ws.numel() < (total * H * width * 4) // 2
    ti.select_pages_(BE, out, lengths, ws, q, kb, tables, pos, 2, 3, True, offsets(counts), max(counts))
    row = 0
    for b, n in enumerate(counts):
        for t0 in range(0, n, 65):
            m = min(65, n - t0)
            a = slice(row + t0, row + t0 + m)
            want = ti.select_pages(BE, q[a], kb, tables[b:b + 1], pos[a], 40, 2, 3, True, None, m)
            assert torch.equal(out[a], want[0]) and torch.equal(lengths[a], want[1])
        row += n
    assert (out[row:] == -5).all() and (lengths[row:] == -5).all()
    hb, hs, ht = kb.bounds.cpu().numpy(), kb.scale.cpu().numpy(), tables.cpu().numpy()
    for r, b, t in ((0, 0, 0), (140, 4, 2), (total - 1, 6, 129)):
        want, want_len = ref.select(q[r].double().cpu().numpy(), hb, hs, ht[b], starts[b] + t, P, 40, 2, 3)
        assert np.array_equal(out[r].cpu().numpy(), want) and np.array_equal(lengths[r].cpu().numpy(), want_len)


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp32"])
@pytest.mark.parametrize("n", [1, 6])
@pytest.mark.parametrize("P", [8, 16, 64])
def test_garbage_in_pages_that_no_key_is_in(gpu, kv, n, P):
    """NaN and infinities behind each row's last key, in the pages of the entries behind it, in the first page (that
    of zero entries) and in every page that no table names."""
    c = Cache(kv, 128, 2, P, [100 * P], seed=53)
    torch.manual_seed(53)
    q = torch.randn((6, 8, 128), device="cuda", dtype=T[kv])
    ids = torch.randperm(c.pages - 1, generator=torch.Generator().manual_seed(53)) + 2    # not the first page
    tables = torch.zeros((6, 2, 8), dtype=torch.int32)
    for r in range(6):
        tables[r, :, :4] = ids[3 * r:3 * r + 4]        # neighbours share one
        tables[r, :, 4] = ids[30 + r]                  # 5 keys, then garbage
        tables[r, :, 5] = ids[40 + r]                  # garbage; then two entries of zero
    tables, lengths = tables.cuda(), torch.full((6, 2), 4 * P + 5, dtype=torch.int32, device="cuda")
    used = torch.zeros(c.pages, dtype=torch.bool)
    used[tables[:, :, :5].cpu().long().reshape(-1) - 1] = True
    assert not used[0] and not used[tables[:, :, 5].cpu().long() - 1].any() and (~used).sum() > 50
    last = tables[:, 0, 4].long() - 1
    keys, values = (c.k.scale, c.v.scale) if kv == "int8" else (c.k, c.v)
    for i, (a, b) in enumerate([(math.nan, math.inf), (math.inf, math.nan), (-math.inf, math.nan)]):
        keys[~used.cuda()], values[~used.cuda()] = a, b
        keys[last, :, 5:], values[last, :, 5:] = a, b
        check_attend(c, q, tables, lengths, n=n)


@pytest.mark.parametrize("kv", ["bf16", "fp32"])
@pytest.mark.parametrize("rows,heads,width", [(6, 2, 7), (6, 2, 24), (300, 8, 8), (64, 64, 4)])
def test_queries_of_tokens_without_keys_are_not_read(gpu, kv, rows, heads, width):
    """NaN there does not send the other tokens of a group, of 16, 32 and 64 rows, down the row by row path, which
    rounds otherwise and is a hundred times as slow: they get the same bits as beside queries of zeros."""
    c = Cache(kv, 128, heads, 16, [60 * 16], seed=56)
    torch.manual_seed(56)
    q = torch.randn((rows, heads * 4, 128), device="cuda", dtype=T[kv])
    tables, lengths = shared(c, rows, width, seed=56)
    pad = torch.arange(rows, device="cuda") % 3 == 1
    lengths[pad] = i32([0, -1] * (heads // 2))
    q[pad] = 0
    want = ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.09, None, rows)
    q[pad] = math.nan
    got = ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.09, None, rows)
    assert torch.equal(got, want) and (got[pad] == 0).all()


@pytest.mark.parametrize("P,width", [(16, 1500), (1, 33500)])
def test_selection_with_many_rows_of_no_sequence(gpu, P, width):
    """A few tokens far behind the start of an array of 3000 rows, over tables that take two launches (with and
    without LDS for a tile's keys): the same as those tokens alone, the other rows as they were."""
    pages, H, first, counts = 4000, 8, 1700, [3, 0, 2, 1]
    starts = [width * P - 4, 0, 50, width * P // 2]
    g = torch.Generator().manual_seed(57)
    tables = torch.randint(1, pages + 1, (4, width), generator=g, dtype=torch.int32).cuda()
    kb = random_bounds(pages, H, 64, P, 57)
    torch.manual_seed(57)
    rows, n = 3000, sum(counts)
    q = torch.randn((rows, H * 4, 64), device="cuda", dtype=torch.bfloat16)
    pos = torch.zeros(rows, dtype=torch.int32, device="cuda")
    pos[first:first + n] = positions(starts, counts)
    out = torch.full((rows, H, 20), -5, dtype=torch.int32, device="cuda")
    lengths = torch.full((rows, H), -5, dtype=torch.int32, device="cuda")
    ws = ti.select_pages_workspace(BE, q, kb, tables)
    ti.select_pages_(BE, out, lengths, ws, q, kb, tables, pos, 1, 2, True, offsets(counts) + first, 3)
    a = slice(first, first + n)
    want = ti.select_pages(BE, q[a], kb, tables, pos[a], 20, 1, 2, True, offsets(counts), 3)
    assert torch.equal(out[a], want[0]) and torch.equal(lengths[a], want[1])
    assert (out[:first] == -5).all() and (out[first + n:] == -5).all() and (lengths[:first] == -5).all()
    hb, hs, ht = kb.bounds.cpu().numpy(), kb.scale.cpu().numpy(), tables.cpu().numpy()
    for r, b, t in ((0, 0, 0), (4, 2, 1), (5, 3, 0)):
        table, length = ref.select(q[first + r].double().cpu().numpy(), hb, hs, ht[b], starts[b] + t, P, 20, 1, 2)
        assert np.array_equal(want[0][r].cpu().numpy(), table) and np.array_equal(want[1][r].cpu().numpy(), length)


def shifted(x, by=1):
    """The same values, `by` elements behind an aligned address."""
    flat = torch.empty(x.numel() + by, dtype=x.dtype, device=x.device)
    flat[by:] = x.reshape(-1)
    return flat[by:].view(x.shape)


@pytest.mark.parametrize("kv", ["bf16", "fp32", "int8"])
@pytest.mark.parametrize("rows", [1, 20])
def test_tensors_aligned_to_their_elements_only(gpu, kv, rows):
    """Queries, outputs, pools, tables, positions and probabilities that begin one element behind an aligned address
    (workspaces and bounds have to be aligned): the bits of aligned ones."""
    D, H, P = 128, 2, 16
    c = Cache(kv, D, H, P, [600], seed=58)
    torch.manual_seed(58)
    q = torch.randn((rows, 8, D), device="cuda", dtype=T[kv])
    pos = positions([600 - rows], [rows])
    results = []
    for f in (lambda x: x, shifted):
        k, v = c.k, c.v
        if kv == "int8":
            lq, ls, sm = f(k.layer_q), f(k.layer_scale), f(k.smooth)
            k, v = ti.Int8Pages(lq, ls, sm, 0), ti.Int8Pages(lq, ls, v.smooth, 1)
        else:
            k, v = f(k), f(v)
        kb = ti.key_bounds(D, P, H, c.pages)
        kb.scale = f(kb.scale)
        bt, qq = f(c.tables), f(q)
        ti.update_key_bounds_(BE, kb, k, v, bt, f(positions([0], [600])), max_query_len=600)
        tables, lengths = f(torch.zeros((rows, H, 9), dtype=torch.int32, device="cuda")), f(torch.zeros((rows, H), dtype=torch.int32, device="cuda"))
        ti.select_pages_(BE, tables, lengths, ti.select_pages_workspace(BE, q, kb, bt), qq, kb, bt, f(pos), max_query_len=rows)
        out = f(torch.zeros_like(q))
        ti.sparse_attention_(BE, out, ti.sparse_attention_workspace(BE, q, k, tables, rows), qq, k, v, tables, lengths, 0.09, None, rows)
        results.append((kb.bounds, kb.scale, tables, lengths, out))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    check_attend(c, q, results[0][2], results[0][3], scale=0.09, n=rows)


@pytest.mark.parametrize("kv,D", [("bf16", 128), ("int8", 128), ("fp32", 64), ("int8_fp32", 64), ("bf16", 64)])
@pytest.mark.parametrize("rows", [1, 2])
def test_long_tables(gpu, kv, D, rows):
    """200000 keys a token, the pages of a small pool named again and again."""
    c = Cache(kv, D, 1, 16, [300 * 16], seed=59)
    g = torch.Generator().manual_seed(59)
    torch.manual_seed(59)
    q = torch.randn((rows, 4, D), device="cuda", dtype=T[kv])
    tables = torch.randint(1, c.pages + 1, (rows, 1, 12500), generator=g, dtype=torch.int32).cuda()
    lengths = i32([[200000], [199991]][:rows])
    check_attend(c, q, tables, lengths, n=rows)
