"""Page bounds, page selection and attention over chosen pages against their definitions in 64 bits
(sparse_ref.py): bounds and selections exactly, attention within the rounding its types imply."""
import math

import numpy as np
import pytest
import torch

import sparse_ref as ref
import tileinfer_hip as ti

pytestmark = pytest.mark.gpu
BE = ti.HipBackend()
T = {"bf16": torch.bfloat16, "fp32": torch.float32, "int8": torch.bfloat16, "int8_fp32": torch.float32}


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Cache:
    """A layer's pools of random keys and values with the block tables of sequences, and the keys and
    values that attention sees (the INT8 ones dequantized) in 64 bits on the CPU."""

    def __init__(self, kv, D, H, P, lens, seed, spare=3):
        g = torch.Generator().manual_seed(seed)
        per = [-(-n // P) for n in lens]
        self.P, self.H, self.D, self.pages, self.kv = P, H, D, sum(per) + spare, kv
        ids = (torch.randperm(self.pages, generator=g)[:sum(per)] + 1).tolist()
        width = max(per) + 2
        self.rows = [[ids[sum(per[:b]) + j] for j in range(n)] for b, n in enumerate(per)]
        self.tables = i32([r + [0] * (width - len(r)) for r in self.rows])
        if kv.startswith("int8"):
            q = torch.randint(-127, 128, (2, self.pages, H, P, D), generator=g, dtype=torch.int8)
            s = torch.rand((2, self.pages, H, P), generator=g) * 0.02 + 0.005
            half = torch.rand(D // 2, generator=g) + 0.5
            self.smooth = torch.cat([half, half])
            lq, ls = q.cuda(), s.cuda()
            self.k = ti.Int8Pages(lq, ls, self.smooth.cuda(), 0)
            self.v = ti.Int8Pages(lq, ls, torch.ones(D, device="cuda"), 1)
            self.hk = (q[0].float() * s[0][..., None] * self.smooth).double().numpy()    # rounded as specified
            self.raw = q[0].double().numpy() * s[0][..., None].double().numpy()           # without smoothing
            self.hv = q[1].double().numpy() * s[1][..., None].double().numpy()
            self.scales = s.double().numpy()
        else:
            k = torch.randn((self.pages, H, P, D), generator=g).to(T[kv])
            v = torch.randn((self.pages, H, P, D), generator=g).to(T[kv])
            self.k, self.v = k.cuda(), v.cuda()
            self.hk, self.hv = k.double().numpy(), v.double().numpy()

    def key_at(self, page, head, count):
        return self.hk[page, head, :count]


def positions(starts, counts):
    return i32([s + t for s, n in zip(starts, counts) for t in range(n)])


def offsets(counts):
    return i32(np.concatenate([[0], np.cumsum(counts)]).tolist())


# ---- bounds ----------------------------------------------------------------------------------------

def check_bounds(c, starts, counts, total_rows=None, prior=7):
    kb = ti.key_bounds(c.D, c.P, c.H, c.pages)
    kb.bounds.fill_(prior)
    kb.scale.fill_(prior)
    pos = positions(starts, counts)
    if total_rows:
        pos = torch.cat([pos, torch.zeros(total_rows - len(pos), dtype=torch.int32, device="cuda")])
    ti.update_key_bounds_(BE, kb, c.k, c.v, c.tables, pos, offsets(counts), max(counts))
    bounds = np.full((c.pages, c.H, 2, c.D), prior, np.float64)
    scale = np.full((c.pages, c.H), prior, np.float64)
    table = c.tables.cpu().numpy()
    for b, (s, n) in enumerate(zip(starts, counts)):
        if n:
            ref.update_bounds(bounds, scale, c.key_at, table[b], s, n, c.P, c.H, c.pages)
    assert np.array_equal(kb.bounds.cpu().numpy(), bounds)
    assert np.array_equal(kb.scale.cpu().numpy().astype(np.float64), scale)
    return kb


@pytest.mark.parametrize("kv", ["bf16", "fp32", "int8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("P", [1, 5, 16, 64])
def test_bounds_of_a_ragged_step(gpu, kv, D, P):
    """From position 0, from the middle and the end of a page, one token, an empty sequence, and rows
    behind the last sequence; untouched pages keep what they held."""
    starts, counts = [0, 3, 63, 64, 130, 7], [1, 70, 1, 33, 0, 9]
    c = Cache(kv, D, 3, P, [s + n for s, n in zip(starts, counts)], seed=P + D)
    check_bounds(c, starts, counts, total_rows=sum(counts) + 5)


def test_bounds_do_not_see_past_the_end(gpu):
    """NaN, infinities and huge values behind a sequence's last key; a key that is not finite below it."""
    c = Cache("bf16", 128, 2, 16, [21, 40], seed=1)
    for value in (math.nan, math.inf, 3e38):
        c.k[c.rows[0][1] - 1, :, 5:] = value
        check_bounds(c, [4, 30], [17, 10])
    for value in (math.nan, math.inf, -math.inf):
        c.k[c.rows[1][2] - 1, 1, 3, 100] = value
        c.hk[c.rows[1][2] - 1, 1, 3, 100] = value
        kb = check_bounds(c, [4, 30], [17, 10])
        assert kb.scale[c.rows[1][2] - 1, 1].item() == math.inf


@pytest.mark.parametrize("size", [0.0, 1e-38, 1e-45, 1.0, 127.0, 127.5, 1e30, 3.3e38])
def test_bounds_of_extreme_values(gpu, size):
    """Zeros, subnormal and largest values, and the border between two powers of two."""
    c = Cache("fp32", 64, 2, 4, [9], seed=2)
    c.k.copy_(torch.sign(c.k) * size)
    c.hk = c.k.double().cpu().numpy()
    check_bounds(c, [0], [9])


def test_bounds_skip_pages_that_are_not_there(gpu):
    """Zero and too large ids, and positions past the table's row."""
    c = Cache("bf16", 64, 2, 4, [30], seed=3)
    c.tables[0, 1], c.tables[0, 3] = 0, c.pages + 1
    check_bounds(c, [0], [30])
    c.tables = c.tables[:, :5].contiguous()
    check_bounds(c, [2], [28])


def test_bounds_after_a_rejected_draft(gpu):
    """A step is taken back and another written over it: the bounds are those of what the cache holds."""
    c = Cache("bf16", 128, 2, 16, [60], seed=4)
    kb = check_bounds(c, [0], [60])
    fresh = ti.key_bounds(c.D, c.P, c.H, c.pages)
    ti.update_key_bounds_(BE, fresh, c.k, c.v, c.tables, positions([0], [41]), max_query_len=41)
    ti.update_key_bounds_(BE, kb, c.k, c.v, c.tables, positions([40], [1]), max_query_len=1)
    i = c.rows[0][2] - 1
    assert torch.equal(kb.bounds[i], fresh.bounds[i]) and torch.equal(kb.scale[i], fresh.scale[i])


# ---- selection -------------------------------------------------------------------------------------

def random_bounds(pages, H, D, P, seed):
    g = torch.Generator().manual_seed(seed)
    mid, out = torch.randn((pages, H, 1, D), generator=g) * 20, torch.rand((pages, H, 2, D), generator=g) * 50
    b = torch.clamp(torch.round(mid + torch.tensor([1.0, -1.0])[:, None] * out), -127, 127).to(torch.int8)
    s = 2.0 ** torch.randint(-7, -4, (pages, H), generator=g).float()
    return ti.KeyBounds(b.cuda(), s.cuda(), P)


def check_select(kb, tables, starts, counts, q, keep, sinks, window, causal, spare=0):
    H = kb.shape[1]
    rows = sum(counts) + spare
    out = torch.full((rows, H, keep), -5, dtype=torch.int32, device="cuda")
    lengths = torch.full((rows, H), -5, dtype=torch.int32, device="cuda")
    pos = torch.cat([positions(starts, counts), torch.zeros(spare, dtype=torch.int32, device="cuda")])
    ws = ti.select_pages_workspace(BE, q, kb, tables)
    ti.select_pages_(BE, out, lengths, ws, q, kb, tables, pos, sinks, window, causal, offsets(counts), max(counts))
    got, got_len = out.cpu().numpy(), lengths.cpu().numpy()
    b, s, qd = kb.bounds.cpu().numpy(), kb.scale.cpu().numpy(), q.double().cpu().numpy()
    table, row = tables.cpu().numpy(), 0
    for i, (start, n) in enumerate(zip(starts, counts)):
        for t in range(n):
            last = start + (t if causal else n - 1)
            want, want_len = ref.select(qd[row], b, s, table[i], last, kb.page_size, keep, sinks, window)
            assert np.array_equal(got[row], want), f"sequence {i} token {t}"
            assert np.array_equal(got_len[row], want_len), f"sequence {i} token {t}"
            row += 1
    assert (got[row:] == -5).all() and (got_len[row:] == -5).all(), "rows behind the last sequence"
    return out, lengths


def tables_for(lens, P, pages, seed, extra=1):
    g = torch.Generator().manual_seed(seed)
    per = [-(-n // P) for n in lens]
    width = max(per) + extra
    rows = [(torch.randperm(pages, generator=g)[:n] + 1).tolist() + [0] * (width - n) for n in per]
    return i32(rows)


@pytest.mark.parametrize("G", [1, 2, 3, 4, 6, 8, 16, 20, 64])
@pytest.mark.parametrize("dtype,D", [("bf16", 128), ("fp32", 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_select_ragged_step(gpu, G, dtype, D, causal):
    starts, counts, P, H, pages = [0, 1000, 37, 333, 500], [9, 1, 21, 0, 5], 16, 2, 90
    tables = tables_for([s + n for s, n in zip(starts, counts)], P, pages, G)
    kb = random_bounds(pages, H, D, P, G)
    torch.manual_seed(G)
    q = torch.randn((sum(counts) + 3, H * G, D), device="cuda", dtype=T[dtype])
    check_select(kb, tables, starts, counts, q, 12, 1, 2, causal, spare=3)


@pytest.mark.parametrize("keep,sinks,window", [(1, 0, 1), (2, 1, 1), (7, 0, 7), (40, 3, 5), (63, 1, 1), (64, 1, 1), (200, 2, 3), (300, 100, 200)])
def test_select_budgets(gpu, keep, sinks, window):
    """Nothing, something and everything kept by score; more kept than there is, forced pages that overlap."""
    starts, counts, P, pages = [63 * 8 + 3, 0, 100], [1, 3, 2], 8, 200
    tables = tables_for([s + n for s, n in zip(starts, counts)], P, pages, keep)
    kb = random_bounds(pages, 3, 64, P, keep)
    torch.manual_seed(keep)
    q = torch.randn((6, 12, 64), device="cuda", dtype=torch.bfloat16)
    check_select(kb, tables, starts, counts, q, keep, sinks, window, True)


@pytest.mark.parametrize("P,pages,ctx", [(1, 700, 600), (5, 40, 150), (16, 9000, 131071), (64, 600, 32768)])
def test_select_long_and_odd_pages(gpu, P, pages, ctx):
    tables = tables_for([ctx + 1, 3], P, pages, ctx)
    kb = random_bounds(pages, 2, 128, P, ctx)
    torch.manual_seed(ctx)
    q = torch.randn((2, 8, 128), device="cuda", dtype=torch.bfloat16)
    check_select(kb, tables, [ctx, 2], [1, 1], q, 64, 1, 2, True)


def test_select_ties_go_to_the_first(gpu):
    """Pages of equal bounds, scores of zero and negative ones, queries of zeros."""
    P, pages = 16, 300
    tables = tables_for([4500], P, pages, 5)
    kb = random_bounds(pages, 2, 64, P, 5)
    torch.manual_seed(5)
    q = torch.randn((1, 8, 64), device="cuda", dtype=torch.bfloat16)
    kb.bounds[:, 0] = kb.bounds[0, 0]
    kb.scale[:, 0] = 2.0 ** -5
    kb.bounds[:, 1, 0] = torch.where(torch.rand((pages, 1), device="cuda") < 0.7, kb.bounds[0, 1, 0], kb.bounds[:, 1, 0])
    check_select(kb, tables, [4499], [1], q, 50, 1, 2, True)
    kb.bounds[:, :, 0], kb.bounds[:, :, 1] = -1, -1          # some products negative, many equal
    check_select(kb, tables, [4499], [1], q, 50, 0, 1, True)
    check_select(kb, tables, [4499], [1], torch.zeros_like(q), 50, 0, 1, True)
    kb.bounds.zero_()
    check_select(kb, tables, [4499], [1], -q, 50, 0, 1, True)


def test_select_not_finite(gpu):
    """Query heads with NaN or infinities count for nothing, pages with an infinite scale for the most."""
    P, pages = 16, 100
    tables = tables_for([1500], P, pages, 6)
    kb = random_bounds(pages, 2, 64, P, 6)
    kb.bounds[17, :, 0], kb.bounds[17, :, 1], kb.scale[17] = 127, -127, math.inf
    kb.scale[31, 1] = math.inf
    kb.bounds[31, 1, 0], kb.bounds[31, 1, 1] = 127, -127
    torch.manual_seed(6)
    q = torch.randn((1, 8, 64), device="cuda")
    check_select(kb, tables, [1499], [1], q, 9, 1, 1, True)
    q[0, 1, 5], q[0, 2, 7], q[0, 3, 9] = math.nan, math.inf, -math.inf
    check_select(kb, tables, [1499], [1], q, 9, 1, 1, True)
    q[0, 0, 63] = math.nan
    check_select(kb, tables, [1499], [1], q, 9, 1, 1, True)


@pytest.mark.parametrize("size", [1e-40, 1e-30, 1e25])
def test_select_sizes_of_queries(gpu, size):
    tables = tables_for([1500], 16, 100, 7)
    kb = random_bounds(100, 2, 64, 16, 7)
    torch.manual_seed(7)
    q = torch.randn((1, 4, 64), device="cuda") * size
    check_select(kb, tables, [1499], [1], q, 9, 1, 1, True)


def test_select_bounds_are_bounds(gpu):
    """No key's product with the whole-number query exceeds its page's score: the kept pages hold every
    page whose best product exceeds the best score of those left out."""
    c = Cache("bf16", 128, 2, 16, [2000], seed=8)
    kb = check_bounds(c, [0], [2000])
    torch.manual_seed(8)
    q = torch.randn((1, 2, 128), device="cuda", dtype=torch.bfloat16)
    out, _ = check_select(kb, c.tables, [1999], [1], q, 20, 0, 1, True)
    for h in range(2):
        row = q[0, h].double().cpu().numpy()
        s = ref.least_power(np.abs(row).max())
        best = [(np.rint(row / s) * s) @ c.hk[i - 1, h].T for i in c.rows[0]]
        b, sc = kb.bounds[:, h].double().cpu().numpy(), kb.scale[:, h].double().cpu().numpy()
        w = np.rint(row / s)
        for j, i in enumerate(c.rows[0]):
            assert best[j].max() <= np.maximum(w * b[i - 1, 0], w * b[i - 1, 1]).sum() * s * sc[i - 1] + 1e-9


# ---- attention over chosen pages -------------------------------------------------------------------

def check_attend(c, q, tables, lengths, scale=None, qsl=None, n=None, out=None):
    rows, Hq, D = q.shape
    G = Hq // c.H
    scale = 1 / math.sqrt(D) if scale is None else scale
    prior = torch.full_like(q, 7)
    ws = ti.sparse_attention_workspace(BE, q, c.k, tables, 1 if n is None else n)
    got = ti.sparse_attention_(BE, prior, ws, q, c.k, c.v, tables, lengths, scale, qsl, n)
    torch.cuda.synchronize()
    got, qd, table, lens = got.double().cpu().numpy(), q.double().cpu().numpy(), tables.cpu().numpy(), lengths.cpu().numpy()
    lo, hi = (0, rows) if qsl is None else (int(qsl[0]), int(qsl[-1]))
    half = torch.finfo(q.dtype).eps / 2
    if c.kv == "int8":
        # the kernel's queries: smoothed, then rounded to fp16's 11 bits (a row's largest scaled into [2^14, 2^15),
        # where every float of 2^-28 of it is normal); weights times value scales in fp16
        x = (q.float().cpu() * c.smooth).double()
        e = 15 - torch.frexp(x.abs().amax(2, keepdim=True)).exponent
        qd = torch.ldexp(torch.ldexp(x, e).to(torch.float16).double(), -e).numpy()
    keys_of = c.raw if c.kv == "int8" else c.hk
    p_eps = {"bf16": 2.0 ** -8, "int8": 2.0 ** -11 + 2.0 ** -23, "fp32": 0.0, "int8_fp32": 2.0 ** -22}[c.kv]
    for r in range(rows):
        for h in range(c.H):
            rows_ = qd[r, h * G:(h + 1) * G]
            mine = got[r, h * G:(h + 1) * G]
            if not lo <= r < hi:
                assert (mine == 7).all(), "rows of no sequence"
                continue
            m = min(max(int(lens[r, h]), 0), tables.shape[2] * c.P)
            at = np.arange(m)
            page = np.clip(table[r, h][at // c.P] - 1, 0, c.pages - 1)
            k, v = keys_of[page, h, at % c.P], c.hv[page, h, at % c.P]
            want, weight, size = ref.attend(rows_, k, v, scale)
            bias = 0.0
            if c.kv == "int8" and m:
                # The kernel multiplies biased values: sums of q (1152 + b) and p s (1152 + b), from which 1152 sum(q)
                # and 1152 sum(p s) come off. |b| <= 127, so every partial sum is at most 1279 (1152) times sum |q|
                # (sum p s), and each of its additions, the other sum's and the subtraction round by 2^-24 of that:
                # 2431 sum |q| s scale takes the place of the scores' size, and 2431 (keys + 2) 2^-24 sum(p s) is
                # added to the output. A weight p s (p <= 1 of the largest, whose own is at least 1 of the sum) below
                # fp16's normal range 2^-14 rounds to a multiple of 2^-24: off by 2^-25 of |b| per key.
                ks, vs = c.scales[0][page, h, at % c.P], c.scales[1][page, h, at % c.P]
                size = 2431 * np.abs(rows_).sum(1).max() * ks.max() * scale
                bias = 2431 * (m + 2) * 2.0 ** -24 * ref.attend(rows_, k, vs[:, None], scale)[0] \
                    + 2.0 ** -25 * np.abs(v / vs[:, None]).sum(0)
            tol = bias + ref.attention_tolerance(want, weight, size, D + (3 if c.kv == "int8_fp32" else 0), m, p_eps, half)
            worst = np.max(np.abs(mine - want) / tol)
            assert worst <= 1, f"row {r} head {h}: {worst:.2f} times the tolerance"
    return got


def chosen(c, rows, width, seed, lens=None):
    """Tables of random distinct pages and lengths that end inside the last one."""
    g = torch.Generator().manual_seed(seed)
    t = torch.stack([torch.stack([torch.randperm(c.pages, generator=g)[:width] + 1 for _ in range(c.H)]) for _ in range(rows)])
    n = torch.randint(1, width * c.P + 1, (rows, c.H), generator=g) if lens is None else torch.tensor(lens).expand(rows, c.H)
    return t.to(torch.int32).cuda().contiguous(), n.to(torch.int32).cuda().contiguous()


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp32", "int8_fp32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("P", [1, 5, 16, 64])
@pytest.mark.parametrize("rows", [1, 5])
def test_attend_pages(gpu, kv, D, P, rows):
    c = Cache(kv, D, 2, P, [40 * P], seed=P + D)
    torch.manual_seed(P)
    q = torch.randn((rows, 8, D), device="cuda", dtype=T[kv])
    tables, lengths = chosen(c, rows, 19, seed=P)
    check_attend(c, q, tables, lengths)
    if rows > 1:
        check_attend(c, q, tables, lengths, n=rows)


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp32"])
@pytest.mark.parametrize("G", [1, 2, 3, 5, 8, 12, 16, 24, 40, 64])
def test_attend_head_groups(gpu, kv, G):
    c = Cache(kv, 128, 2, 16, [500], seed=G)
    torch.manual_seed(G)
    q = torch.randn((7, 2 * G, 128), device="cuda", dtype=T[kv])
    tables, lengths = chosen(c, 7, 11, seed=G)
    check_attend(c, q, tables, lengths)
    check_attend(c, q, tables, lengths, n=7)


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp32"])
@pytest.mark.parametrize("rows", [1, 40])
def test_attend_lengths(gpu, kv, rows):
    """No keys, one, the ends of tiles and pages, a full table, lengths past it and negative ones."""
    c = Cache(kv, 128, 8, 16, [900], seed=11)
    torch.manual_seed(11)
    q = torch.randn((rows, 32, 128), device="cuda", dtype=T[kv])
    tables, lengths = chosen(c, rows, 24, seed=11)
    lengths[0] = i32([0, 1, 15, 16, 17, 384, 1000, -3])
    lengths[-1, :3] = i32([2 ** 31 - 1, -2 ** 31, 0])
    check_attend(c, q, tables, lengths)
    lengths.zero_()
    assert (check_attend(c, q, tables, lengths) == 0).all()


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp32"])
@pytest.mark.parametrize("n", [None, 13])
def test_attend_same_page_twice_and_ids_outside_the_pool(gpu, kv, n):
    c = Cache(kv, 64, 2, 16, [300], seed=12)
    torch.manual_seed(12)
    q = torch.randn((13, 8, 64), device="cuda", dtype=T[kv])
    tables, lengths = chosen(c, 13, 9, seed=12)
    tables[:, :, 4] = tables[:, :, 2]
    tables[3, 1] = tables[3, 1, 0]
    check_attend(c, q, tables, lengths, n=n)
    tables[5, 0, 1], tables[5, 0, 2], tables[6, 1, 0], tables[6, 1, 1] = 0, -7, c.pages + 1, 2 ** 31 - 1
    check_attend(c, q, tables, lengths, n=n)


@pytest.mark.parametrize("n", [1, 4, 9])
def test_attend_rows_of_no_sequence(gpu, n):
    c = Cache("bf16", 128, 2, 16, [300], seed=13)
    torch.manual_seed(13)
    q = torch.randn((17, 8, 128), device="cuda", dtype=torch.bfloat16)
    tables, lengths = chosen(c, 17, 9, seed=13)
    check_attend(c, q, tables, lengths, qsl=i32([2, 2, 6, 11]), n=n)


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp32"])
def test_attend_does_not_see_past_the_last_key(gpu, kv):
    """NaN and infinities in the last page's rows behind the length, and in pages no table names."""
    c = Cache(kv, 128, 2, 16, [400], seed=14)
    torch.manual_seed(14)
    q = torch.randn((6, 8, 128), device="cuda", dtype=T[kv])
    tables, lengths = chosen(c, 6, 5, seed=14, lens=4 * 16 + 7)
    used = torch.zeros(c.pages + 1, dtype=torch.bool)
    used[tables[:, :, :4].cpu().long().reshape(-1)] = True
    for r in range(6):        # a last page of each row's own, garbage behind its 7 keys
        tables[r, :, 4] = c.rows[0][r]
        tables[r, :, :4] = i32(c.rows[0][6 + 3 * r:10 + 3 * r])
    for r in range(6):
        i = c.rows[0][r] - 1
        if kv == "int8":
            c.k.scale[i, :, 7:], c.v.scale[i, :, 7:] = math.nan, math.inf
        else:
            c.k[i, :, 7:], c.v[i, :, 7:] = math.nan, math.inf
    check_attend(c, q, tables, lengths)
    check_attend(c, q, tables, lengths, n=6)


def shared(c, rows, width, seed, common=0.8):
    """Tables as the tokens of a step select them: most pages are the same from token to token, and every
    token's last page is partly filled, to another position."""
    g = torch.Generator().manual_seed(seed)
    liked = torch.rand((c.H, c.pages), generator=g)
    t = torch.zeros((rows, c.H, width), dtype=torch.int32)
    for r in range(rows):
        rank = common * liked + (1 - common) * torch.rand((c.H, c.pages), generator=g)
        t[r] = torch.sort(torch.topk(rank, width, dim=1).indices, dim=1).values + 1
    n = torch.randint(1, width * c.P + 1, (rows, c.H), generator=g)
    n[: rows // 2] = (width - 1) * c.P + torch.randint(1, c.P + 1, (rows // 2, c.H), generator=g)
    return t.cuda().contiguous(), n.to(torch.int32).cuda().contiguous()


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp32"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("G,P", [(4, 16), (4, 64), (1, 16), (2, 32), (3, 16), (7, 64), (8, 16), (12, 16), (16, 32)])
@pytest.mark.parametrize("rows", [2, 16, 33])
def test_attend_steps_that_share_pages(gpu, kv, D, G, P, rows):
    c = Cache(kv, D, 2, P, [40 * P], seed=G + P)
    torch.manual_seed(G)
    q = torch.randn((rows, 2 * G, D), device="cuda", dtype=T[kv])
    tables, lengths = shared(c, rows, 13, seed=G)
    check_attend(c, q, tables, lengths, n=rows)
    lengths[0], lengths[rows // 2, 0], lengths[-1] = 0, 1, 13 * P
    check_attend(c, q, tables, lengths, n=rows)


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp32"])
@pytest.mark.parametrize("width", [1, 5, 70, 200, 600, 1100])
def test_attend_steps_of_any_width(gpu, kv, width):
    """As many tokens as their tables leave room for: 32 rows, 16, fewer tokens than fill them, one."""
    c = Cache(kv, 64, 8, 16, [16 * (width + 40)], seed=width)
    torch.manual_seed(width)
    rows = 520 if width <= 5 else 12
    q = torch.randn((rows, 32, 64), device="cuda", dtype=T[kv])
    tables, lengths = shared(c, rows, width, seed=width)
    check_attend(c, q, tables, lengths, n=rows)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["k", "v"])
@pytest.mark.parametrize("rows,heads,kv", [(6, 2, "bf16"), (300, 8, "bf16"), (6, 2, "fp32"), (300, 8, "fp32")])
def test_attend_values_that_are_not_finite_stay_with_their_tokens(gpu, value, where, rows, heads, kv):
    """A key or value that is not finite in a page that some tokens of a step keep, or behind the last key
    of others: tokens that do not see it are as without it, those that do are as their own attention."""
    c = Cache(kv, 128, heads, 16, [60 * 16], seed=31)
    torch.manual_seed(31)
    q = torch.randn((rows, heads * 4, 128), device="cuda", dtype=T[kv])
    tables, lengths = shared(c, rows, 9, seed=31)
    lengths[:] = 8 * 16 + 9
    bad = tables[1, 0, 2].item()
    last = tables[3, 1, 8].item()
    pool = c.k if where == "k" else c.v
    pool[bad - 1, :, 5, 17] = value
    pool[last - 1, :, 9, 3] = value                # seen where this page is not the last one
    alone = torch.empty_like(q)
    ti.sparse_attention_(BE, alone, ti.sparse_attention_workspace(BE, q, c.k, tables), q, c.k, c.v, tables, lengths, 0.09)
    got = ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.09, None, rows)
    touched = (((tables == bad) | (tables == last)) & ~((tables == last) & (torch.arange(9, device="cuda") == 8)
                                                     & (tables != bad))).any(2)
    touched = touched.repeat_interleave(4, 1)
    assert touched.any() and not touched.all()
    clean = pool.clone()
    clean[bad - 1, :, 5, 17], clean[last - 1, :, 9, 3] = 0, 0
    k, clean_v = (clean, c.v) if where == "k" else (c.k, clean)
    want = ti.sparse_attention(BE, q, k, clean_v, tables, lengths, 0.09, None, rows)
    # rows of the wave-by-row path round otherwise: each is within 2^-7 of the exact weights and output
    assert torch.isfinite(got[~touched]).all()
    tol = 4 * 2.0 ** -8 * c.v[torch.isfinite(c.v)].float().abs().max()
    assert (got[~touched].float() - want[~touched].float()).abs().max() <= tol
    a, b = alone[touched].float(), got[touched].float()
    assert torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(torch.isinf(a), torch.isinf(b))
    fine = torch.isfinite(a)
    assert ((a[fine] - b[fine]).abs() <= tol).all()


def test_attend_sequences_do_not_touch_each_other(gpu):
    """Steps of several sequences whose rows fall into one group: NaN in one sequence's cache."""
    c = Cache("bf16", 128, 2, 16, [160, 160, 160], seed=32)
    torch.manual_seed(32)
    q = torch.randn((9, 8, 128), device="cuda", dtype=torch.bfloat16)
    kb = ti.key_bounds(128, 16, 2, c.pages)
    pos = positions([157, 157, 157], [3, 3, 3])
    for i in c.rows[1]:
        c.k[i - 1], c.v[i - 1] = math.nan, math.nan
    ti.update_key_bounds_(BE, kb, c.k, c.v, c.tables, positions([0, 0, 0], [160] * 3), max_query_len=160)
    tables, lengths = ti.select_pages(BE, q, kb, c.tables, pos, 6, max_query_len=3)
    got = ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.09, None, 3)
    assert torch.isnan(got[3:6]).all() and torch.isfinite(got[:3]).all() and torch.isfinite(got[6:]).all()


def test_attend_large_and_small_scores(gpu):
    """Scores far apart (weights that underflow) and a scale that makes them all alike."""
    c = Cache("bf16", 128, 2, 64, [2000], seed=15)
    torch.manual_seed(15)
    q = torch.randn((3, 8, 128), device="cuda", dtype=torch.bfloat16)
    tables, lengths = chosen(c, 3, 30, seed=15)
    check_attend(c, q, tables, lengths, scale=1e-6)
    check_attend(c, q * 0, tables, lengths)
    check_attend(c, q, tables, lengths, scale=0.6)


def test_attend_all_pages_is_paged_attention(gpu):
    """Tables that name every page of a sequence: the dense operator's result for the same keys."""
    c = Cache("bf16", 128, 8, 16, [1000, 77], seed=16)
    torch.manual_seed(16)
    q = torch.randn((2, 32, 128), device="cuda", dtype=torch.bfloat16)
    pos = i32([999, 76])
    dense = torch.empty_like(q)
    ws = ti.attention_workspace(BE, q, c.k, num_seqs=2)
    ti.paged_attention_(BE, dense, ws, q, c.k, c.v, c.tables, pos, 0.09)
    kb = ti.key_bounds(128, 16, 8, c.pages)
    tables, lengths = ti.select_pages(BE, q, kb, c.tables, pos, keep=63)
    assert (lengths[0] == 1000).all() and (lengths[1] == 77).all()
    got = ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.09)
    check_attend(c, q, tables, lengths, scale=0.09)
    # each is within its rounding of the exact result: weights 2^-8, output 2^-8
    assert (got.float() - dense.float()).abs().max() <= 4 * 2.0 ** -8 * c.v.float().abs().max()


def test_attend_is_repeatable(gpu):
    """The same call gives the same bits (no sum depends on the order of work-groups)."""
    c = Cache("bf16", 128, 8, 16, [4000], seed=17)
    torch.manual_seed(17)
    q = torch.randn((16, 32, 128), device="cuda", dtype=torch.bfloat16)
    pos = positions([3984], [16])
    kb = check_bounds(c, [0], [4000])
    tables, lengths = ti.select_pages(BE, q, kb, c.tables, pos, keep=32, max_query_len=16)
    first = ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.09, None, 16)
    for _ in range(5):
        assert torch.equal(ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.09, None, 16), first)


# ---- refusals that need tensors on the GPU ---------------------------------------------------------

def test_refusals(gpu):
    c = Cache("bf16", 128, 8, 16, [100], seed=18)
    kb = ti.key_bounds(128, 16, 8, c.pages)
    q = torch.zeros((2, 32, 128), device="cuda", dtype=torch.bfloat16)
    pos, tables, lengths = i32([98, 99]), torch.zeros((2, 8, 4), dtype=torch.int32, device="cuda"), torch.zeros((2, 8), dtype=torch.int32, device="cuda")
    ws = ti.select_pages_workspace(BE, q, kb, c.tables)

    def refused(f, *a, **kw):
        with pytest.raises(ti.ArgumentError):
            f(BE, *a, **kw)

    refused(ti.update_key_bounds_, ti.key_bounds(128, 32, 8, c.pages), c.k, c.v, c.tables, pos)
    refused(ti.update_key_bounds_, kb, c.k, c.v, c.tables.long(), pos)
    refused(ti.update_key_bounds_, kb, c.k, c.v, c.tables, pos, offsets([2]))              # no max_query_len
    refused(ti.update_key_bounds_, kb, c.k, c.v, c.tables, pos, offsets([1, 1]), 1)         # two sequences, one table
    refused(ti.update_key_bounds_, kb, c.k.half(), c.v.half(), c.tables, pos)
    refused(ti.select_pages_, tables, lengths, None, q, kb, c.tables, pos)
    refused(ti.select_pages_, tables, lengths, ws[:64], q, kb, c.tables, pos)
    refused(ti.select_pages_, tables, lengths, ws, q[:, :30].contiguous(), kb, c.tables, pos)
    refused(ti.select_pages_, tables, lengths, ws, q.half(), kb, c.tables, pos)
    refused(ti.select_pages_, tables, lengths, ws, q.transpose(0, 1), kb, c.tables, pos)
    refused(ti.select_pages_, tables, lengths[:1], ws, q, kb, c.tables, pos)
    refused(ti.select_pages_, tables, lengths, ws, q, kb, c.tables, pos[:1])
    refused(ti.select_pages_, tables, lengths, ws, q, kb, c.tables, pos, sinks=3, window=2)
    refused(ti.select_pages_, tables, lengths, ws, q, kb, c.tables, pos, sinks=1, window=0)
    refused(ti.select_pages_, tables.long(), lengths, ws, q, kb, c.tables, pos)
    out = torch.empty_like(q)
    sws = ti.sparse_attention_workspace(BE, q, c.k, tables)
    refused(ti.sparse_attention_, out, sws, q, c.k.float(), c.v.float(), tables, lengths, 0.1)
    refused(ti.sparse_attention_, out, sws, q, c.k, c.v, tables[:1], lengths, 0.1)
    refused(ti.sparse_attention_, out, sws, q, c.k, c.v, tables, lengths, 0.0)
    refused(ti.sparse_attention_, out, sws, q, c.k, c.v, tables, lengths, math.nan)
    refused(ti.sparse_attention_, out, sws, q[:, :, :64].contiguous(), c.k, c.v, tables, lengths, 0.1)
    refused(ti.sparse_attention_, out, sws, q, c.k, c.v, tables, lengths, 0.1, offsets([1, 1]))
    refused(ti.sparse_attention_, out, sws, q, c.k, c.v, tables, lengths, 0.1, None, 3)
    refused(ti.sparse_attention_, out, sws, q, c.k, c.v, tables.cpu(), lengths, 0.1)
    refused(ti.sparse_attention_, out.cpu(), sws, q, c.k, c.v, tables, lengths, 0.1)


# ---- largest sizes and launch limits ---------------------------------------------------------------

@pytest.mark.parametrize("B,width", [(64, 34000), (64, 16300), (130, 16300), (1, 34000), (1, 40000), (2, 2100), (4, 760), (64, 2040), (130, 4000)])
def test_select_wide_tables(gpu, B, width):
    """Tables as wide as LDS holds in one launch and in two, wider than it holds, and with several tokens of one
    sequence; one sequence is long, the others short."""
    P, pages, H, n = 1, 3000, 2, 2
    g = torch.Generator().manual_seed(width + B)
    tables = torch.randint(1, pages + 1, (B, width), generator=g, dtype=torch.int32).cuda()
    kb = random_bounds(pages, H, 64, P, width)
    torch.manual_seed(B)
    starts = [width - n] + [5 + b for b in range(1, B)]
    q = torch.randn((B * n, H * 4, 64), device="cuda", dtype=torch.bfloat16)
    check_select(kb, tables, starts, [n] * B, q, 70, 2, 3, True)


@pytest.mark.parametrize("B,H,pages", [(64, 8, 256), (1, 2, 900), (2, 2, 9000)])
def test_select_infinite_scores(gpu, B, H, pages):
    """Many pages of infinite scores of either sign beside finite ones, more of the largest than are kept."""
    kb = random_bounds(pages, H, 64, 16, B)
    kb.bounds[:], sign = kb.bounds.abs(), torch.arange(pages, device="cuda") % 5
    kb.scale[sign > 0] = math.inf
    kb.bounds[sign == 1] *= -1
    tables = tables_for([16 * (pages - 20 - b) for b in range(B)], 16, pages, B)
    torch.manual_seed(B)
    q = torch.rand((B, H * 4, 64), device="cuda", dtype=torch.bfloat16) + 0.25
    check_select(kb, tables, [16 * (pages - 20 - b) - 1 for b in range(B)], [1] * B, q, 40, 1, 1, True)
    kb.scale[sign > 1] = 2.0 ** -120
    kb.scale[sign == 2] = 2.0 ** 100
    check_select(kb, tables, [16 * (pages - 20 - b) - 1 for b in range(B)], [1] * B, q, pages // 2, 1, 1, True)


def test_select_captured_with_much_lds(gpu):
    """A launch that needs more LDS than a kernel gets by default, recorded in a graph and replayed."""
    P, pages, B = 16, 9000, 64
    tables = tables_for([140000] + [300] * (B - 1), P, pages, 3)
    kb = random_bounds(pages, 2, 128, P, 3)
    torch.manual_seed(3)
    q = torch.randn((B, 8, 128), device="cuda", dtype=torch.bfloat16)
    pos = i32([139999] + [250] * (B - 1))
    out, lengths = torch.zeros((B, 2, 32), dtype=torch.int32, device="cuda"), torch.zeros((B, 2), dtype=torch.int32, device="cuda")
    ws = ti.select_pages_workspace(BE, q, kb, tables)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ti.select_pages_(BE, out, lengths, ws, q, kb, tables, pos)
    for i in range(3):
        q.normal_()
        pos[1:] += 7
        g.replay()
        torch.cuda.synchronize()
        got = out.clone(), lengths.clone()
        want = ti.select_pages(BE, q, kb, tables, pos, 32)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp32"])
@pytest.mark.parametrize("rows,heads,width", [(16, 2, 64), (256, 16, 16), (32, 2, 32)])
def test_attend_groups_of_many_tokens(gpu, kv, rows, heads, width):
    """One query head per KV head: 16 and 32 tokens in a group, whose lists take the most LDS."""
    c = Cache(kv, 128, heads, 16, [16 * (width + 30)], seed=width)
    torch.manual_seed(width)
    q = torch.randn((rows, heads, 128), device="cuda", dtype=T[kv])
    tables, lengths = shared(c, rows, width, seed=width)
    check_attend(c, q, tables, lengths, n=rows)


@pytest.mark.parametrize("kv", ["bf16", "int8"])
@pytest.mark.parametrize("D,P,heads,G,rows,width", [(128, 16, 32, 4, 131, 5), (128, 64, 32, 4, 128, 3), (128, 16, 64, 2, 260, 4),
                                                    (128, 32, 64, 3, 84, 6), (128, 16, 128, 12, 11, 9), (64, 16, 64, 4, 131, 5),
                                                    (64, 16, 64, 16, 67, 3), (128, 16, 128, 8, 35, 130)])
def test_attend_many_rows_in_a_group(gpu, kv, D, P, heads, G, rows, width):
    """Steps with so many tokens and KV heads that a group has up to 64 query rows; the last group is not full."""
    c = Cache(kv, D, heads, P, [P * (width + 20)], seed=rows)
    torch.manual_seed(rows)
    q = torch.randn((rows, heads * G, D), device="cuda", dtype=T[kv])
    tables, lengths = shared(c, rows, width, seed=rows)
    lengths[3], lengths[5, 1] = 0, 1
    check_attend(c, q, tables, lengths, n=rows)
    check_attend(c, q, tables, lengths, scale=0.05, qsl=i32([2, rows // 2, rows - 1]), n=rows)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["k", "v"])
def test_attend_many_rows_with_values_that_are_not_finite(gpu, value, where):
    rows, heads = 64, 64
    c = Cache("bf16", 128, heads, 16, [40 * 16], seed=32)
    torch.manual_seed(32)
    q = torch.randn((rows, heads * 4, 128), device="cuda", dtype=torch.bfloat16)
    tables, lengths = shared(c, rows, 4, seed=32)
    bad = tables[1, 0, 2].item()
    pool = c.k if where == "k" else c.v
    want = ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.09, None, rows)
    pool[bad - 1, :, 5, 17] = value
    got = ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.09, None, rows)
    used = torch.arange(4, device="cuda") * 16 < lengths[..., None]
    touched = ((tables == bad) & used).any(2).repeat_interleave(4, 1)
    assert touched.any() and not touched.all()
    assert torch.isfinite(got[~touched]).all()
    # rows of the wave-by-row path round otherwise: each is within 2^-7 of the exact weights and output
    size = c.v[torch.isfinite(c.v)].abs().max().item()
    assert (got[~touched].float() - want[~touched].float()).abs().max().item() <= 2 * 2.0 ** -7 * size
    alone = ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.09)
    assert torch.equal(torch.isfinite(got), torch.isfinite(alone))


def test_attend_captured_with_much_lds(gpu):
    """Groups of 32 tokens whose joined tables need 64 KB of LDS beside the tiles', recorded in a graph and replayed."""
    rows, heads, width = 36, 256, 32
    c = Cache("bf16", 64, heads, 16, [(width + 20) * 16], seed=33)
    torch.manual_seed(33)
    q = torch.randn((rows, heads * 2, 64), device="cuda", dtype=torch.bfloat16)
    tables, lengths = shared(c, rows, width, seed=33)
    out, ws = torch.zeros_like(q), ti.sparse_attention_workspace(BE, q, c.k, tables, rows)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ti.sparse_attention_(BE, out, ws, q, c.k, c.v, tables, lengths, 0.125, None, rows)
    size = c.v.abs().max().item()
    for i in range(3):
        q.normal_()
        lengths.sub_(3)
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(got, ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.125, None, rows))
        # token by token: weights rounded to bf16 (2^-8 each, their sum too) and the output (2^-8), on either side
        alone = ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.125)
        assert (got.float() - alone.float()).abs().max().item() <= 2 * 3 * 2.0 ** -8 * size


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, 1e38])
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("rows,heads", [(6, 2), (300, 8)])
def test_attend_int8_scales_that_are_not_finite_stay_with_their_tokens(gpu, value, half, rows, heads):
    """INT8: a key's or value's scale that is not finite, or so large that scores overflow, in a page that some
    tokens of a step keep and behind the last key of others: the same operations on the same numbers for the rest."""
    c = Cache("int8", 128, heads, 16, [60 * 16], seed=34)
    torch.manual_seed(34)
    q = torch.randn((rows, heads * 4, 128), device="cuda", dtype=torch.bfloat16)
    tables, lengths = shared(c, rows, 9, seed=34)
    lengths[:] = 8 * 16 + 9
    bad, last = tables[1, 0, 2].item(), tables[3, 1, 8].item()
    want = ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.09, None, rows)
    scales = c.k.layer_scale
    scales[half, bad - 1, :, 5] = value
    scales[half, last - 1, :, 12] = value              # seen where this page is not the last one
    got = ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.09, None, rows)
    end = torch.arange(9, device="cuda") == 8
    touched = ((tables == bad) | ((tables == last) & ~end)).any(2).repeat_interleave(4, 1)
    assert touched.any() and not touched.all()
    assert torch.equal(got[~touched], want[~touched])
    alone = ti.sparse_attention(BE, q, c.k, c.v, tables, lengths, 0.09)
    assert torch.equal(torch.isfinite(got[~touched]), torch.isfinite(alone[~touched]))


@pytest.mark.parametrize("n", [1, 4])
def test_offsets_past_32_bits(gpu, n):
    """Pools of more than 2^31 elements: pages at their end, through bounds, selection and attention."""
    P, H, D = 16, 8, 128
    pages = 2 ** 31 // (P * H * D) + 64
    c = Cache("bf16", D, H, P, [300], seed=40)
    k = torch.zeros((pages, H, P, D), dtype=torch.bfloat16, device="cuda")
    v = torch.zeros_like(k)
    k[-c.pages:], v[-c.pages:] = c.k, c.v
    tables = torch.where(c.tables > 0, c.tables + (pages - c.pages), 0).to(torch.int32)
    pos = positions([300 - n], [n])
    torch.manual_seed(40)
    q = torch.randn((n, 32, D), device="cuda", dtype=torch.bfloat16)
    results = []
    for kp, vp, t in ((k, v, tables), (c.k, c.v, c.tables)):
        kb = ti.key_bounds(D, P, H, kp.shape[0])
        ti.update_key_bounds_(BE, kb, kp, vp, t, positions([0], [300]), max_query_len=300)
        chosen, lengths = ti.select_pages(BE, q, kb, t, pos, 9, max_query_len=n)
        out = ti.sparse_attention(BE, q, kp, vp, chosen, lengths, 0.09, None, n)
        results.append((kb.bounds[-c.pages:], kb.scale[-c.pages:], chosen, lengths, out))
    a, b = results
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[3], b[3])
    assert torch.equal(torch.where(b[2] > 0, b[2] + (pages - c.pages), 0), a[2])
    if n == 1:
        assert torch.equal(a[4], b[4])
    else:       # the joined list's order is that of the tables, whatever the ids
        assert torch.equal(a[4], b[4])


def test_long_step(gpu):
    """More query tokens than a launch's grid holds tiles for one by one."""
    n, P = 70000, 64
    tables = tables_for([n], P, 1200, 41)
    kb = random_bounds(1200, 1, 64, P, 41)
    torch.manual_seed(41)
    q = torch.randn((n, 16, 64), device="cuda", dtype=torch.bfloat16)
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    out, lengths = ti.select_pages(BE, q, kb, tables, pos, 6, max_query_len=n)
    b, s, table = kb.bounds.cpu().numpy(), kb.scale.cpu().numpy(), tables[0].cpu().numpy()
    for t in (0, 63, 64, 32767, 32768, 32769, 65535, 65536, n - 1):
        want, want_len = ref.select(q[t].double().cpu().numpy(), b, s, table, t, P, 6, 1, 1)
        assert np.array_equal(out[t].cpu().numpy(), want) and np.array_equal(lengths[t].cpu().numpy(), want_len), t
    assert (lengths > 0).all()
