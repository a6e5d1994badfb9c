"""The 8-bit block cache: store_kv_ and attention_inputs_ byte for byte against the definition (scales, rounding, blocks that
grow, rows anywhere in the call), and attention over it, causal and not, against 64 bits."""
import math

import numpy as np
import pytest
import torch

import tileinfer_hip as ti
from window_ref import Step, check, decode, i32, store

pytestmark = pytest.mark.gpu
BE = ti.HipBackend()


def pools(D, P, H, pages, g=None):
    """Fresh pools, or ones that hold random rows in blocks of random scales."""
    k, v = ti.fp8_kv_pools(D, P, H, pages)
    if g is not None:
        codes = g.integers(0, 256, k.layer_q.shape).astype(np.uint8)
        codes[(codes & 127) == 127] = 0
        k.layer_q.copy_(torch.from_numpy(codes))
        k.layer_scale.copy_(torch.from_numpy(2.0 ** g.integers(-12, 4, k.layer_scale.shape).astype(np.float32)))
    return k, v


def rows(g, n, H, D, T):
    size = np.exp(2.0 * g.standard_normal((n, H, 1)))
    return torch.from_numpy((g.standard_normal((n, H, D)) * size).astype(np.float32)).to(T)


def same(k, q, scale):
    """Bytes and scales; a NaN is any of its two codes."""
    got, gs = k.layer_q.view(torch.uint8).cpu().numpy(), k.layer_scale.cpu().numpy()
    assert np.array_equal(gs, scale, equal_nan=True)
    nan = (q & 127) == 127
    assert np.array_equal((got & 127) == 127, nan)
    assert np.array_equal(got[~nan], q[~nan])


SLOTS = {
    "one": lambda g, P: [5 * P + 1],
    "inside": lambda g, P: [2 * P + 7],
    "page": lambda g, P: list(range(P + 1, 2 * P + 1)),
    "prompt": lambda g, P: list(range(3 * P + 1, 5 * P + 4)),
    "middle": lambda g, P: list(range(2 * P + 9, 4 * P + 3)),
    "batch": lambda g, P: [i * P + 1 + int(g.integers(0, P)) for i in range(9)],
    "two to a page": lambda g, P: [P + 3, 4 * P + 2, P + 4, 4 * P + 9, P + 12],
    "any order": lambda g, P: list(g.permutation(10 * P)[:5 * P] + 1),
    "outside": lambda g, P: [0, -3, 10 * P + 1, 2 ** 31 - 1, -2 ** 31, 4 * P + 5, 10 * P],
    "twice": lambda g, P: [P + 4, 3 * P, P + 4, P + 4, 3 * P],
    "many": lambda g, P: list(g.permutation(10 * P)[:9 * P] + 1) * 3,
}


@pytest.mark.parametrize("T", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,H,P", [(128, 2, 16), (64, 3, 64), (128, 8, 32), (64, 17, 16)])
@pytest.mark.parametrize("slots", SLOTS)
def test_store(gpu, T, D, H, P, slots):
    g = np.random.Generator(np.random.PCG64(len(slots) + D + P))
    k, v = pools(D, P, H, 10, g)
    q, scale = k.layer_q.cpu().numpy(), k.layer_scale.cpu().numpy()
    at = SLOTS[slots](g, P)
    for _ in range(2):
        x, y = rows(g, len(at), H, D, T), rows(g, len(at), H, D, T)
        ti.store_kv_(BE, k, v, x.cuda(), y.cuda(), i32(at))
        store(q, scale, x.float().numpy(), y.float().numpy(), at)
        same(k, q, scale)


@pytest.mark.parametrize("P", [128, 256, 1024])
def test_large_pages(gpu, P):
    g = np.random.Generator(np.random.PCG64(P))
    D, H = 64, 2
    k, v = pools(D, P, H, 3, g)
    q, scale = k.layer_q.cpu().numpy(), k.layer_scale.cpu().numpy()
    for at in (list(range(1, 2 * P + 40)), [2 * P + 41], list(range(2 * P + 42, 3 * P + 1))):
        x, y = rows(g, len(at), H, D, torch.bfloat16), rows(g, len(at), H, D, torch.bfloat16)
        ti.store_kv_(BE, k, v, x.cuda(), y.cuda(), i32(at))
        store(q, scale, x.float().numpy(), y.float().numpy(), at)
        same(k, q, scale)


def test_rounding_of_every_value(gpu):
    """Every bf16 value, in rows whose largest is at and next to the borders of a scale; NaN and infinities."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    D, P = 128, 64
    x = bits.view(512, 1, D)
    order = torch.argsort(torch.nan_to_num(x.float().abs(), 0.0, 0.0).amax((1, 2)))
    for rows_of in (x, x[order]):
        k, v = pools(D, P, 1, 8)
        q, scale = k.layer_q.cpu().numpy(), k.layer_scale.cpu().numpy()
        y = torch.flip(rows_of, (0,)).contiguous()
        ti.store_kv_(BE, k, v, rows_of.contiguous().cuda(), y.cuda(), i32(range(1, 513)))
        store(q, scale, rows_of.float().numpy(), y.float().numpy(), range(1, 513))
        same(k, q, scale)
    # one token at a time: blocks grow, and hold what is zero or not finite
    k, v = pools(D, 16, 1, 6)
    q, scale = k.layer_q.cpu().numpy(), k.layer_scale.cpu().numpy()
    for i, top in enumerate([0.0, 2.0 ** -133, 448.0, 449.0, 448.0 * 2 ** 20, math.inf, math.nan, 3e38, 1.0, 464.0, 896.0]):
        a = torch.linspace(-1, 1, D).mul(0.0 if not math.isfinite(top) else top).view(1, 1, D).float()
        a[0, 0, 3] = top
        ti.store_kv_(BE, k, v, a.cuda(), (-a).cuda(), i32([i + 18]))
        store(q, scale, a.numpy(), -a.numpy(), [i + 18])
        same(k, q, scale)


@pytest.mark.parametrize("T", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("D,nq,H,P,n", [(128, 8, 2, 16, 1), (128, 8, 2, 16, 37), (64, 6, 3, 64, 200), (128, 32, 8, 64, 300), (64, 7, 1, 32, 33)])
def test_fused_inputs_are_the_ops_in_a_row(gpu, T, norm, D, nq, H, P, n):
    g = np.random.Generator(np.random.PCG64(n + D))
    pages = 3 * n // P + 4
    a, b = pools(D, P, H, pages, g), None
    b = ti.fp8_kv_pools(D, P, H, pages)
    b[0].layer_q.copy_(a[0].layer_q)
    b[0].layer_scale.copy_(a[0].layer_scale)
    qkv = torch.from_numpy(g.standard_normal((n, (nq + 2 * H) * D)).astype(np.float32)).to(T).cuda()
    table = ti.RotaryTable.build(D, 600, 1e4, T)
    pos = i32(g.integers(0, 600, n))
    slots = i32(g.permutation(pages * P)[:n] + 1)
    bad = n > 30
    if bad:
        pos[3], pos[9], slots[5], slots[17] = 600, -1, 0, pages * P + 5
    wq, wk = ((torch.rand(D, device="cuda") + 0.5).to(T) for _ in range(2))
    q = torch.full((n, nq, D), 5.0, dtype=T, device="cuda")
    ti.attention_inputs_(BE, q, *a, qkv, wq if norm else None, wk if norm else None, table, pos, slots, 1e-6)
    x = qkv.view(n, nq + 2 * H, D)
    heads = x[:, :nq + H].contiguous()
    if norm:
        heads[:, :nq] = ti.rmsnorm(BE, heads[:, :nq].contiguous(), wq, 1e-6)
        heads[:, nq:] = ti.rmsnorm(BE, heads[:, nq:].contiguous(), wk, 1e-6)
    c, s = table.cos_sin[:, 0].contiguous(), table.cos_sin[:, 1].contiguous()
    turned = ti.rope(BE, heads, c, s, pos)
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    if bad:
        keep[[3, 9]] = False
    ti.store_kv_(BE, *b, turned[keep][:, nq:].contiguous(), x[keep][:, nq + H:].contiguous(), slots[keep].contiguous())
    assert torch.equal(q[keep], turned[keep][:, :nq]) and bool((q[~keep] == 5).all())
    assert torch.equal(a[0].layer_scale, b[0].layer_scale) and torch.equal(a[0].layer_q, b[0].layer_q)


def long_slots(g, n, P, pages):
    """Mostly runs in order, as prompts are; among them single tokens of other sequences, slots again, slots outside."""
    at, free = [], list(g.permutation(pages) * P)
    while len(at) < n:
        run = int(g.integers(1, 6 * P))
        take = [free.pop() for _ in range(min(-(-run // P), len(free)))]
        at += [b + o + 1 for b in take for o in range(P)][:run]
        if not free:
            free = list(g.permutation(pages) * P)
    at = np.array(at[:n], np.int64)
    where = g.integers(0, n, n // 50)
    at[where] = g.integers(1, pages * P + 1, len(where))
    where = g.integers(0, n, 40)
    at[where] = g.choice([0, -1, -2 ** 31, 2 ** 31 - 1, pages * P + 1], 40)
    return at


@pytest.mark.parametrize("T,D,H,P,n,aligned", [(torch.bfloat16, 128, 8, 16, 20000, True), (torch.bfloat16, 64, 8, 64, 40001, True),
                                               (torch.float32, 64, 5, 32, 17000, True), (torch.bfloat16, 64, 17, 16, 9000, False),
                                               (torch.bfloat16, 64, 4, 16, 70003, True), (torch.float32, 64, 8, 256, 20000, True)])
def test_long_calls(gpu, T, D, H, P, n, aligned):
    """Calls whose work-groups take several heads and pages each, into blocks that hold rows already."""
    g = np.random.Generator(np.random.PCG64(n))
    pages = n // P + 50
    k, v = pools(D, P, H, pages, g)
    q, scale = k.layer_q.cpu().numpy(), k.layer_scale.cpu().numpy()
    at = long_slots(g, n, P, pages)
    x, y = rows(g, n, H, D, T), rows(g, n, H, D, T)
    slots = torch.empty(n + 1, dtype=torch.int32, device="cuda")[0 if aligned else 1:][:n].copy_(i32(at))
    ti.store_kv_(BE, k, v, x.cuda(), y.cuda(), slots)
    store(q, scale, x.float().numpy(), y.float().numpy(), at)
    same(k, q, scale)


@pytest.mark.parametrize("tokens", [(1, 17), (3, 17), (1, 32), (1, 33), (1, 64), (8, 8), (1, 256), (1, 257), (5, 51)])
@pytest.mark.parametrize("H,P", [(8, 64), (3, 16)])
def test_few_tokens_of_a_page(gpu, tokens, H, P):
    """Few tokens, one after the other in a page or more of each sequence."""
    seqs, each = tokens
    g = np.random.Generator(np.random.PCG64(seqs * each))
    pages = seqs * (each // P + 2)
    k, v = pools(128, P, H, pages, g)
    q, scale = k.layer_q.cpu().numpy(), k.layer_scale.cpu().numpy()
    for start in (0, 5):
        at = [b * (each // P + 2) * P + start + t + 1 for b in range(seqs) for t in range(each)]
        x, y = rows(g, len(at), H, 128, torch.bfloat16), rows(g, len(at), H, 128, torch.bfloat16)
        ti.store_kv_(BE, k, v, x.cuda(), y.cuda(), i32(at))
        store(q, scale, x.float().numpy(), y.float().numpy(), at)
        same(k, q, scale)


def test_long_fused_inputs_are_the_ops_in_a_row(gpu):
    test_fused_inputs_are_the_ops_in_a_row(gpu, torch.bfloat16, True, 128, 2, 8, 16, 20000)


CASES = [
    ([(300, 1)], 4, 16), ([(0, 1)], 4, 16), ([(4000, 1), (1, 1), (999, 1)], 4, 64), ([(200, 5), (40, 0), (3, 2)], 4, 16),
    ([(500, 16), (90, 16)], 4, 64), ([(0, 333)], 4, 16), ([(150, 200), (0, 64)], 4, 64), ([(700, 1)] * 40, 4, 16), ([(64, 1), (10, 1)], 33, 16),
    ([(100, 3)], 16, 32), ([(1000, 600)], 3, 64), ([(0, 1500)], 1, 64), ([(60, 129)], 64, 16), ([(10, 140)] * 20, 4, 16),
]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens,G,P", CASES)
def test_attention(gpu, D, causal, lens, G, P):
    s = Step("fp8", lens, D=D, G=G, P=P, seed=G)
    k, v = s.layer.device()
    tables, positions, starts = s.args()
    q = s.q.cuda()
    out = torch.full_like(q, 7.0)
    ws = ti.attention_workspace(BE, q, k, len(lens), s.most)
    ti.paged_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, causal, starts, s.most)
    check(out, *s.want(causal), s.T)


@pytest.mark.parametrize("lens,G,P", CASES[:8])
def test_float32_queries(gpu, lens, G, P):
    s = Step("fp8", lens, G=G, P=P, seed=G, dtype=torch.float32)
    k, v = s.layer.device()
    tables, positions, starts = s.args()
    q = s.q.cuda()
    out = torch.empty_like(q)
    ti.paged_attention_(BE, out, ti.attention_workspace(BE, q, k, len(lens), s.most), q, k, v, tables, positions, s.scale, True, starts, s.most)
    check(out, *s.want(), s.T)


@pytest.mark.parametrize("path", range(8))
def test_paths(gpu, path):
    """Every path runs (the decode kernel or the library's pick), with a workspace and where it may without one."""
    for lens in ([(300, 4), (77, 4)], [(0, 90)]):
        s = Step("fp8", lens, P=16, seed=path)
        if path == ti.TI_PATH_DECODE and s.most * s.G > 64:
            continue
        k, v = s.layer.device()
        tables, positions, starts = s.args()
        q = s.q.cuda()
        out = torch.empty_like(q)
        ws = ti.attention_workspace(BE, q, k, len(lens), s.most, path)
        ti.paged_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, True, starts, s.most, path)
        check(out, *s.want(), s.T)


def test_one_sequence_and_allocating_forms(gpu):
    s = Step("fp8", [(210, 3)], seed=1)
    k, v = s.layer.device()
    tables, positions, _ = s.args()
    check(ti.attention(BE, s.q.cuda(), k, v, tables[0], positions, s.scale), *s.want(), s.T)


def test_a_chat(gpu):
    """A cache filled by a prompt and single tokens, taken back and written again: what attention returns is that of the
    values the cache stands for, and these are near what was written."""
    D, H, HQ, P = 128, 2, 8, 16
    cache = ti.PagedKVCache(1, D, H, 12, page_size=P, quantize="fp8")
    k, v = cache.k[0], cache.v[0]
    seq = cache.new_sequence()
    g = torch.Generator(device="cuda").manual_seed(1)
    keys, values = torch.zeros((0, H, D), device="cuda"), torch.zeros((0, H, D), device="cuda")
    for step, n in enumerate([50, 1, 1, 5, 1, 33]):
        if step == 4:
            ti.truncate(cache.blocks, seq, 53)
            keys, values = keys[:53], values[:53]
        start = len(seq)
        ti.reserve(cache.blocks, seq, n)
        x, y = (torch.randn((n, H, D), generator=g, device="cuda").bfloat16() for _ in range(2))
        ti.store_kv_(BE, k, v, x, y, i32(ti.slots(cache.blocks, seq, start, n)))
        seq.tokens.extend([0] * n)
        keys, values = torch.cat([keys, x.float()]), torch.cat([values, y.float()])
        q = torch.randn((n, HQ, D), generator=g, device="cuda").bfloat16()
        out = ti.attention(BE, q, k, v, i32(seq.block_table), i32(range(start, start + n)), D ** -0.5)
        at = torch.arange(start + n, device="cuda")
        page = torch.tensor(seq.block_table, device="cuda")[at // P] - 1
        kc, vc = k.values()[page, :, at % P], v.values()[page, :, at % P]
        # values: half a step of e4m3 (2^-4), or of the smallest step at the block's scale (2^-10, at most 8 / 448 * 2 of it)
        assert bool(((kc - keys).abs() <= keys.abs() / 16 + 2.0 ** -10 / 16).all())
        s = torch.einsum("nhgd,khd->hgnk", q.double().cpu().view(n, H, HQ // H, D), kc.double().cpu()) * D ** -0.5
        s = s.masked_fill(torch.arange(start + n)[None] > torch.arange(start, start + n)[:, None], -math.inf)
        w = torch.softmax(s, 3)
        want = torch.einsum("hgnk,khd->nhgd", w, vc.double().cpu()).reshape(n, HQ, D).numpy()
        size = torch.einsum("hgnk,khd->nhgd", w, vc.double().cpu().abs()).reshape(n, HQ, D).numpy()
        check(out, want, size, torch.bfloat16)


def test_noalloc_and_graphs(gpu):
    import ctypes

    from tileinfer_hip import _lib
    from tileinfer_hip.backend import _attention_args, _stream, kv_cache_struct
    for lens in ([(900, 1), (300, 1)], [(40, 60)]):
        s = Step("fp8", lens, P=16, seed=3)
        k, v = s.layer.device()
        tables, positions, starts = s.args()
        q = s.q.cuda()
        out = torch.empty_like(q)
        a = _attention_args(out, q, tables, positions, s.scale, True, 0, len(lens), s.most, starts, None)
        c = kv_cache_struct(k, v)
        _lib.check(_lib.load().ti_attention_noalloc(ctypes.byref(a), ctypes.byref(c), _stream(q)))
        check(out, *s.want(), s.T)
        ws = ti.attention_workspace(BE, q, k, len(lens), s.most)
        graph = torch.cuda.CUDAGraph()
        n = i32(range(1, 1 + s.tokens))
        new = torch.randn((s.tokens, s.H, s.D), device="cuda").bfloat16()
        with torch.cuda.graph(graph):
            ti.store_kv_(BE, k, v, new, new, n)
            ti.paged_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, True, starts, s.most)
        for r in range(3):
            new.normal_()
            graph.replay()
            torch.cuda.synchronize()
            again = torch.empty_like(q)
            ti.store_kv_(BE, k, v, new, new, n)
            ti.paged_attention_(BE, again, ws, q, k, v, tables, positions, s.scale, True, starts, s.most)
            assert torch.equal(out, again)


@pytest.mark.parametrize("T", [torch.bfloat16, torch.float32])
def test_tensors_aligned_to_their_elements_only(gpu, T):
    def shifted(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        room[1:].copy_(t.reshape(-1))
        return room[1:].view(t.shape)

    g = np.random.Generator(np.random.PCG64(8))
    D, P, H = 128, 16, 2
    for n in (1, 40, 600):
        k, v = pools(D, P, H, 40, g)
        q, scale = k.layer_q.cpu().numpy(), k.layer_scale.cpu().numpy()
        x, y = rows(g, n, H, D, T), rows(g, n, H, D, T)
        at = list(g.permutation(40 * P)[:n] + 1)
        ti.store_kv_(BE, k, v, shifted(x), shifted(y), shifted(i32(at)))
        store(q, scale, x.float().numpy(), y.float().numpy(), at)
        same(k, q, scale)


def test_positions_that_no_table_holds(gpu):
    for lens in ([(100, 1), (50, 1)], [(100, 5), (50, 5)], [(100, 60), (50, 60)]):
        s = Step("fp8", lens, seed=13)
        want, size = s.want()
        n = lens[0][1]
        k, v = s.layer.device()
        q = s.q.cuda()
        for first in (2 ** 31 - 1, 10 ** 6):
            s.positions[0] = first
            tables, positions, starts = s.args()
            out = torch.zeros_like(q)
            ws = ti.attention_workspace(BE, q, k, 2, n)
            ti.paged_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, True, starts, n)
            torch.cuda.synchronize()
            check(out[n:], want[n:], size[n:], s.T)
