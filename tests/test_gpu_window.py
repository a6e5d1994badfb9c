"""window_attention_ against its definition in 64 bits: caches of every kind, one token to long prompts, odd windows, sinks
and pages, ragged steps with empty sequences, pages that were given back, and garbage (NaN where the cache's kind has it)
in every row that no query sees and in rows that only others see."""
import math

import numpy as np
import pytest
import torch

import tileinfer_hip as ti
from window_ref import Step, check, i32

pytestmark = pytest.mark.gpu
BE = ti.HipBackend()
KINDS = ("bf16", "fp32", "int8", "fp8")


def run(s, window=None, sinks=None, out=None, workspace=None, uniform=False):
    k, v = s.layer.device()
    tables, positions, starts = s.args()
    q = s.q.cuda()
    if out is None:
        out = torch.full_like(q, 7.0)
    W, S = s.window if window is None else window, s.sinks if sinks is None else sinks
    ws = ti.window_attention_workspace(BE, q, k, W, S, len(s.lens), s.most) if workspace is None else workspace
    if uniform:
        return ti.window_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, W, S)
    return ti.window_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, W, S, starts, s.most)


STEPS = {
    "token": [(300, 1)],
    "first": [(0, 1)],
    "tokens": [(300, 1), (0, 1), (1, 1), (63, 1), (64, 1), (777, 1)],
    "block": [(200, 5), (3, 2), (40, 0), (129, 7)],
    "drafts": [(500, 16), (90, 16), (31, 9)],
    "prompt": [(0, 333)],
    "ragged": [(0, 200), (150, 33), (0, 1), (700, 1), (64, 64), (10, 0)],
}


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("step", STEPS)
@pytest.mark.parametrize("window,sinks", [(64, 4), (1, 0), (17, 0), (100, 33), (4096, 5)])
def test_steps(gpu, kv, step, window, sinks):
    s = Step(kv, STEPS[step], window, sinks, seed=len(step))
    check(run(s), *s.want(), s.T)


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("D,H,G,P", [(64, 2, 4, 16), (64, 1, 8, 64), (128, 3, 1, 32), (128, 1, 3, 64), (128, 2, 16, 16), (64, 1, 33, 16),
                                     (128, 1, 64, 128)])
@pytest.mark.parametrize("lens", [[(250, 1), (80, 1)], [(130, 6)], [(40, 100)]])
def test_heads_and_pages(gpu, kv, D, H, G, P, lens):
    s = Step(kv, lens, 70, 3, D=D, H=H, G=G, P=P, seed=G)
    check(run(s), *s.want(), s.T)


@pytest.mark.parametrize("kv", ["bf16", "fp32", "int8"])
@pytest.mark.parametrize("P", [1, 5, 8, 24, 48])
@pytest.mark.parametrize("lens", [[(250, 1), (80, 1)], [(130, 6)], [(40, 100), (0, 9)]])
def test_odd_pages(gpu, kv, P, lens):
    s = Step(kv, lens, 70, 3, P=P, seed=P)
    check(run(s), *s.want(), s.T)


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("lens,window,sinks", [([(5000, 1)] * 3, 2000, 4), ([(3000, 300)], 1000, 0), ([(0, 1300)], 300, 50),
                                               ([(2100, 16)] * 4, 1500, 4), ([(900, 1)] * 40, 512, 1), ([(100, 520)] * 3, 129, 0)])
def test_longer(gpu, kv, lens, window, sinks):
    s = Step(kv, lens, window, sinks, P=64, H=2, G=4, seed=5)
    check(run(s), *s.want(), s.T)


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("lens", [[(100, 1)], [(90, 9)], [(0, 70)]])
def test_window_past_everything(gpu, kv, lens):
    """A window or sinks of 2^31 - 1 are all keys."""
    s = Step(kv, lens, 0, 0, seed=2)
    want = s.want()
    check(run(s, 2 ** 31 - 1, 0), *want, s.T)
    check(run(s, 2 ** 31 - 1, 2 ** 31 - 1), *want, s.T)
    check(run(s, 1, 2 ** 31 - 1), *want, s.T)


@pytest.mark.parametrize("kv", KINDS)
def test_uniform_steps(gpu, kv):
    s = Step(kv, [(70, 6), (200, 6), (0, 6)], 50, 2, seed=3)
    check(run(s, uniform=True), *s.want(), s.T)


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("most", [3, 40, 300])
def test_rows_of_no_sequence(gpu, kv, most):
    """Rows in front of the first and behind the last sequence stay as they were; a max_query_len larger than any count."""
    s = Step(kv, [(60, 3), (9, 0), (33, 2)], 40, 4, seed=4)
    k, v = s.layer.device()
    tables, _, _ = s.args()
    front, behind = 4, 6
    q = torch.cat([torch.full((front, *s.q.shape[1:]), math.nan), s.q.float(), torch.full((behind, *s.q.shape[1:]), math.nan)]).to(s.T).cuda()
    pos = torch.cat([i32([10 ** 6] * front), i32(s.positions), i32([-5] * behind)])
    out = torch.full_like(q, 3.0)
    ws = ti.window_attention_workspace(BE, q, k, 40, 4, 3, most)
    ti.window_attention_(BE, out, ws, q, k, v, tables, pos, s.scale, 40, 4, i32(s.starts) + front, most)
    check(out[front:front + s.tokens], *s.want(), s.T)
    assert bool((out[:front] == 3).all()) and bool((out[front + s.tokens:] == 3).all())


@pytest.mark.parametrize("kv", ["bf16", "fp32", "fp8"])
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("lens,at", [([(40, 24)], 30), ([(300, 16), (20, 3)], 290), ([(0, 200)], 100), ([(100, 1), (80, 1)], 95)])
def test_rows_that_only_some_see(gpu, kv, half, value, lens, at):
    """A row that is not finite reaches the queries that see it alone."""
    window, sinks = 20, 2
    s = Step(kv, lens, window, sinks, seed=6)
    page = int(s.tables[0][at // s.P]) - 1
    s.layer.put(half, page, 1, at % s.P, value)
    with np.errstate(all="ignore"):
        want, size = s.want()
    got = run(s).double().cpu().numpy()
    c, n = lens[0]
    sees = np.zeros(s.tokens, bool)
    sees[:n] = [at <= c + t and at > c + t - window for t in range(n)]
    heads = np.zeros(s.H * s.G, bool)
    heads[s.G:2 * s.G] = True
    hit = sees[:, None] & heads[None]
    fine = ~hit
    assert sees.any() and (n == 1 or not sees[:n].all())
    from window_ref import tolerance
    assert np.isfinite(got[fine]).all()
    assert (np.abs(got - want)[fine] <= tolerance(s.T, want, size)[fine]).all()
    if half == 1:
        gone = np.nan if kv == "fp8" or math.isnan(value) else value
        assert np.array_equal(got[hit], np.full(got[hit].shape, gone), equal_nan=True)
    elif math.isnan(value) or kv == "fp8":
        assert np.isnan(got[hit]).all()


def test_garbage_tables(gpu):
    """Entries of pages that hold no visible key may be anything; visible ones outside the pool are clamped into it."""
    for kv in KINDS:
        s = Step(kv, [(500, 1), (300, 4), (64, 40)], 30, 2, seed=8)
        want = s.want()
        hidden = s.tables == 0
        s.tables[hidden] = np.resize([2 ** 31 - 1, -2 ** 31, 10 ** 9, -1], int(hidden.sum()))
        check(run(s), *want, s.T)
        s.tables[:] = 2 ** 31 - 1
        run(s)
        torch.cuda.synchronize()


def test_large_pool_offsets(gpu):
    """Pages past element 2^31 of a pool, and past 2^32 of an 8-bit layer."""
    H, P, D, G = 8, 64, 128, 4
    for kv, pages in (("bf16", 33000), ("fp8", 66000)):
        if kv == "bf16":
            k = torch.zeros((pages, H, P, D), dtype=torch.bfloat16, device="cuda")
            v = torch.zeros_like(k)
            ids = torch.tensor([pages, 5, pages - 1, pages - 7], device="cuda")
            k[ids - 1] = torch.randn((4, H, P, D), device="cuda").bfloat16()
            v[ids - 1] = torch.randn((4, H, P, D), device="cuda").bfloat16()
            kd, vd = k[ids - 1].double(), v[ids - 1].double()
        else:
            k, v = ti.fp8_kv_pools(D, P, H, pages)
            ids = torch.tensor([pages, 5, pages - 1, pages - 7], device="cuda")
            codes = (torch.randn((2, 4, H, P, D), device="cuda") * 60).to(torch.float8_e4m3fn)
            k.layer_q[:, ids - 1] = codes.view(torch.uint8)
            k.layer_scale[:, ids - 1] = 2.0 ** -6
            kd, vd = (codes.double() * 2.0 ** -6).unbind(0)
        kd, vd = (x.transpose(0, 1).reshape(H, 4 * P, D) for x in (kd, vd))
        for n in (1, 40):
            start = 4 * P - n
            q = torch.randn((n, H * G, D), device="cuda").bfloat16()
            pos = torch.arange(start, start + n, dtype=torch.int32, device="cuda")
            got = ti.window_attention(BE, q, k, v, ids.to(torch.int32)[None], pos, D ** -0.5, 150, 3)
            i = torch.arange(4 * P, device="cuda")
            see = (i <= pos[:, None]) & ((i > pos[:, None] - 150) | (i < 3))
            s = torch.einsum("nhgd,hkd->hgnk", q.double().cpu().view(n, H, G, D), kd.cpu()) * D ** -0.5
            w = torch.softmax(s.masked_fill(~see.cpu(), -math.inf), 3)
            want = torch.einsum("hgnk,hkd->nhgd", w, vd.cpu()).reshape(n, H * G, D).numpy()
            size = torch.einsum("hgnk,hkd->nhgd", w, vd.cpu().abs()).reshape(n, H * G, D).numpy()
            check(got, want, size, torch.bfloat16)
        del k, v
        torch.cuda.empty_cache()


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("lens", [[(700, 1), (30, 1)], [(90, 9)], [(20, 90)]])
def test_streams_and_graphs(gpu, kv, lens):
    """On another stream, and captured: replays with other queries, positions and tables, eager work between them."""
    s = Step(kv, lens, 60, 4, seed=9)
    want = s.want()
    k, v = s.layer.device()
    tables, positions, starts = s.args()
    q = s.q.cuda()
    out = torch.zeros_like(q)
    ws = ti.window_attention_workspace(BE, q, k, 60, 4, len(lens), s.most)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ti.window_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, 60, 4, starts, s.most)
    side.synchronize()
    check(out, *want, s.T)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ti.window_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, 60, 4, starts, s.most)
    first = q.clone()
    for r in range(4):
        out.zero_()
        q.copy_(first if r % 2 == 0 else torch.zeros_like(first))
        graph.replay()
        torch.cuda.synchronize()
        eager = ti.window_attention(BE, q, k, v, tables, positions, s.scale, 60, 4, starts, s.most)
        assert torch.equal(out, eager)
        if r % 2 == 0:
            check(out, *want, s.T)


def test_same_result_twice(gpu):
    for kv in KINDS:
        s = Step(kv, [(700, 3), (200, 130), (0, 40)], 100, 4, seed=10)
        a, b = run(s), run(s)
        assert torch.equal(a, b)


def test_rows_of_large_values_that_no_query_sees(gpu):
    """Hidden rows of a tile at a window's edge, finite and huge: no row-by-row path, no trace of them."""
    for kv, lens in (("bf16", [(200, 9), (90, 1)]), ("fp32", [(200, 9), (90, 1)]), ("fp8", [(200, 9), (90, 1)]), ("bf16", [(0, 200)]),
                     ("fp8", [(60, 200)]), ("fp32", [(60, 200)])):
        s = Step(kv, lens, 37, 3, seed=12)
        want = s.want()
        big = 3e4 if kv != "fp8" else 448.0
        for x, half in ((s.layer.k, 0), (s.layer.v, 1)):
            x[np.isnan(x)] = big
            if kv == "fp8":
                s.layer.q[half][s.layer.q[half] == 127] = 126
        if kv == "fp8":
            s.layer.scale[np.isnan(s.layer.scale)] = 2.0 ** 100
        check(run(s), *want, s.T)


def test_positions_that_no_table_holds(gpu):
    """Positions out of contract: every access stays inside, and the call ends; the other sequences are right."""
    for kv in KINDS:
        for n in (1, 5, 40):
            s = Step(kv, [(100, n), (50, n)], 30, 2, seed=13)
            want, size = s.want()
            s.positions[:n] = np.resize([2 ** 31 - 1, 2 ** 30, 10 ** 6, -2 ** 31], n)
            for first in (2 ** 31 - 1, 10 ** 6):
                s.positions[0] = first
                got = run(s)
                torch.cuda.synchronize()
                check(got[n:], want[n:], size[n:], s.T)


@pytest.mark.parametrize("kv", KINDS)
@pytest.mark.parametrize("lens", [[(300, 1)], [(100, 6), (40, 2)], [(30, 150)], [(100, 700)]])
def test_tensors_aligned_to_their_elements_only(gpu, kv, lens):
    def shifted(t):
        room = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        room[1:].copy_(t.reshape(-1))
        return room[1:].view(t.shape)

    s = Step(kv, lens, 64, 4, seed=14)
    k, v = s.layer.device()
    if kv in ("bf16", "fp32"):
        k, v = shifted(k), shifted(v)
    tables, positions, starts = (shifted(t) for t in s.args())
    q = shifted(s.q.cuda())
    out = shifted(torch.zeros_like(q))
    ws = ti.window_attention_workspace(BE, q, k, 64, 4, len(lens), s.most)
    ti.window_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, 64, 4, starts, s.most)
    check(out, *s.want(), s.T)


@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("value", [math.nan, math.inf])
@pytest.mark.parametrize("lens,at", [([(0, 200)], 77), ([(100, 130), (0, 33)], 160), ([(1000, 500)], 1400)])
def test_rows_that_only_later_queries_see(gpu, kv, half, value, lens, at):
    """A window over all that the tables hold: the rows in front of a row that is not finite are as without it."""
    window = 1 << 20
    s = Step(kv, lens, window, 0, seed=15)
    want, size = s.want()
    s.layer.put(half, int(s.tables[0][at // s.P]) - 1, 1, at % s.P, value)
    got = run(s).double().cpu().numpy()
    c, n = lens[0]
    hit = np.zeros(got.shape[:2], bool)
    hit[at - c:n, s.G:2 * s.G] = True
    from window_ref import tolerance
    assert np.isfinite(got[~hit]).all()
    assert (np.abs(got - want)[~hit] <= tolerance(s.T, want, size)[~hit]).all()
    if half == 1:
        assert not np.isfinite(got[hit]).any()


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("G", [1, 2, 3, 4, 32])
@pytest.mark.parametrize("lens", [[(0, 512)], [(1000, 200), (0, 0), (17, 65)], [(0, 33)] * 5])
def test_windows_over_whole_tables(gpu, kv, G, lens):
    """No key hidden but the later ones: the steps that run on other kernels than with hidden keys, and agree with them."""
    s = Step(kv, lens, 1 << 20, 0, G=G, seed=16)
    want = s.want()
    check(run(s), *want, s.T)
    most = max(c + n for c, n in lens)
    check(run(s, window=most), *want, s.T)      # the tables reach past the window, no query does


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n", [1, 5, 40, 300, 2000])
@pytest.mark.parametrize("window,G", [(40, 4), (1 << 20, 4), (700, 1)])
def test_queries_over_int8_caches_keep_11_bits(gpu, D, n, window, G):
    """Two keys of scores 64 and 64 (1 + 2^-9): half of the smoothing is 1 + 2^-9, which times a query of 1 has 10 bits, and
    bf16 holds 8. Their weights are to each other as 1 to e^(1/8), their values 1 and -1, so every output is -tanh(1/16);
    with such queries rounded to 8 bits it were 0. The other keys' scores are 0, their weights e^-64."""
    H, P, ctx = 2, 64, 70
    pages = -(-(ctx + n) // P)
    q8 = np.zeros((2, pages, H, P, D), np.int8)
    scale = np.full((2, pages, H, P), 1 / 127, np.float32)
    q8[0, 0, :, 0, :D // 2] = q8[0, 0, :, 1, D // 2:] = 127
    q8[1, 0, :, 0], q8[1, 0, :, 1] = 127, -127
    smooth = np.ones(D, np.float32)
    smooth[D // 2:] += 2.0 ** -9
    q8, scale, smooth = (torch.from_numpy(x).cuda() for x in (q8, scale, smooth))
    k, v = ti.Int8Pages(q8, scale, smooth, 0), ti.Int8Pages(q8, scale, torch.ones_like(smooth), 1)
    q = torch.ones((n, H * G, D), dtype=torch.bfloat16, device="cuda")
    positions = torch.arange(ctx, ctx + n, dtype=torch.int32, device="cuda")
    tables = torch.arange(1, pages + 1, dtype=torch.int32, device="cuda")[None]
    out = ti.window_attention(BE, q, k, v, tables, positions, 128 / D, window, 2).double().cpu()
    # the weights' rounding and the output's: 2^-8 of (weight times |value|) = 1 and of the output
    assert float((out + math.tanh(1 / 16)).abs().max()) <= 2.0 ** -8 * (1 + 1 / 16) + 2.0 ** -12
