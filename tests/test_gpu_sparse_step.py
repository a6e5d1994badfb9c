"""The chosen-page operators together, as a speculative step of a long chat runs them: the step's keys and
values into the cache, bounds, selection and attention for the drafted block, the verification of its
tokens, and the rejected positions given back; eagerly, on another stream, and in captured graphs."""
import math

import numpy as np
import pytest
import torch

import sparse_ref as ref
import tileinfer_hip as ti
from test_gpu_sparse import Cache, check_attend, i32, offsets

pytestmark = pytest.mark.gpu
BE = ti.HipBackend()
H, HQ, D, EPS = 2, 8, 128, 1e-6


class View:
    """A layer of a PagedKVCache as check_attend reads it."""

    def __init__(self, cache):
        self.k, self.v = cache.k[0], cache.v[0]
        self.P, self.H, self.D, self.pages = cache.page_size(), H, D, cache.num_pages()
        if cache.quantize:
            self.kv, self.smooth = "int8", self.k.smooth.cpu()
            q, s = self.k.layer_q.cpu().double().numpy(), self.k.layer_scale.cpu().double().numpy()
            self.hk = (self.k.q.float() * self.k.scale[..., None] * self.k.smooth).double().cpu().numpy()
            self.raw, self.hv, self.scales = q[0] * s[0][..., None], q[1] * s[1][..., None], s
        else:
            self.kv = "bf16"
            self.hk, self.hv = self.k.double().cpu().numpy(), self.v.double().cpu().numpy()

    def key_at(self, page, head, count):
        return self.hk[page, head, :count]


@pytest.mark.parametrize("quantize", [None, "int8"])
def test_speculative_steps(gpu, quantize):
    P, B, N, V, keep, sinks, window = 16, 3, 4, 1000, 12, 1, 2
    torch.manual_seed(3)
    smoothing = [torch.rand(D) + 0.5] if quantize else None
    cache = ti.PagedKVCache(1, D, H, 150, page_size=P, quantize=quantize, key_smoothing=smoothing, bounds=True)
    table = ti.RotaryTable.build(D, 2048, 1e6)
    seqs = [cache.new_sequence() for _ in range(B)]
    g = torch.Generator(device="cuda").manual_seed(4)

    def step(counts):
        """One step of counts[b] tokens; its attention, checked against what the cache then holds."""
        starts = [len(s) for s in seqs]
        for s, n in zip(seqs, counts):
            ti.reserve(cache.blocks, s, n)
        slots = i32([x for s, st, n in zip(seqs, starts, counts) for x in ti.slots(cache.blocks, s, st, n)])
        pos = i32([st + t for st, n in zip(starts, counts) for t in range(n)])
        width = max(len(s.block_table) for s in seqs)
        tables = i32([s.block_table + [0] * (width - len(s.block_table)) for s in seqs])
        rows = sum(counts)
        qkv = torch.randn((rows, (HQ + 2 * H) * D), generator=g, device="cuda").bfloat16()
        q = torch.empty((rows, HQ, D), device="cuda", dtype=torch.bfloat16)
        ti.attention_inputs_(BE, q, cache.k[0], cache.v[0], qkv, None, None, table, pos, slots, EPS)
        qsl, most, kb = offsets(counts), max(counts), cache.bounds[0]
        ti.update_key_bounds_(BE, kb, cache.k[0], cache.v[0], tables, pos, qsl, most)
        chosen, lengths = ti.select_pages(BE, q, kb, tables, pos, keep, sinks, window, True, qsl, most)
        v = View(cache)
        bounds, scale = kb.bounds.cpu().numpy(), kb.scale.cpu().numpy()
        row = 0
        for s, st, n in zip(seqs, starts, counts):
            want_b, want_s = bounds.astype(np.float64).copy(), scale.astype(np.float64).copy()
            ref.update_bounds(want_b, want_s, v.key_at, s.block_table, 0, st + n, P, H, v.pages)   # every page of it
            assert np.array_equal(want_b, bounds) and np.array_equal(want_s, scale)
            for t in range(n):
                ids, keys = ref.select(q[row].double().cpu().numpy(), bounds, scale, s.block_table, st + t, P, keep, sinks, window)
                assert np.array_equal(chosen[row].cpu().numpy(), ids) and np.array_equal(lengths[row].cpu().numpy(), keys)
                row += 1
        check_attend(v, q, chosen, lengths, qsl=qsl, n=most)
        for s, n in zip(seqs, counts):
            s.tokens.extend([0] * n)

    step([700, 150, 40])                                     # prompts
    kept = []
    for _ in range(6):
        counts = [N + 1] * B                                   # the last token and N drafts
        step(counts)
        logits = torch.randn((B, N + 1, V), generator=g, device="cuda")
        p = torch.softmax(logits, 2)
        d = torch.softmax(logits[:, :N] + 0.8 * torch.randn((B, N, V), generator=g, device="cuda"), 2)
        x = torch.multinomial(d.reshape(B * N, V), 1, generator=g).reshape(B, N).to(torch.int32)
        u = torch.rand((B, N + 1), generator=g, device="cuda")
        accepted, tokens = ti.verify_draft(BE, x, p, d, u)
        for b, s in enumerate(seqs):
            a, t = ref.verify(x[b].cpu().numpy(), p[b].cpu().numpy(), d[b].cpu().numpy(), u[b].cpu().numpy(), N)
            assert int(accepted[b]) == a and tokens[b].tolist() == t
            ti.truncate(cache.blocks, s, len(s) - (N - a))      # the rejected drafts' positions go back
            kept.append(a)
    assert 0 < sum(kept) < len(kept) * N                      # some were rejected, some accepted


def make_step(kv, B, n, keep, seed, ctx):
    c = Cache(kv, D, H, 16, ctx, seed)
    T = torch.float32 if kv == "fp32" else torch.bfloat16
    s = dict(c=c, pos=i32([0] * (B * n)), slots=i32([0] * (B * n)), qkv=torch.empty((B * n, (HQ + 2 * H) * D), device="cuda", dtype=T),
             q=torch.empty((B * n, HQ, D), device="cuda", dtype=T), kb=ti.key_bounds(D, 16, H, c.pages),
             tables=torch.zeros((B * n, H, keep), dtype=torch.int32, device="cuda"),
             lengths=torch.zeros((B * n, H), dtype=torch.int32, device="cuda"), n=n, B=B,
             table=ti.RotaryTable.build(D, 4096, 1e6, T))
    s["out"] = torch.empty_like(s["q"])
    if n > 1:
        V = 3000
        s["p"], s["d"] = torch.empty((B, n, V), device="cuda"), torch.empty((B, n - 1, V), device="cuda")
        s["x"], s["u"] = torch.zeros((B, n - 1), dtype=torch.int32, device="cuda"), torch.empty((B, n), device="cuda")
        s["accepted"], s["tokens"] = i32([0] * B), torch.zeros((B, n), dtype=torch.int32, device="cuda")
    return s


def workspaces(s):
    return (ti.select_pages_workspace(BE, s["q"], s["kb"], s["c"].tables),
            ti.sparse_attention_workspace(BE, s["q"], s["c"].k, s["tables"], s["n"]),
            ti.verify_draft_workspace(BE, s["p"]) if "p" in s else None)


def set_step(s, starts, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    pos = [st + t for st in starts for t in range(s["n"])]
    rows = [b for b in range(s["B"]) for _ in range(s["n"])]
    s["pos"].copy_(i32(pos))
    s["slots"].copy_(i32([(s["c"].rows[b][p // 16] - 1) * 16 + p % 16 + 1 for b, p in zip(rows, pos)]))
    s["qkv"].normal_(generator=g)
    if "p" in s:
        logits = torch.randn(s["p"].shape, generator=g, device="cuda")
        s["p"].copy_(torch.softmax(logits, 2))
        s["d"].copy_(torch.softmax(logits[:, :-1] + 0.5 * torch.randn(s["d"].shape, generator=g, device="cuda"), 2))
        s["x"].copy_(s["d"].argmax(2))
        s["u"].uniform_(generator=g)


def run_step(s, ws):
    c, n = s["c"], s["n"]
    ti.attention_inputs_(BE, s["q"], c.k, c.v, s["qkv"], None, None, s["table"], s["pos"], s["slots"], EPS)
    ti.update_key_bounds_(BE, s["kb"], c.k, c.v, c.tables, s["pos"], max_query_len=n)
    ti.select_pages_(BE, s["tables"], s["lengths"], ws[0], s["q"], s["kb"], c.tables, s["pos"], 1, 2, True, None, n)
    ti.sparse_attention_(BE, s["out"], ws[1], s["q"], c.k, c.v, s["tables"], s["lengths"], 1 / math.sqrt(D), None, n)
    if "p" in s:
        ti.verify_draft_(BE, s["accepted"], s["tokens"], ws[2], s["x"], s["p"], s["d"], s["u"])


def results(s):
    names = ["q", "tables", "lengths", "out"] + (["accepted", "tokens"] if "p" in s else [])
    return [s[k].clone() for k in names] + [s["kb"].bounds.clone(), s["kb"].scale.clone()]


@pytest.mark.parametrize("kv", ["bf16", "int8", "fp32"])
@pytest.mark.parametrize("B,n", [(1, 1), (5, 1), (2, 6)])
def test_graphs_replay_as_sequences_grow(gpu, kv, B, n):
    """Two graphs of the step share one set of workspaces; their replays, with eager work between, equal
    eager steps on a second cache bit for bit."""
    ctx = [700 + 90 * b for b in range(B)]
    captured, eager = (make_step(kv, B, n, 10, 5, ctx) for _ in range(2))
    ws, ews = workspaces(captured), workspaces(eager)
    starts = [c - 9 * n - 3 - 40 for c in ctx]
    set_step(captured, starts, 1)
    run_step(captured, ws)                      # warm: nothing is loaded during the capture
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run_step(captured, ws)
        graphs.append(g)
    captured, eager = captured, eager
    set_step(eager, starts, 1)
    run_step(eager, ews)
    for i in range(6):
        starts = [s + n + (7 if i == 3 else 0) for s in starts]
        set_step(captured, starts, 10 + i)
        set_step(eager, starts, 10 + i)
        run_step(eager, ews)
        want = results(eager)
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        for a, b in zip(results(captured), want):
            assert torch.equal(a, b), f"replay {i}"
        torch.randn((1 << 20,), device="cuda").sum().item()      # the program's own work between


def test_another_stream(gpu):
    """A step on a side stream that waits for the inputs: the same bits as on the default stream."""
    a, b = (make_step("bf16", 2, 4, 10, 6, [900, 500]) for _ in range(2))
    set_step(a, [800, 400], 2)
    set_step(b, [800, 400], 2)
    run_step(a, workspaces(a))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run_step(b, workspaces(b))
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(results(a), results(b)):
        assert torch.equal(x, y)


def test_two_calls_at_once(gpu):
    """Steps of two caches on two streams, each with its own workspaces."""
    steps = [make_step(kv, 3, 1, 10, 7, [900, 500, 100]) for kv in ("bf16", "bf16", "int8", "int8")]
    for s in steps:
        set_step(s, [880, 480, 90], 3)
    spaces = [workspaces(s) for s in steps]
    run_step(steps[0], spaces[0])
    run_step(steps[2], spaces[2])
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for st, s, ws in zip(streams, (steps[1], steps[3]), (spaces[1], spaces[3])):
            with torch.cuda.stream(st):
                run_step(s, ws)
    torch.cuda.synchronize()
    for i in (0, 2):
        for x, y in zip(results(steps[i]), results(steps[i + 1])):
            assert torch.equal(x, y)


def test_native_calls_and_ctypes_agree(gpu, monkeypatch):
    """Every op of the step through the native call path, and through backend.py's own checks."""
    from test_gpu_calls import _Counted, _NotPlain
    from tileinfer_hip import _lib
    ti.load_library()
    real = _lib.calls
    for kv in ("bf16", "int8", "fp32"):
        got = []
        for calls in (_Counted(real), _NotPlain()):
            monkeypatch.setattr(_lib, "calls", calls)
            s = make_step(kv, 2, 4, 10, 8, [900, 500])
            set_step(s, [800, 400], 4)
            run_step(s, workspaces(s))
            got.append(results(s))
            assert isinstance(calls, _NotPlain) or calls.made == 5, "an op was left to ctypes"
        for a, b in zip(*got):
            assert torch.equal(a, b)
