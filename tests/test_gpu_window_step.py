"""The step of a serving batch with a sliding window, as a program runs it: pages reserved on the GPU, the step's keys and
values written, attention, and what is not kept given back; eagerly, on another stream and as one captured graph."""
import math

import numpy as np
import pytest
import torch

import tileinfer_hip as ti
from window_ref import check, i32

pytestmark = pytest.mark.gpu
BE = ti.HipBackend()
H, HQ, D, EPS = 2, 8, 128, 1e-6


class Server:
    """A layer's cache of a kind, its pages on the GPU, and on the host what every sequence has been told."""

    def __init__(self, quantize, P, S, pages, width, window, sinks, room, seed):
        smooth = [torch.exp2(torch.randint(-1, 2, (D // 2,)).float()).repeat(2)] if quantize == "int8" else None
        self.cache = ti.PagedKVCache(1, D, H, pages, page_size=P, quantize=quantize, key_smoothing=smooth)
        self.pool = ti.page_pool(pages, P, S, width, window, sinks)
        self.P, self.S, self.window, self.sinks, self.room = P, S, window, sinks, room
        self.table = ti.RotaryTable.build(D, width * P, 1e5)
        self.g = torch.Generator(device="cuda").manual_seed(seed)
        i = dict(dtype=torch.int32, device="cuda")
        self.counts, self.keep = torch.zeros(S, **i), torch.zeros(S, **i)
        self.pos, self.slots, self.qsl, self.short = torch.zeros(room, **i), torch.zeros(room, **i), torch.zeros(S + 1, **i), torch.zeros(1, **i)
        self.qkv = torch.zeros((room, (HQ + 2 * H) * D), device="cuda", dtype=torch.bfloat16)
        self.q = torch.zeros((room, HQ, D), device="cuda", dtype=torch.bfloat16)
        self.out = torch.zeros_like(self.q)
        self.scale = D ** -0.5
        self.ws = {}

    def run(self, most):
        """The step's calls: nothing in them depends on the host but `most`."""
        k, v = self.cache.k[0], self.cache.v[0]
        if most not in self.ws:
            self.ws[most] = ti.window_attention_workspace(BE, self.q, k, self.window, self.sinks, self.S, most)
        ti.reserve_pages_(BE, self.pool, self.counts, self.pos, self.slots, self.qsl, self.short)
        ti.attention_inputs_(BE, self.q, k, v, self.qkv, None, None, self.table, self.pos, self.slots, EPS)
        ti.window_attention_(BE, self.out, self.ws[most], self.q, k, v, self.pool.tables, self.pos, self.scale, self.window, self.sinks,
                             self.qsl, most)

    def give_back(self):
        ti.release_pages_(BE, self.pool, self.keep)

    def look(self, before, counts):
        """The outputs against the definition over what the cache now holds, page by page."""
        assert int(self.short) == 0
        tables = self.pool.tables.cpu().numpy()
        k, v = self.cache.k[0], self.cache.v[0]
        if self.cache.quantize == "fp8":
            hk, hv = (x.values().double().cpu().numpy() for x in (k, v))
        elif self.cache.quantize == "int8":
            hk, hv = ((x.q.double() * x.scale.double()[..., None]).cpu().numpy() for x in (k, v))
            hk = hk * k.smooth.double().cpu().numpy()
        else:
            hk, hv = k.double().cpu().numpy(), v.double().cpu().numpy()
        q = self.q.double().cpu().numpy()
        starts = np.concatenate([[0], np.cumsum(counts)])
        assert self.qsl.tolist() == starts.tolist()
        want, size = np.zeros((starts[-1], HQ, D)), np.zeros((starts[-1], HQ, D))
        for b, (c, n) in enumerate(zip(before, counts)):
            for t in range(n):
                p, row = c + t, starts[b] + t
                i = np.arange(p + 1)
                i = i[(i > p - self.window) | (i < self.sinks)]
                page, off = tables[b][i // self.P] - 1, i % self.P
                assert (page >= 0).all()
                for h in range(H):
                    s = q[row, h * 4:h * 4 + 4] @ hk[page, h, off].T * self.scale
                    w = np.exp(s - s.max(1, keepdims=True))
                    w /= w.sum(1, keepdims=True)
                    want[row, h * 4:h * 4 + 4] = w @ hv[page, h, off]
                    size[row, h * 4:h * 4 + 4] = w @ np.abs(hv[page, h, off])
        check(self.out[:starts[-1]], want, size, torch.bfloat16)


@pytest.mark.parametrize("quantize", [None, "int8", "fp8"])
@pytest.mark.parametrize("P,window,sinks", [(16, 70, 4), (64, 40, 0), (16, 5, 33)])
def test_serving(gpu, quantize, P, window, sinks):
    S, width = 4, 40 * 16 // P
    s = Server(quantize, P, S, S * (window // P + 4 + sinks // P) + 500 // P, width, window, sinks, 520, seed=P + window)
    lengths, g = [0] * S, np.random.Generator(np.random.PCG64(window))
    least = None
    for r in range(14):
        if r in (0, 9):
            counts = [250, 130, 3, 0] if r == 0 else [1, 0, 200, 140]      # prompts, one of them in a finished chat's place
        elif r % 3 == 1:
            counts = [int(x) for x in g.integers(0, 6, S)]                    # drafted blocks
        else:
            counts = [1] * S
        s.counts.copy_(i32(counts))
        s.qkv.normal_(generator=s.g)
        s.out.fill_(9.0)
        if r % 2:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                s.run(max(counts))
            torch.cuda.current_stream().wait_stream(side)
        else:
            s.run(max(counts))
        s.look(lengths, counts)
        assert bool((s.out[sum(counts):] == 9).all())
        lengths = [c + n for c, n in zip(lengths, counts)]
        if r % 3 == 1:
            lengths = [max(n - int(g.integers(0, max(c, 1))), 0) for n, c in zip(lengths, counts)]   # rejected drafts
        if r == 8:
            lengths[2], lengths[3] = 0, 0                                     # finished
        s.keep.copy_(i32(lengths))
        s.give_back()
        held = int((s.pool.tables > 0).sum())
        assert held + int(s.pool.free_count) == s.cache.num_pages()
        most = sum(min(-(-n // P), (window - 2) // P + 2 + -(-sinks // P)) for n in lengths)
        assert held <= most                                                  # nothing behind the window is held
        least = held if least is None else min(least, held)
    ids = torch.cat([s.pool.tables[s.pool.tables > 0], s.pool.free[:int(s.pool.free_count)]])
    assert ids.sort().values.tolist() == list(range(1, s.cache.num_pages() + 1))


@pytest.mark.parametrize("quantize", [None, "int8", "fp8"])
def test_a_captured_step(gpu, quantize):
    """One graph of a whole step, replayed as the chats grow, with eager work between the replays."""
    P, S, window, sinks = 16, 3, 50, 4
    s = Server(quantize, P, S, 40, 60, window, sinks, 12, seed=5)
    s.counts.fill_(4)
    s.run(4)                                                                 # (a first run outside of the graph)
    s.keep.zero_()
    s.give_back()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.run(4)
        s.give_back()
    lengths, g = [0] * S, np.random.Generator(np.random.PCG64(1))
    for r in range(90):
        counts = [int(x) for x in g.integers(0, 5, S)]
        keep = [n + int(g.integers(0, c + 1)) for n, c in zip(lengths, counts)]
        s.counts.copy_(i32(counts))
        s.keep.copy_(i32(keep))
        s.qkv.normal_(generator=s.g)
        state = [t.clone() for t in (s.pool.free, s.pool.free_count, s.pool.tables, s.pool.lengths, s.pool.behind)]
        layer = [t.clone() for t in ([s.cache.k[0], s.cache.v[0]] if quantize is None else [s.cache.k[0].layer_q, s.cache.k[0].layer_scale])]
        graph.replay()
        torch.cuda.synchronize()
        got, after = s.out.clone(), s.pool.tables.clone()
        # the same eagerly, from the same state
        for t, x in zip((s.pool.free, s.pool.free_count, s.pool.tables, s.pool.lengths, s.pool.behind), state):
            t.copy_(x)
        for t, x in zip([s.cache.k[0], s.cache.v[0]] if quantize is None else [s.cache.k[0].layer_q, s.cache.k[0].layer_scale], layer):
            t.copy_(x)
        s.run(4)
        n = sum(counts)
        assert torch.equal(s.out[:n], got[:n])
        s.look(lengths, counts)
        s.give_back()
        assert torch.equal(s.pool.tables, after) and s.pool.lengths.tolist() == keep
        lengths = keep
    assert max(lengths) > window + 2 * P
