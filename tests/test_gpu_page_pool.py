"""reserve_pages_ and release_pages_ against BlockManager on the host, sequence by sequence; what they do when pages run
out, and steps taken back."""
import numpy as np
import pytest
import torch

import tileinfer_hip as ti
from window_ref import i32

pytestmark = pytest.mark.gpu
BE = ti.HipBackend()


class Host:
    """The same pool as lists: sequences in order for reserve, in the opposite order for release."""

    def __init__(self, pages, P, S, W, window=0, sinks=0):
        self.P, self.W, self.window, self.sinks = P, W, window, sinks
        self.free = list(range(pages, 0, -1))
        self.rows, self.lengths = [[0] * W for _ in range(S)], [0] * S

    def reserve(self, counts, room):
        P = self.P
        need = [-(-(n + max(c, 0)) // P) - -(-n // P) for n, c in zip(self.lengths, counts)]
        if any(n + max(c, 0) > self.W * P for n, c in zip(self.lengths, counts)) or sum(max(c, 0) for c in counts) > room:
            return [0] * room, [0] * room, [0] * (len(counts) + 1), -1
        if sum(need) > len(self.free):
            return [0] * room, [0] * room, [0] * (len(counts) + 1), sum(need) - len(self.free)
        positions, slots, starts = [], [], [0]
        for b, c in enumerate(counts):
            for p in range(self.lengths[b], self.lengths[b] + max(c, 0)):
                if p % P == 0:
                    self.rows[b][p // P] = self.free.pop()
                positions.append(p)
                slots.append((self.rows[b][p // P] - 1) * P + p % P + 1)
            starts.append(len(slots))
            self.lengths[b] += max(c, 0)
        pad = [0] * (room - len(slots))
        return positions + pad, slots + pad, starts, 0

    def release(self, keep):
        P = self.P
        for b in reversed(range(len(keep))):
            n = min(max(keep[b], 0), self.lengths[b])
            for i in reversed(range(self.W)):
                hidden = self.window and (i + 1) * P <= n - self.window + 1 and i * P >= self.sinks
                if self.rows[b][i] and (i * P >= n or hidden):
                    self.free.append(self.rows[b][i])
                    self.rows[b][i] = 0
            self.lengths[b] = n


def same(pool, host):
    assert pool.lengths.tolist() == host.lengths
    assert pool.tables.tolist() == host.rows
    n = int(pool.free_count)
    assert pool.free[:n].tolist() == host.free
    assert int(pool.ticket) == 0


def step(pool, host, counts, room):
    S = len(counts)
    pos, slots = (torch.full((room,), 9, dtype=torch.int32, device="cuda") for _ in range(2))
    qsl, short = torch.full((S + 1,), 9, dtype=torch.int32, device="cuda"), i32([9])
    ti.reserve_pages_(BE, pool, i32(counts), pos, slots, qsl, short)
    want = host.reserve(counts, room)
    assert (pos.tolist(), slots.tolist(), qsl.tolist(), int(short)) == (want[0], want[1], want[2], want[3])
    same(pool, host)
    return int(short)


@pytest.mark.parametrize("P", [16, 64, 5, 1])
@pytest.mark.parametrize("S,W,window,sinks", [(1, 40, 0, 0), (7, 30, 0, 0), (300, 12, 0, 0), (5, 60, 37, 0), (5, 60, 100, 20), (70, 40, 1, 4),
                                              (3, 30, 10 ** 6, 0), (4, 30, 50, 10 ** 6)])
def test_random_steps(gpu, P, S, W, window, sinks):
    g = np.random.Generator(np.random.PCG64(S + P))
    pages = S * W * 2 // 3 + 1
    pool, host = ti.page_pool(pages, P, S, W, window, sinks), Host(pages, P, S, W, window, sinks)
    refused = 0
    for r in range(24):
        most = [1, 5, P, 4 * P, W * P // 3][r % 5]
        counts = [int(x) for x in g.integers(-1, most + 1, S)]
        refused += step(pool, host, counts, sum(max(c, 0) for c in counts) + int(g.integers(0, 5))) != 0
        # rejected drafts, finished requests, others kept whole (and lengths that cannot be are clamped)
        back = 0 if window else int(g.integers(0, 2 * P))
        keep = [n if x > 0.3 else (0 if x < 0.1 else (n - back if not window else n + 5)) for n, x in zip(host.lengths, g.random(S))]
        ti.release_pages_(BE, pool, i32(keep))
        host.release(keep)
        same(pool, host)
    assert refused < 24


@pytest.mark.parametrize("P", [16, 3])
def test_cut_into_what_went_back(gpu, P):
    """A finished request, and one cut far back, on a pool with a window."""
    pool, host = ti.page_pool(40, P, 2, 20, 2 * P, P + 1), Host(40, P, 2, 20, 2 * P, P + 1)
    step(pool, host, [15 * P + 2, 9 * P], 30 * P)
    for keep in ([15 * P + 2, 9 * P], [7 * P + 1, 9 * P], [7 * P + 1, 3], [0, 0]):
        ti.release_pages_(BE, pool, i32(keep))
        host.release(keep)
        same(pool, host)
        step(pool, host, [2, P + 1], 40)


def test_taken_back_whole(gpu):
    """The stack, tables and lengths are as before the step, bit for bit."""
    g = np.random.Generator(np.random.PCG64(3))
    pool, host = ti.page_pool(5000, 16, 200, 40), Host(5000, 16, 200, 40)
    step(pool, host, [int(x) for x in g.integers(0, 300, 200)], 70000)
    state = [t.clone() for t in (pool.free, pool.free_count, pool.tables, pool.lengths)]
    before = pool.lengths.clone()
    for most in (1, 9, 200):
        counts = i32(g.integers(0, most + 1, 200))
        T = int(counts.sum())
        out = [torch.zeros(T, dtype=torch.int32, device="cuda") for _ in range(2)] + [torch.zeros(201, dtype=torch.int32, device="cuda"), i32([0])]
        ti.reserve_pages_(BE, pool, counts, *out)
        assert int(out[3]) == 0
        ti.release_pages_(BE, pool, before)
        for a, b in zip(state, (pool.free, pool.free_count, pool.tables, pool.lengths)):
            assert torch.equal(a, b)


def test_block_manager(gpu):
    """One sequence is BlockManager's."""
    P = 16
    pool, b, seq = ti.page_pool(30, P, 1, 30), ti.BlockManager(30, P), ti.Sequence()
    pos, slots = (torch.zeros(100, dtype=torch.int32, device="cuda") for _ in range(2))
    qsl, short = torch.zeros(2, dtype=torch.int32, device="cuda"), i32([0])
    for n, keep in ((50, 50), (1, 51), (30, 60), (100, 100), (7, 107), (3, 0), (40, 39)):
        start = len(seq)
        ti.reserve_pages_(BE, pool, i32([n]), pos, slots, qsl, short)
        ti.reserve(b, seq, n)
        assert slots[:n].tolist() == ti.slots(b, seq, start, n) and qsl.tolist() == [0, n]
        seq.tokens.extend([0] * n)
        ti.release_pages_(BE, pool, i32([keep]))
        ti.truncate(b, seq, keep)
        assert pool.free[:int(pool.free_count)].tolist() == b.free
        assert pool.tables[0].tolist()[:len(seq.block_table)] == seq.block_table and int(pool.tables.count_nonzero()) == len(seq.block_table)


def test_out_of_pages_and_room(gpu):
    pool, host = ti.page_pool(10, 16, 3, 8), Host(10, 16, 3, 8)
    assert step(pool, host, [60, 16, 20], 100) == 0           # 4 + 1 + 2 pages of 10
    assert step(pool, host, [4, 49, 0], 100) == 1             # one missing: nothing is given
    assert step(pool, host, [4, 48, 0], 100) == 0
    assert step(pool, host, [1, 0, 0], 100) == 1
    assert step(pool, host, [0, 65, 0], 100) == -1            # past its table
    assert step(pool, host, [0, 0, 12], 11) == -1             # past the step
    assert step(pool, host, [0, 0, 2 ** 31 - 1], 100) == -1
    assert step(pool, host, [-2 ** 31, 0, 12], 12) == 0
    assert step(pool, host, [0, 0, 0], 0) == 0


def test_many_sequences(gpu):
    g = np.random.Generator(np.random.PCG64(5))
    S, W = 4096, 6
    pool, host = ti.page_pool(S * W, 16, S, W), Host(S * W, 16, S, W)
    for _ in range(3):
        counts = [int(x) for x in g.integers(0, 30, S)]
        step(pool, host, counts, sum(counts) + 3)
        keep = [int(x) for x in g.integers(0, 60, S)]
        ti.release_pages_(BE, pool, i32(keep))
        host.release(keep)
        same(pool, host)


def test_captured(gpu):
    """A reserve and a release in one graph, replayed with other counts."""
    S, P = 9, 16
    pool, host = ti.page_pool(100, P, S, 20), Host(100, P, S, 20)
    counts, keep = (torch.zeros(S, dtype=torch.int32, device="cuda") for _ in range(2))
    pos, slots = (torch.zeros(200, dtype=torch.int32, device="cuda") for _ in range(2))
    qsl, short = torch.zeros(S + 1, dtype=torch.int32, device="cuda"), i32([0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ti.reserve_pages_(BE, pool, counts, pos, slots, qsl, short)
        ti.release_pages_(BE, pool, keep)
    g = np.random.Generator(np.random.PCG64(1))
    for _ in range(6):
        c = [int(x) for x in g.integers(0, 20, S)]
        k = [int(x) for x in g.integers(0, 200, S)]
        counts.copy_(i32(c))
        keep.copy_(i32(k))
        graph.replay()
        torch.cuda.synchronize()
        want = host.reserve(c, 200)
        host.release(k)
        assert (pos.tolist(), slots.tolist(), qsl.tolist(), int(short)) == want
        same(pool, host)
