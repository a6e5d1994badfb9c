"""PagePool over tables and lengths that a program has already: pages that went back behind the window before are not
given back again, with `behind` from the tables or from the program."""
import numpy as np
import pytest
import torch

import tileinfer_hip as ti
from window_ref import i32

BE = ti.HipBackend()


def i32_cpu(x):
    return torch.tensor(x, dtype=torch.int32)


def host_pool(tables, lengths, P, window, sinks, **kw):
    held = [p for row in tables for p in row if p]
    free = [p for p in range(60, 0, -1) if p not in held]
    return ti.PagePool(i32_cpu(free + [0] * (60 - len(free))), i32_cpu([len(free)]), i32_cpu(tables), i32_cpu(lengths), P, window, sinks, **kw)


@pytest.mark.parametrize("sinks,first", [(0, 0), (4, 1), (16, 1), (17, 2)])
def test_behind_from_the_tables(sinks, first):
    P, window, W = 16, 40, 8
    kept = [list(range(1 + 8 * b, 1 + 8 * b + first)) for b in range(5)]

    def row(b, gone, held):
        """Sinks, pages [first, gone) given back, pages [gone, held) held."""
        return kept[b] + [0] * (gone - first) + [40 + b + i for i in range(held - gone)] + [0] * (W - max(held, gone))

    tables = [row(0, first, first), row(1, first, first + 2), row(2, 4, 6), row(3, 7, 8), [0] * W]
    # the last: an empty sequence, which holds no sinks either
    pool = host_pool(tables, [first * P, (first + 2) * P, 6 * P - 3, 8 * P, 0], P, window, sinks)
    assert pool.behind.dtype == torch.int32 and pool.behind.tolist() == [first, first, 4, 7, first]


def test_everything_in_front_of_the_window_is_back():
    """A window of one position, a length that is whole pages: nothing is held behind the sinks."""
    pool = host_pool([[1, 0, 0, 0, 0], [2, 0, 0, 9, 0]], [64, 50], 16, 1, 4)
    assert pool.behind.tolist() == [4, 3]


def test_sinks_past_the_tables():
    assert host_pool([[1, 2, 0], [0, 0, 0]], [20, 0], 16, 5, 1000).behind.tolist() == [63, 63]


def test_behind_of_the_program():
    tables, lengths = [[1, 0, 0, 4, 0]], [60]
    assert host_pool(tables, lengths, 16, 5, 4, behind=i32_cpu([3])).behind.tolist() == [3]
    for bad in (i32_cpu([3, 3]), torch.tensor([3]), torch.tensor([3.0])):
        with pytest.raises(ti.ArgumentError):
            host_pool(tables, lengths, 16, 5, 4, behind=bad)
    with pytest.raises(ti.ArgumentError):
        host_pool(tables, lengths, 16, 0, 0, behind=i32_cpu([0]))      # no window: nothing is behind it
    assert host_pool(tables, lengths, 16, 0, 0).behind is None


@pytest.mark.gpu
@pytest.mark.parametrize("P,window,sinks", [(16, 40, 4), (16, 1, 0), (5, 33, 11), (64, 100, 0)])
@pytest.mark.parametrize("given", [False, True])
def test_taken_over(gpu, P, window, sinks, given):
    """A pool made anew of another's arrays in the middle of its work goes on as the other does, and no page is lost,
    held twice, or none."""
    S, W, pages = 6, 30, 200
    g = np.random.Generator(np.random.PCG64(P + window))
    a = ti.page_pool(pages, P, S, W, window, sinks)
    b = None
    lengths = np.zeros(S, np.int64)
    for r in range(12):
        counts = g.integers(0, [3 * P, 2][r % 2] + 1, S)
        counts = np.minimum(counts, W * P - lengths)
        T = int(counts.sum())
        keep = lengths + counts
        if r == 8:
            keep[1] = 0                                                 # a finished chat
        states = []
        for pool in (a, b):
            if pool is None:
                continue
            pos, slots = (torch.zeros(max(T, 1), dtype=torch.int32, device="cuda") for _ in range(2))
            qsl, short = torch.zeros(S + 1, dtype=torch.int32, device="cuda"), i32([9])
            ti.reserve_pages_(BE, pool, i32(counts), pos, slots, qsl, short)
            assert int(short) == 0 and bool((slots[:T] > 0).all())
            ti.release_pages_(BE, pool, i32(keep))
            n = int(pool.free_count)
            ids = torch.cat([pool.tables[pool.tables > 0], pool.free[:n]])
            assert ids.sort().values.tolist() == list(range(1, pages + 1))
            states.append([pos.tolist(), slots.tolist(), pool.tables.tolist(), pool.lengths.tolist(), pool.free[:n].tolist(),
                           pool.behind.tolist()])
        assert all(s == states[0] for s in states)
        lengths = keep
        if r in (3, 8):
            b = ti.PagePool(*(t.clone() for t in (a.free, a.free_count, a.tables, a.lengths)), P, window, sinks,
                            **(dict(behind=a.behind.clone()) if given else {}))


@pytest.mark.parametrize("what", [dict(window=2 ** 32 + 40), dict(window=2 ** 31), dict(window=40, sinks=2 ** 32), dict(sinks=2 ** 31),
                                  dict(page_size=2 ** 32 + 16), dict(window=39.5), dict(window=40, sinks=0.5), dict(page_size=16.5),
                                  dict(window=True), dict(window=-1), dict(sinks=-1), dict(page_size=0)])
def test_numbers_that_the_library_does_not_hold(what):
    """A window of 2^32 + 40 would be one of 40 in 32 bits, and pages that later queries see would go back."""
    with pytest.raises(ti.ArgumentError):
        ti.page_pool(10, **dict(dict(page_size=16, num_seqs=2, max_pages=4, device="cpu"), **what))


def test_whole_numbers_of_other_types():
    p = ti.page_pool(10, np.int64(16), 2, 4, np.int32(40), 4.0, device="cpu")
    assert (p.page_size, p.window, p.sinks) == (16, 40, 4) and all(type(x) is int for x in (p.page_size, p.window, p.sinks))
    assert ti.page_pool(10, 16, 2, 4, 2 ** 31 - 1, 2 ** 31 - 1, device="cpu").window == 2 ** 31 - 1
