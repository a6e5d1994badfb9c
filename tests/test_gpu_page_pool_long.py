"""reserve_pages_ over the longest token arrays that a call takes, 2^31 - 1: a step of their length and one of a few tokens."""
import pytest
import torch

import tileinfer_hip as ti
from window_ref import i32

pytestmark = pytest.mark.gpu
BE = ti.HipBackend()


def test_longest_token_arrays(gpu):
    T, P, pages = 2 ** 31 - 1, 1 << 20, 2047
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("two arrays of 8.6 GB")
    room = torch.empty((2, T + 1), dtype=torch.int32, device="cuda")
    for shift in (0, 1):                                     # arrays aligned to 16 bytes, and to their elements only
        pos, slots = (room[i, shift:shift + T] for i in (0, 1))
        for counts in ([pages * P, 0], [7, 1000], [5, 2 ** 31 - 6 - (pages - 1) * P]):
            room.fill_(9)
            pool = ti.page_pool(pages, P, 2, pages)
            qsl, short = torch.zeros(3, dtype=torch.int32, device="cuda"), i32([9])
            ti.reserve_pages_(BE, pool, i32(counts), pos, slots, qsl, short)
            n = sum(counts)
            assert int(short) == 0 and qsl.tolist() == [0, counts[0], n]
            for lo in range(0, T, 1 << 28):
                hi = min(lo + (1 << 28), T)
                t = torch.arange(lo, hi, dtype=torch.int64, device="cuda")
                first = t < counts[0]
                want = torch.where(first, t, t - counts[0])
                held = -(-counts[0] // P)                    # pages are handed out in increasing order
                slot = want + 1 + torch.where(first, 0, held * P)
                real = t < n
                assert torch.equal(pos[lo:hi].long(), torch.where(real, want, 0))
                assert torch.equal(slots[lo:hi].long(), torch.where(real, slot, 0))
            ends = room[:, T if shift == 0 else 0]
            assert ends.tolist() == [9, 9]
            ti.release_pages_(BE, pool, i32([0, 0]))
            assert int(pool.free_count) == pages and pool.free.tolist() == list(range(pages, 0, -1))
    del room, pos, slots
    torch.cuda.empty_cache()
