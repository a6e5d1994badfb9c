"""Edges of the chosen-page operators over steps of several tokens: lengths at the ends of their type, tokens
without keys, garbage in whatever a table does not name."""
import math

import pytest
import torch

import tileinfer_hip as ti
from test_gpu_sparse import Cache, T, check_attend, i32, shared

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
