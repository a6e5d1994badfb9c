"""Windows at the end of the longest block tables, 2^30 positions: the outputs of the same step near the tables' front."""
import numpy as np
import pytest
import torch

import tileinfer_hip as ti
from window_forms import want
from window_ref import Step, check, i32

pytestmark = pytest.mark.gpu
BE = ti.HipBackend()


@pytest.mark.parametrize("P", [16, 1024])
@pytest.mark.parametrize("kv", ["bf16", "fp32", "int8", "fp8"])
@pytest.mark.parametrize("lens,H", [([(4000, 1)], 2), ([(4000, 5), (3333, 3)], 2), ([(4000, 90)], 2), ([(3500, 1100)], 8), ([(3500, 600), (4000, 690)], 8)])
def test_far_positions(gpu, kv, lens, H, P):
    window = 1500
    s = Step(kv, lens, window, 0, H=H, G=4, P=P, seed=P)
    expected = want(s)
    width = (1 << 30) // P
    shift = width - s.tables.shape[1]                        # pages; the longest sequence ends in the table's last
    if P == 16:
        shift -= shift % 2                                   # tiles of 32 keys as before
    k, v = s.layer.device()
    tables = torch.zeros((len(lens), width), dtype=torch.int32, device="cuda")
    tables[:, shift:shift + s.tables.shape[1]] = torch.from_numpy(s.tables).cuda()
    positions, starts = i32(s.positions.astype(np.int64) + shift * P), i32(s.starts)
    out = ti.window_attention(BE, s.q.cuda(), k, v, tables, positions, s.scale, window, 0, starts, s.most)
    check(out, *expected, s.T)


@pytest.mark.parametrize("n", [1, 40])
def test_far_sinks(gpu, n):
    """The first keys and the last ones of a chat of 2^30."""
    P, window, sinks, D, G = 1024, 700, 1100, 128, 4
    width = (1 << 30) // P
    g = torch.Generator(device="cuda").manual_seed(n)
    k, v = (torch.randn((4, 1, P, D), generator=g, device="cuda").bfloat16() for _ in range(2))
    q = torch.randn((n, G, D), generator=g, device="cuda").bfloat16()
    tables = torch.zeros((1, width), dtype=torch.int32, device="cuda")
    tables[0, :2], tables[0, -2:] = i32([3, 1]), i32([4, 2])
    pos = torch.arange((1 << 30) - n, 1 << 30, dtype=torch.int32, device="cuda")
    out = ti.window_attention(BE, q, k, v, tables, pos, D ** -0.5, window, sinks)
    kd, vd = (x.double()[[2, 0, 3, 1]].reshape(4 * P, D) for x in (k, v))
    at = torch.cat([torch.arange(2 * P, device="cuda"), torch.arange((1 << 30) - 2 * P, 1 << 30, device="cuda")])
    sees = (at <= pos[:, None]) & ((at > pos[:, None] - window) | (at < sinks))
    x = (q.double().reshape(n * G, D) @ kd.T.contiguous() * D ** -0.5).masked_fill(~sees.repeat_interleave(G, 0), -torch.inf)
    w = torch.softmax(x, 1)
    check(out, (w @ vd).view(n, G, D).cpu().numpy(), (w @ vd.abs()).view(n, G, D).cpu().numpy(), torch.bfloat16)
