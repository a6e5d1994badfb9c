"""Float32 queries over INT8 and 8-bit block caches with a window (the vector kernel that counts each query's own keys through),
and the ping-pong forms over 8-bit block caches without one, against 64 bits."""
import numpy as np
import pytest
import torch

import tileinfer_hip as ti
from window_forms import KSPLIT, SHARED, SOLO, pick, want
from window_ref import Step, check

BE = ti.HipBackend()
LENS = [[(300, 1)], [(0, 1)], [(777, 1), (0, 1), (64, 1), (1, 1)], [(200, 5), (3, 2), (40, 0), (129, 7)], [(0, 150)], [(700, 33), (10, 0), (64, 64)]]


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["int8", "fp8"])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("window,sinks", [(64, 4), (1, 0), (17, 33), (4096, 5), (2 ** 31 - 1, 0)])
@pytest.mark.parametrize("D,H,G,P", [(128, 2, 4, 16), (64, 3, 1, 64)])
def test_float32_queries(gpu, kv, lens, window, sinks, D, H, G, P):
    s = Step(kv, lens, window, sinks, D=D, H=H, G=G, P=P, seed=window % 100, dtype=torch.float32)
    k, v = s.layer.device()
    tables, positions, starts = s.args()
    q = s.q.cuda()
    out = torch.full_like(q, 7.0)
    ws = ti.window_attention_workspace(BE, q, k, window, sinks, len(lens), s.most)
    ti.window_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, window, sinks, starts, s.most)
    check(out, *s.want(), s.T)


@pytest.mark.gpu
@pytest.mark.parametrize("P", [1, 5, 24])
def test_float32_queries_odd_pages(gpu, P):
    s = Step("int8", [(250, 1), (40, 60)], 70, 3, P=P, seed=P, dtype=torch.float32)
    k, v = s.layer.device()
    tables, positions, starts = s.args()
    out = ti.window_attention(BE, s.q.cuda(), k, v, tables, positions, s.scale, 70, 3, starts, s.most)
    check(out, *s.want(), s.T)


FP8 = [(SHARED, 128, [(3000, 1500)], 8, 4, 64), (SHARED, 128, [(0, 700), (1000, 690), (90, 650)], 8, 4, 16), (KSPLIT, 128, [(1000, 1500)], 8, 4, 16),
       (KSPLIT, 64, [(333, 900)], 8, 4, 64), (SOLO, 128, [(300, 150), (0, 20), (90, 130)] * 6, 8, 4, 16), (SOLO, 64, [(500, 700)] * 3, 8, 4, 16)]


@pytest.mark.parametrize("form,D,lens,H,G,P", FP8)
def test_cases_reach_their_forms(form, D, lens, H, G, P):
    assert pick("fp8", lens, 0, 0, D, H, G, P) == form


@pytest.mark.gpu
@pytest.mark.parametrize("garbage", ["finite", "nan"])
@pytest.mark.parametrize("form,D,lens,H,G,P", FP8)
def test_forms_over_8_bit_blocks(gpu, form, D, lens, H, G, P, garbage):
    s = Step("fp8", lens, D=D, H=H, G=G, P=P, seed=len(lens))
    expected = want(s)
    if garbage == "finite":
        s.layer.q[s.layer.q == 127] = 126
        s.layer.scale[np.isnan(s.layer.scale)] = 2.0 ** 10
    k, v = s.layer.device()
    tables, positions, starts = s.args()
    q = s.q.cuda()
    out = torch.full_like(q, 7.0)
    ti.paged_attention_(BE, out, ti.attention_workspace(BE, q, k, len(lens), s.most), q, k, v, tables, positions, s.scale, True, starts, s.most)
    check(out, *expected, s.T)
