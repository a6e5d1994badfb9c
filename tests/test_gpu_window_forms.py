"""The windowed forms of the ping-pong prefill kernel (prompts and chunks of many tokens) with keys that the window hides: every
form of every cache kind, against 64 bits, with finite and with NaN garbage in the rows that no query sees, and with rows
that are not finite and that only some queries see."""
import math

import numpy as np
import pytest
import torch

import tileinfer_hip as ti
from window_forms import FORMS, KSPLIT, SHARED, SOLO, pick, want
from window_ref import Step, check, tolerance

BE = ti.HipBackend()


@pytest.mark.parametrize("form,kv,D,lens,H,G,P,window,sinks", FORMS)
def test_cases_reach_their_forms(form, kv, D, lens, H, G, P, window, sinks):
    assert pick(kv, lens, window, sinks, D, H, G, P) == form
    # keys are hidden from some query of each of the longer sequences, between the sinks and its window
    assert all(c + n - window > sinks for c, n in lens if c + n > 300 + window) and max(c + n for c, n in lens) > window + sinks


def test_every_form_is_reached():
    assert {(f[0], f[1], f[2]) for f in FORMS} == {
        (SHARED, "bf16", 128), (KSPLIT, "bf16", 128), (SOLO, "bf16", 128), (KSPLIT, "bf16", 64), (SOLO, "bf16", 64), (KSPLIT, "int8", 128),
        (KSPLIT, "int8", 64), (SOLO, "int8", 128), (SOLO, "int8", 64), (SHARED, "fp8", 128), (KSPLIT, "fp8", 128), (SOLO, "fp8", 128),
        (KSPLIT, "fp8", 64), (SOLO, "fp8", 64)}


def finite_garbage(s):
    """Large finite values in the rows that no query sees."""
    for half, x in ((0, s.layer.k), (1, s.layer.v)):
        x[np.isnan(x)] = 3e4
        if s.layer.kv == "fp8":
            s.layer.q[half][s.layer.q[half] == 127] = 126
    if s.layer.kv != "bf16":
        s.layer.scale[np.isnan(s.layer.scale)] = 2.0 ** 10


def run(s):
    k, v = s.layer.device()
    tables, positions, starts = s.args()
    q = s.q.cuda()
    out = torch.full_like(q, 7.0)
    ws = ti.window_attention_workspace(BE, q, k, s.window, s.sinks, len(s.lens), s.most)
    return ti.window_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, s.window, s.sinks, starts, s.most)


@pytest.mark.gpu
@pytest.mark.parametrize("garbage", ["finite", "nan"])
@pytest.mark.parametrize("form,kv,D,lens,H,G,P,window,sinks", FORMS)
def test_forms(gpu, form, kv, D, lens, H, G, P, window, sinks, garbage):
    s = Step(kv, lens, window, sinks, D=D, H=H, G=G, P=P, seed=len(lens) + window)
    expected = want(s)
    if garbage == "finite":
        finite_garbage(s)
    got = run(s)
    check(got, *expected, s.T)
    assert torch.equal(got, run(s))


@pytest.mark.gpu
@pytest.mark.parametrize("half", [0, 1])
@pytest.mark.parametrize("form,kv,D,lens,H,G,P,window,sinks", [f for f in FORMS if f[1] != "int8" and len(f[3]) < 6])
def test_rows_that_only_some_see(gpu, form, kv, D, lens, H, G, P, window, sinks, half):
    """A NaN reaches the queries that see it, and no other."""
    s = Step(kv, lens, window, sinks, D=D, H=H, G=G, P=P, seed=window)
    expected, size = want(s)
    finite_garbage(s)
    c, n = lens[0]
    at = c + n // 2
    s.layer.put(half, int(s.tables[0][at // P]) - 1, H - 1, at % P, math.nan)
    got = run(s).double().cpu().numpy()
    hit = np.zeros(got.shape[:2], bool)
    hit[at - c:min(at - c + window, n), (H - 1) * G:] = True
    assert np.isnan(got[hit]).all() and np.isfinite(got[~hit]).all()
    assert (np.abs(got - expected)[~hit] <= tolerance(s.T, expected, size)[~hit]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("form,kv,D,lens,H,G,P,window,sinks", [f for f in FORMS if f[6] == 16 and f[5] == 4 and len(f[3]) < 4])
def test_captured_on_another_stream(gpu, form, kv, D, lens, H, G, P, window, sinks):
    """Replays with other queries, eager work between them."""
    s = Step(kv, lens, window, sinks, D=D, H=H, G=G, P=P, seed=3)
    finite_garbage(s)
    k, v = s.layer.device()
    tables, positions, starts = s.args()
    q = s.q.cuda()
    out = torch.zeros_like(q)
    ws = ti.window_attention_workspace(BE, q, k, window, sinks, len(lens), s.most)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ti.window_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, window, sinks, starts, s.most)
    for r in range(3):
        q.normal_()
        out.zero_()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        side.synchronize()
        assert torch.equal(out, ti.window_attention(BE, q, k, v, tables, positions, s.scale, window, sinks, starts, s.most))
