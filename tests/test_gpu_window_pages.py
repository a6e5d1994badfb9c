"""Pages that went back behind a window, and may be anyone's: table entries of pages that hold no visible key are not used,
so what such pages hold neither changes an output nor makes a step slower (a product that is not finite sends the rows of a
work-group through a path of their own, hundreds of times as long)."""
import math
import statistics

import numpy as np
import pytest
import torch

import tileinfer_hip as ti
from window_forms import KSPLIT, NONE, SHARED, SOLO, pick, want
from window_ref import Step, check

pytestmark = pytest.mark.gpu
BE = ti.HipBackend()
# The first key of the first query's window and the end of the sinks lie between pages of 16 keys, in the middle of 32: tiles
# of 32 keys have a half there whose page went back.
CACHED, P, LO, SINKS = 1000, 16, 592, 48


def gpu_ms(f):
    f()
    torch.cuda.synchronize()
    times = []
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        f()
        b.record()
        b.synchronize()
        times.append(a.elapsed_time(b))
    return statistics.median(times)


CASES = [
    ("bf16", 128, [(CACHED, 1500)], 8, SHARED), ("bf16", 128, [(CACHED, 900)], 8, KSPLIT), ("bf16", 128, [(CACHED, 150)] * 16, 8, SOLO),
    ("bf16", 128, [(CACHED, 300)], 2, NONE), ("bf16", 128, [(CACHED, 64), (CACHED, 40)], 2, NONE), ("bf16", 128, [(CACHED, 5)], 2, None),
    ("bf16", 128, [(CACHED, 1)], 2, None), ("bf16", 64, [(CACHED, 900)], 8, KSPLIT), ("bf16", 64, [(CACHED, 700)] * 3, 8, SOLO),
    ("bf16", 64, [(CACHED, 300)], 2, NONE), ("int8", 128, [(CACHED, 700)] * 3, 8, SOLO), ("int8", 64, [(CACHED, 700)] * 3, 8, SOLO),
    ("int8", 128, [(CACHED, 300)], 2, NONE), ("int8", 128, [(CACHED, 1)], 2, None), ("fp8", 128, [(CACHED, 1500)], 8, SHARED),
    ("fp8", 128, [(CACHED, 900)], 8, KSPLIT), ("fp8", 128, [(CACHED, 150)] * 16, 8, SOLO), ("fp8", 64, [(CACHED, 900)], 8, KSPLIT),
    ("fp8", 128, [(CACHED, 300)], 2, NONE), ("fp8", 128, [(CACHED, 1)], 2, None), ("fp32", 128, [(CACHED, 200)], 2, None),
    ("fp32", 128, [(CACHED, 1)], 2, None),
]


@pytest.mark.parametrize("entry", ["none", "first", "last", "beyond"])
@pytest.mark.parametrize("kv,D,lens,H,form", CASES)
def test_pages_of_others(gpu, kv, D, lens, H, form, entry):
    window, lo = CACHED + 1 - LO, LO
    if form is not None:
        assert pick(kv, lens, window, SINKS, D, H, 4, P) == form
    s = Step(kv, lens, window, SINKS, D=D, H=H, G=4, P=P, seed=D, spare=0)
    expected = want(s)
    # the pool's first and last page are another's: NaN all over
    for name, axis in (("k", 0), ("v", 0), ("q", 1), ("scale", 1)):
        x = getattr(s.layer, name, None)
        if x is not None:
            pad = np.full_like(x.take([0], axis), math.nan if x.dtype.kind == "f" else 127)
            setattr(s.layer, name, np.concatenate([pad, x, pad], axis))
    hidden = s.tables == 0
    assert hidden[:, lo // P - 1].all() and hidden[:, SINKS // P].all()
    s.tables[~hidden] += 1
    finite = s.tables.copy()
    finite[hidden] = s.tables[0, 0]
    s.tables[hidden] = {"none": 0, "first": 1, "last": s.layer.k.shape[0], "beyond": 2 ** 31 - 1}[entry]
    k, v = s.layer.device()
    tables, positions, starts = s.args()
    finite = torch.from_numpy(finite).cuda()
    q = s.q.cuda()
    out = torch.empty_like(q)
    ws = ti.window_attention_workspace(BE, q, k, window, SINKS, len(lens), s.most)

    def run(t):
        return ti.window_attention_(BE, out, ws, q, k, v, t, positions, s.scale, window, SINKS, starts, s.most)

    check(run(tables), *expected, s.T)
    usual, took = gpu_ms(lambda: run(finite)), gpu_ms(lambda: run(tables))
    assert took < 3 * usual + 0.05, f"{took:.3f} ms, {usual:.3f} with tables of finite pages"
