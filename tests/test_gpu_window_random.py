"""Windowed steps of random shapes over caches of every kind, against 64 bits; garbage (finite or NaN) in every row that no
query sees."""
import numpy as np
import pytest
import torch

import tileinfer_hip as ti
from window_forms import want
from window_ref import Step, check

pytestmark = pytest.mark.gpu
BE = ti.HipBackend()


def shape(seed):
    g = np.random.Generator(np.random.PCG64(1000 + seed))

    def spread(lo, hi):
        return int(np.exp(g.uniform(np.log(lo), np.log(hi + 1))))

    kv = ("bf16", "fp32", "int8", "fp8")[seed % 4]
    D = int(g.choice([64, 128]))
    H, G = int(g.choice([1, 2, 3, 4, 8])), int(g.choice([1, 2, 3, 4, 5, 7, 8, 16, 32]))
    P = int(g.choice([16, 32, 64, 128] if kv == "fp8" or g.random() < 0.7 else [1, 4, 8, 12, 24, 48]))
    most = spread(1, 1500 if kv != "fp32" else 300)
    seqs = max(1, min(spread(1, 24), 6000 // most, 40000 // (most * H * G) + 1))
    lens = [(int(g.choice([0, spread(1, 3000), spread(1, 300)])), int(g.choice([most, g.integers(0, most + 1)]))) for _ in range(seqs)]
    window = spread(1, 3000)
    sinks = int(g.choice([0, 4, spread(1, 300)]))
    dtype = torch.float32 if kv in ("int8", "fp8") and g.random() < 0.15 else None
    return dict(kv=kv, lens=lens, window=window, sinks=sinks, D=D, H=H, G=G, P=P, seed=seed, dtype=dtype), g.random() < 0.5


@pytest.mark.parametrize("seed", range(48))
def test_random_shapes(gpu, seed):
    kw, finite = shape(seed)
    print(kw, finite, flush=True)
    s = Step(**kw)
    if s.tokens == 0:
        return
    expected = want(s)
    if finite:
        for half, x in ((0, s.layer.k), (1, s.layer.v)):
            x[np.isnan(x)] = 3e4
            if s.layer.kv == "fp8":
                s.layer.q[half][s.layer.q[half] == 127] = 126
        if s.layer.kv in ("int8", "fp8"):
            s.layer.scale[np.isnan(s.layer.scale)] = 2.0 ** 10
    k, v = s.layer.device()
    tables, positions, starts = s.args()
    q = s.q.cuda()
    out = torch.full_like(q, 7.0)
    ws = ti.window_attention_workspace(BE, q, k, s.window, s.sinks, len(s.lens), s.most)
    ti.window_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, s.window, s.sinks, starts, s.most)
    check(out, *expected, s.T)
