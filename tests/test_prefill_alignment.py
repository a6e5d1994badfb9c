"""Prefill steps whose queries or pools are aligned to their elements only: the kernels whose tiles come by direct loads of 16 bytes
(pools of dense caches, queries of the 16-row kernel for every cache) are not picked for them."""
import ctypes

import pytest
import torch

import tileinfer_hip as ti
from tileinfer_hip import _lib
from window_ref import Step, check

BE = ti.HipBackend()


class Plan(ctypes.Structure):
    """ti_prefill_plan."""
    _fields_ = [(n, ctypes.c_int) for n in "pp dl pair r16 wpg ng splits TQ qtiles rows".split()] + [("bytes", ctypes.c_size_t)]


class Window(ctypes.Structure):
    _fields_ = [("size", ctypes.c_int), ("sinks", ctypes.c_int)]


def plan(kind, q, pools, path=_lib.TI_PATH_AUTO, window=0, n=512):
    f = getattr(ti.load_library(), "_Z15ti_plan_prefillPK17ti_attention_argsPK11ti_kv_cacheb9ti_window")
    f.restype, f.argtypes = Plan, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_bool, Window]
    c = _lib.KVCache()
    c.kind, c.head_dim, c.page_size, c.kv_heads, c.num_pages = kind, 128, 16, 8, 1000
    c.k_pages = c.v_pages = pools
    c.layer_q = c.layer_scale = c.smooth = 4096
    a = _lib.AttentionArgs()
    a.dtype, a.q_heads, a.num_seqs, a.max_query_len, a.total_tokens, a.block_table_stride = _lib.TI_BF16, 32, 1, n, n, 40
    a.q, a.out, a.positions, a.block_tables, a.scale, a.causal, a.path = q, 4096, 4096, 4096, 1.0, 1, path
    return f(ctypes.byref(a), ctypes.byref(c), True, Window(window, 0))


@pytest.mark.parametrize("kind", [_lib.TI_KV_DENSE, _lib.TI_KV_INT8, _lib.TI_KV_FP8])
@pytest.mark.parametrize("path", [_lib.TI_PATH_AUTO, _lib.TI_PATH_PREFILL_PAIRED16])
def test_picks(kind, path):
    assert plan(kind, 4096, 4096, path).r16 == 1
    for q in (4098, 4104):
        assert plan(kind, q, 4096, path).r16 == 0
    if kind == _lib.TI_KV_DENSE:
        for p in (path, _lib.TI_PATH_PREFILL_DIRECT, _lib.TI_PATH_PREFILL_PAIRED):
            assert plan(kind, 4096, 4096, p).dl == 1
            for pools in (4098, 4104):
                got = plan(kind, 4096, pools, p)
                assert (got.dl, got.pair, got.r16) == (0, 0, 0)
        assert plan(kind, 4096, 4096, window=64).dl == 1 and plan(kind, 4096, 4098, window=64).dl == 0


def shifted(t):
    room = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
    room[1:].copy_(t.reshape(-1))
    return room[1:].view(t.shape)


LENS = [[(300, 1)], [(100, 6), (40, 2)], [(0, 512)], [(100, 300), (0, 40), (30, 0)], [(100, 900)]]


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "int8", "fp8"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", LENS)
@pytest.mark.parametrize("window", [0, 1 << 20])
def test_outputs(gpu, kv, D, lens, window):
    """Without a window, and with one that reaches over all that the tables hold."""
    s = Step(kv, lens, window, 0, D=D, H=4, seed=D)
    k, v = s.layer.device()
    if kv == "bf16":
        k, v = shifted(k), shifted(v)
    tables, positions, starts = (shifted(t) for t in s.args())
    q = shifted(s.q.cuda())
    out = shifted(torch.zeros_like(q))
    if window:
        ws = ti.window_attention_workspace(BE, q, k, window, 0, len(lens), s.most)
        ti.window_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, window, 0, starts, s.most)
    else:
        ws = ti.attention_workspace(BE, q, k, len(lens), s.most)
        ti.paged_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, True, starts, s.most)
    check(out, *s.want(), s.T)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["bf16", "fp8"])
@pytest.mark.parametrize("path", range(2, 8))
def test_pinned_paths(gpu, kv, path):
    s = Step(kv, [(100, 300), (0, 40)], H=4, seed=path)
    k, v = s.layer.device()
    if kv == "bf16":
        k, v = shifted(k), shifted(v)
    tables, positions, starts = s.args()
    q = shifted(s.q.cuda())
    out = torch.zeros_like(q)
    ws = ti.attention_workspace(BE, q, k, 2, s.most, path)
    ti.paged_attention_(BE, out, ws, q, k, v, tables, positions, s.scale, True, starts, s.most, path)
    check(out, *s.want(), s.T)
