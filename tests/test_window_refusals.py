"""What window attention, 8-bit block caches and the page bookkeeping refuse, before any HIP call (no GPU)."""
import ctypes

import pytest
import torch

import tileinfer_hip as ti
from tileinfer_hip import _lib
from tileinfer_hip._lib import AttentionArgs, KVCache, PagePoolArgs

OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 3
BE = ti.HipBackend()


def cache(kind=_lib.TI_KV_FP8, D=128, P=16, H=2, pages=10, **kw):
    c = KVCache()
    c.kind, c.head_dim, c.page_size, c.kv_heads, c.num_pages = kind, D, P, H, pages
    c.k_pages = c.v_pages = c.layer_q = c.layer_scale = c.smooth = 16
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def args(**kw):
    a = AttentionArgs()
    a.dtype, a.q_heads, a.num_seqs, a.max_query_len, a.total_tokens, a.block_table_stride = _lib.TI_BF16, 8, 2, 1, 2, 4
    a.q = a.out = a.positions = a.block_tables = 16
    a.scale, a.causal = 1.0, 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def window_bytes(a, c, window=64, sinks=4):
    size = ctypes.c_size_t(77)
    st = _lib.load().ti_window_attention_workspace_bytes(ctypes.byref(a), window, sinks, ctypes.byref(c), ctypes.byref(size))
    return st, size.value


def test_window_arguments():
    for kind in (0, 1, 2):
        c = cache(kind)
        assert window_bytes(args(), c)[0] == OK
        assert window_bytes(args(), c, 2 ** 31 - 1, 2 ** 31 - 1)[0] == OK
        for window, sinks in ((0, 0), (-1, 0), (1, -1)):
            assert window_bytes(args(), c, window, sinks) == (INVALID, 0)
        for bad in (dict(causal=0), dict(q=None), dict(out=None), dict(positions=None), dict(block_tables=None), dict(scale=0.0),
                    dict(scale=float("inf")), dict(num_seqs=0), dict(max_query_len=0), dict(total_tokens=3), dict(q_heads=7),
                    dict(block_table_stride=0), dict(dtype=5)):
            assert window_bytes(args(**bad), c)[0] == INVALID, bad
        assert window_bytes(args(path=_lib.TI_PATH_DECODE), c)[0] == UNSUPPORTED
        assert window_bytes(args(num_seqs=65536, total_tokens=65536), c)[0] == UNSUPPORTED
        assert window_bytes(args(), cache(kind, D=96))[0] == UNSUPPORTED
    L = _lib.load()
    assert L.ti_window_attention_workspace_bytes(ctypes.byref(args()), 1, 0, ctypes.byref(cache()), None) == INVALID
    assert L.ti_window_attention_workspace_bytes(None, 1, 0, ctypes.byref(cache()), ctypes.byref(ctypes.c_size_t())) == INVALID
    # a workspace that is missing, short or not aligned
    a, c = args(num_seqs=1, total_tokens=1), cache(_lib.TI_KV_DENSE)
    need = window_bytes(a, c, 8192, 0)[1]
    assert need > 0
    assert L.ti_window_attention(ctypes.byref(a), 8192, 0, ctypes.byref(c), None) == WORKSPACE
    a.workspace, a.workspace_bytes = 4096, need - 1
    assert L.ti_window_attention(ctypes.byref(a), 8192, 0, ctypes.byref(c), None) == WORKSPACE
    a.workspace, a.workspace_bytes = 4097, need
    assert L.ti_window_attention(ctypes.byref(a), 8192, 0, ctypes.byref(c), None) == INVALID


def test_fp8_caches():
    L, size = _lib.load(), ctypes.c_size_t()
    for c, st in ((cache(), OK), (cache(P=1024), OK), (cache(P=8), UNSUPPORTED), (cache(P=24), UNSUPPORTED), (cache(P=2048), UNSUPPORTED),
                  (cache(D=96), UNSUPPORTED), (cache(layer_q=None), INVALID), (cache(layer_scale=None), INVALID), (cache(layer_q=24), INVALID),
                  (cache(smooth=None), OK)):
        assert L.ti_attention_workspace_bytes(ctypes.byref(args()), ctypes.byref(c), ctypes.byref(size)) == st
        assert window_bytes(args(), c)[0] == st
        assert L.ti_store_kv(_lib.TI_BF16, ctypes.byref(c), None, None, None, 1, None) == (st or INVALID)
        assert L.ti_store_kv(_lib.TI_BF16, ctypes.byref(c), None, None, None, 0, None) == st
        assert L.ti_attention_inputs(_lib.TI_BF16, None, ctypes.byref(c), None, None, None, None, 5, None, None, 0, 4, 1e-6, None) == st
    # not for page bounds and sparse attention
    kb = _lib.KeyBoundsArgs(16, 16, None)
    assert L.ti_update_key_bounds(_lib.TI_BF16, ctypes.byref(cache()), ctypes.byref(kb), 16, 4, 16, None, 1, 1, 1, None) == UNSUPPORTED
    s = _lib.SparseAttentionArgs()
    s.dtype, s.q_heads, s.total_tokens, s.table_width, s.num_seqs, s.max_query_len = _lib.TI_BF16, 8, 1, 4, 1, 1
    s.q = s.out = s.tables = s.lengths = 16
    s.scale = 1.0
    assert L.ti_sparse_attention_workspace_bytes(ctypes.byref(s), ctypes.byref(cache()), ctypes.byref(size)) == UNSUPPORTED
    assert L.ti_attention_workspace_bytes(ctypes.byref(args()), ctypes.byref(cache(kind=3)), ctypes.byref(size)) == INVALID
    assert L.ti_attention_workspace_bytes(ctypes.byref(args(path=9)), ctypes.byref(cache()), ctypes.byref(size)) == INVALID


def pool(**kw):
    p = PagePoolArgs(100, 16, 4, 20, 0, 0, 16, 16, 16, 16, None, 16)
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_pools():
    L = _lib.load()

    def reserve(p, counts=None, tokens=5, positions=16, slots=16, qsl=16, short=16):
        return L.ti_reserve_pages(ctypes.byref(p), counts, tokens, positions, slots, qsl, short, None)

    for p, st in ((pool(), INVALID), (pool(num_pages=0), INVALID), (pool(page_size=0), INVALID), (pool(num_seqs=0), INVALID), (pool(table_width=0), INVALID),
                  (pool(window=-1), INVALID), (pool(sinks=-1), INVALID), (pool(window=5), INVALID), (pool(free=None), INVALID),
                  (pool(ticket=None), INVALID), (pool(num_seqs=4097), UNSUPPORTED), (pool(num_pages=2 ** 30, page_size=2), UNSUPPORTED)):
        assert reserve(p) == st                                # counts are missing at the least
        assert L.ti_release_pages(ctypes.byref(p), None, None) == st
    for bad in (dict(tokens=-1), dict(positions=None), dict(slots=None), dict(qsl=None), dict(short=None)):
        assert reserve(pool(), 16, **bad) == INVALID
    assert L.ti_reserve_pages(None, 16, 5, 16, 16, 16, 16, None) == INVALID


def test_python_refusals():
    q = torch.zeros((2, 8, 128), dtype=torch.bfloat16)
    k, v = ti.fp8_kv_pools(128, 16, 2, 10, device="cpu")
    assert k.shape == (10, 2, 16, 128) and k.q.dtype == torch.float8_e4m3fn and k.scale.shape == (10, 2)
    with pytest.raises(ti.ArgumentError):
        ti.fp8_layer_arrays(v, k)
    with pytest.raises(ti.ArgumentError):
        ti.fp8_layer_arrays(k, ti.fp8_kv_pools(128, 16, 2, 10, device="cpu")[1])
    with pytest.raises(ti.ArgumentError):
        ti.Fp8Pages(k.layer_q.float(), k.layer_scale, 0)
    with pytest.raises(ti.ArgumentError):
        ti.Fp8Pages(k.layer_q, k.layer_scale[:, :5], 0)
    bt, pos = torch.zeros((1, 4), dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ti.ArgumentError, match="GPU"):
        ti.window_attention_(BE, q, None, q, k, v, bt, pos, 1.0, 5)
    with pytest.raises(ti.ArgumentError, match="GPU"):
        ti.store_kv_(BE, k, v, q, q, pos)
    for window, sinks in ((0, 0), (5, -1), (2 ** 31, 0), (1.5, 0), (True, 0)):
        with pytest.raises(ti.ArgumentError):
            ti.window_attention_workspace(BE, q, k, window, sinks)
    p = ti.page_pool(10, 16, 3, 5, device="cpu")
    assert p.free.tolist() == list(range(10, 0, -1)) and p.behind is None
    assert ti.page_pool(10, 16, 3, 5, 7, 17, device="cpu").behind.tolist() == [2, 2, 2]
    with pytest.raises(ti.ArgumentError, match="GPU"):
        ti.release_pages_(BE, p, torch.zeros(3, dtype=torch.int32))
    with pytest.raises(ti.ArgumentError):
        ti.PagePool(p.free, p.free_count, p.tables.long(), p.lengths, 16)
    with pytest.raises(ti.ArgumentError):
        ti.PagePool(p.free, p.free_count, p.tables, p.lengths, 0)
    with pytest.raises(ti.ArgumentError):
        ti.PagedKVCache(1, 128, 2, 4, quantize="fp8", bounds=True, device="cpu")
    assert ti.PagedKVCache(2, 128, 2, 4, quantize="fp8", device="cpu").v[1].half == 1
    assert ti.bytes_per_token(2, 8, 128, quantize="fp8") == 2 * 2 * 8 * 128
    for op in ("window_attention", "window_attention!", "reserve_pages!", "release_pages!"):
        assert ti.has_kernel(BE, op)
