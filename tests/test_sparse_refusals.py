"""What the chosen-page and draft-verification entry points refuse, without a GPU: the C ABI's status codes
before any HIP call, and the Python package's argument errors."""
import ctypes

import pytest
import torch

import tileinfer_hip as ti
from tileinfer_hip import _lib

BE = ti.HipBackend()


def cache(**kw):
    c = _lib.KVCache()
    c.kind, c.head_dim, c.page_size, c.kv_heads, c.num_pages = 0, 128, 16, 8, 100
    c.k_pages = c.v_pages = 0x1000
    for k, v in kw.items():
        setattr(c, k, v)
    return c


def bounds_call(c=None, kb=(0x1000, 0x1000), **kw):
    a = dict(dtype=1, bt=0x1000, stride=64, pos=0x1000, qsl=None, seqs=4, n=1, total=4)
    a.update(kw)
    k = None if kb is None else ctypes.byref(_lib.KeyBoundsArgs(*kb))
    return ti.load_library().ti_update_key_bounds(a["dtype"], ctypes.byref(c or cache()), k, a["bt"], a["stride"], a["pos"], a["qsl"],
                                                  a["seqs"], a["n"], a["total"], None)


@pytest.mark.parametrize("kw", [dict(kb=None), dict(kb=(0, 0x1000)), dict(kb=(0x1000, 0)), dict(kb=(0x1008, 0x1000)), dict(bt=None),
                                dict(stride=0), dict(pos=None), dict(seqs=0), dict(n=0), dict(total=0), dict(total=5), dict(dtype=2),
                                dict(c=cache(k_pages=0)), dict(c=cache(page_size=0))])
def test_bounds_invalid(kw):
    assert bounds_call(**kw) == _lib.TI_ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(c=cache(head_dim=96)), dict(seqs=65536, total=65536)])
def test_bounds_unsupported(kw):
    assert bounds_call(**kw) == _lib.TI_ERR_UNSUPPORTED


def select_args(**kw):
    a = _lib.SelectArgs()
    a.dtype, a.q_heads, a.kv_heads, a.head_dim, a.page_size, a.num_pages = 1, 32, 8, 128, 16, 100
    a.num_seqs, a.max_query_len, a.total_tokens, a.block_table_stride = 4, 1, 4, 100
    a.keep, a.sinks, a.window, a.causal = 8, 1, 2, 1
    a.q = a.bounds.bounds = a.bounds.scale = a.positions = a.block_tables = a.tables = a.lengths = 0x1000
    for k, v in kw.items():
        if k in ("bounds", "scale"):
            setattr(a.bounds, k, v)
        else:
            setattr(a, k, v)
    return a


def select_call(a):
    L, size = ti.load_library(), ctypes.c_size_t(7)
    st = L.ti_select_pages_workspace_bytes(ctypes.byref(a), ctypes.byref(size))
    return st, size.value, L.ti_select_pages(ctypes.byref(a), None)


def test_select_workspace():
    st, n, call = select_call(select_args())
    assert st == 0 and n >= 4 * 8 * 100 * 4          # a score per token, KV head and table entry
    assert call == _lib.TI_ERR_WORKSPACE               # none given
    assert select_call(select_args(workspace=0x1000, workspace_bytes=n - 1))[2] == _lib.TI_ERR_WORKSPACE
    assert select_call(select_args(workspace=0x1008, workspace_bytes=n))[2] == _lib.TI_ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(dtype=5), dict(q_heads=30), dict(kv_heads=0), dict(page_size=0), dict(num_pages=0), dict(num_seqs=0),
                                dict(total_tokens=5), dict(block_table_stride=0), dict(keep=0), dict(sinks=-1), dict(window=0),
                                dict(sinks=7, window=2), dict(sinks=2 ** 31 - 1, window=2 ** 31 - 1), dict(causal=2), dict(q=None),
                                dict(bounds=None), dict(scale=None), dict(bounds=0x1004), dict(positions=None), dict(block_tables=None),
                                dict(tables=None), dict(lengths=None)])
def test_select_invalid(kw):
    assert select_call(select_args(**kw)) == (_lib.TI_ERR_INVALID_ARG, 0, _lib.TI_ERR_INVALID_ARG)


@pytest.mark.parametrize("kw", [dict(head_dim=96), dict(q_heads=520), dict(num_seqs=65536, total_tokens=65536),
                                dict(keep=1 << 28)])
def test_select_unsupported(kw):
    assert select_call(select_args(**kw))[0] == _lib.TI_ERR_UNSUPPORTED


def sparse_args(**kw):
    a = _lib.SparseAttentionArgs()
    a.dtype, a.q_heads, a.total_tokens, a.table_width, a.num_seqs, a.max_query_len = 1, 32, 4, 64, 4, 1
    a.q = a.out = a.tables = a.lengths = 0x1000
    a.scale = 0.088
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def sparse_call(a, c=None):
    L, c, size = ti.load_library(), c or cache(), ctypes.c_size_t(7)
    st = L.ti_sparse_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(c), ctypes.byref(size))
    return st, size.value, L.ti_sparse_attention(ctypes.byref(a), ctypes.byref(c), None)


def test_sparse_workspace():
    st, n, call = sparse_call(sparse_args())
    assert st == 0 and n > 0 and call == _lib.TI_ERR_WORKSPACE
    assert sparse_call(sparse_args(workspace=0x1000, workspace_bytes=n - 1))[2] == _lib.TI_ERR_WORKSPACE
    assert sparse_call(sparse_args(workspace=0x1004, workspace_bytes=n))[2] == _lib.TI_ERR_INVALID_ARG
    # 32 tokens of 8 KV heads fill the chip unsplit
    assert sparse_call(sparse_args(num_seqs=32, total_tokens=32))[:2] == (0, 0)


@pytest.mark.parametrize("kw", [dict(dtype=5), dict(q_heads=30), dict(total_tokens=0), dict(table_width=0), dict(num_seqs=0),
                                dict(max_query_len=0), dict(total_tokens=5), dict(q=None), dict(out=None), dict(tables=None),
                                dict(lengths=None), dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf"))])
def test_sparse_invalid(kw):
    assert sparse_call(sparse_args(**kw)) == (_lib.TI_ERR_INVALID_ARG, 0, _lib.TI_ERR_INVALID_ARG)


def test_sparse_unsupported():
    assert sparse_call(sparse_args(), cache(head_dim=96))[0] == _lib.TI_ERR_UNSUPPORTED
    assert sparse_call(sparse_args(q_heads=65 * 8))[0] == _lib.TI_ERR_UNSUPPORTED
    assert sparse_call(sparse_args(table_width=1 << 28))[0] == _lib.TI_ERR_UNSUPPORTED
    assert sparse_call(sparse_args(num_seqs=1 << 16, total_tokens=1 << 16))[0] == _lib.TI_ERR_UNSUPPORTED
    assert sparse_call(sparse_args(num_seqs=1, max_query_len=1 << 23, total_tokens=1 << 23))[0] == _lib.TI_ERR_UNSUPPORTED


def verify_args(**kw):
    a = _lib.VerifyArgs()
    a.dtype, a.num_seqs, a.max_drafts, a.vocab = 0, 4, 3, 1000
    a.draft_tokens = a.target = a.draft = a.uniforms = a.accepted = a.tokens = 0x1000
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def verify_call(a):
    L, size = ti.load_library(), ctypes.c_size_t(7)
    st = L.ti_verify_draft_workspace_bytes(ctypes.byref(a), ctypes.byref(size))
    return st, size.value, L.ti_verify_draft(ctypes.byref(a), None)


def test_verify_workspace():
    st, n, call = verify_call(verify_args())
    assert st == 0 and n > 0 and call == _lib.TI_ERR_WORKSPACE
    assert verify_call(verify_args(workspace=0x1004, workspace_bytes=n))[2] == _lib.TI_ERR_INVALID_ARG


@pytest.mark.parametrize("kw", [dict(dtype=3), dict(num_seqs=0), dict(max_drafts=-1), dict(vocab=0), dict(draft_tokens=None),
                                dict(target=None), dict(uniforms=None), dict(accepted=None), dict(tokens=None)])
def test_verify_invalid(kw):
    assert verify_call(verify_args(**kw)) == (_lib.TI_ERR_INVALID_ARG, 0, _lib.TI_ERR_INVALID_ARG)


def test_verify_unsupported():
    assert verify_call(verify_args(num_seqs=65536))[0] == _lib.TI_ERR_UNSUPPORTED
    assert verify_call(verify_args(vocab=2 ** 31 - 1))[0] == _lib.TI_ERR_UNSUPPORTED


def test_no_size_pointer():
    L = ti.load_library()
    assert L.ti_select_pages_workspace_bytes(ctypes.byref(select_args()), None) == _lib.TI_ERR_INVALID_ARG
    assert L.ti_sparse_attention_workspace_bytes(ctypes.byref(sparse_args()), ctypes.byref(cache()), None) == _lib.TI_ERR_INVALID_ARG
    assert L.ti_verify_draft_workspace_bytes(ctypes.byref(verify_args()), None) == _lib.TI_ERR_INVALID_ARG


# ---- the Python package: tensors that are not on the GPU are refused by every op -----------------

def test_cpu_tensors_are_refused():
    kb = ti.key_bounds(128, 16, 8, 10, device="cpu")
    k = torch.zeros((10, 8, 16, 128), dtype=torch.bfloat16)
    i = torch.zeros(4, dtype=torch.int32)
    q = torch.zeros((1, 32, 128), dtype=torch.bfloat16)
    t, n = torch.zeros((1, 8, 4), dtype=torch.int32), torch.zeros((1, 8), dtype=torch.int32)
    with pytest.raises(ti.ArgumentError):
        ti.update_key_bounds_(BE, kb, k, k, i, i[:1])
    with pytest.raises(ti.ArgumentError):
        ti.select_pages_(BE, t, n, None, q, kb, i, i[:1])
    with pytest.raises(ti.ArgumentError):
        ti.sparse_attention_(BE, q, None, q, k, k, t, n, 0.1)
    p = torch.rand((2, 3, 100))
    with pytest.raises(ti.ArgumentError):
        ti.verify_draft(BE, torch.zeros((2, 2), dtype=torch.int32), p, p[:, :2].contiguous(), torch.rand((2, 3)))


def test_key_bounds_shapes():
    kb = ti.key_bounds(64, 16, 8, 10, device="cpu")
    assert kb.shape == (10, 8, 16, 64) and kb.bounds.dtype == torch.int8 and kb.scale.shape == (10, 8)
    with pytest.raises(ti.ArgumentError):
        ti.KeyBounds(kb.bounds.float(), kb.scale, 16)
    with pytest.raises(ti.ArgumentError):
        ti.KeyBounds(kb.bounds, kb.scale[:5], 16)
    with pytest.raises(ti.ArgumentError):
        ti.KeyBounds(kb.bounds, kb.scale, 0)
    c = ti.PagedKVCache(3, 64, 8, 10, page_size=16, device="cpu", bounds=True)
    assert len(c.bounds) == 3 and c.bounds[0].shape == tuple(c.k[0].shape)
    assert ti.PagedKVCache(1, 64, 8, 10, page_size=16, device="cpu").bounds is None


def test_ops_are_listed():
    for op in ("update_key_bounds!", "select_pages", "sparse_attention!", "verify_draft"):
        assert ti.has_kernel(BE, op)
