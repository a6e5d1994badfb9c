"""Workspaces that a serving loop makes once: the sizes hold for every smaller call, without a GPU."""
import ctypes

import pytest
import torch

import tileinfer_hip as ti
from tileinfer_hip import _lib

BE = ti.HipBackend()
PTR = 0x1000


def attend_size(name, tokens, n, width, heads=32, kv_heads=8, D=128, P=16, dtype=1, int8=False):
    c = _lib.KVCache()
    c.kind, c.head_dim, c.page_size, c.kv_heads, c.num_pages = int(int8), D, P, kv_heads, 4096
    c.k_pages = c.v_pages = c.layer_q = c.layer_scale = c.smooth = PTR
    a = _lib.SparseAttentionArgs()
    a.dtype, a.q_heads, a.total_tokens, a.table_width, a.num_seqs, a.max_query_len = dtype, heads, tokens, width, 1, n
    a.q = a.out = a.tables = a.lengths = a.query_start_loc = PTR
    a.scale = 0.1
    size = ctypes.c_size_t(7)
    assert getattr(ti.load_library(), name)(ctypes.byref(a), ctypes.byref(c), ctypes.byref(size)) == 0
    return size.value


TYPES = [dict(), dict(int8=True), dict(dtype=0), dict(dtype=0, int8=True)]
SHAPES = [dict(), dict(P=64), dict(P=5), dict(heads=8), dict(heads=24), dict(heads=96, kv_heads=4), dict(heads=64, kv_heads=2),
          dict(heads=256, kv_heads=256), dict(heads=600, kv_heads=600), dict(D=64), dict(D=64, heads=16, P=64)]


@pytest.mark.parametrize("types", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_attend_bound_holds_for_smaller_calls(types, shape):
    """For every plan up to its sizes, and it grows with them."""
    kw = {**types, **shape}
    exact = lambda *a: attend_size("ti_sparse_attention_workspace_bytes", *a, **kw)
    bound = lambda *a: attend_size("ti_sparse_attention_workspace_bound", *a, **kw)
    counts = list(range(1, 70)) + [100, 127, 128, 129, 255, 256, 257, 511, 512, 513, 2048, 5000]
    last = {}
    for T in counts:
        for n in (1, 2, 3, 4, 7, 8, 16, 33):
            for width in (1, 2, 7, 8, 31, 33, 64, 130, 300, 700, 1500):
                b = bound(T, n, width)
                assert exact(T, n, width) <= b
                for smaller in ((T, max(1, n // 2), width), (T, n, max(1, width // 2))):
                    assert bound(*smaller) <= b
                assert last.get((n, width), 0) <= b
                last[n, width] = b
    for T, n, width in ((300, 16, 700), (64, 8, 64)):     # against all that is smaller
        b = bound(T, n, width)
        for t in range(1, T + 1, 7):
            for m in range(1, n + 1):
                for w in (1, 3, 8, 30, 64, 100, 256, 300, 512, 513, 700):
                    if w <= width:
                        assert exact(t, m, w) <= b


def test_attend_workspace_is_made_once():
    """The workspace of the largest batch serves the smaller and the drafted ones: as the batch shrinks, its keys
    are split more, so a launch of 32 tokens needs nothing where one of 31 does."""
    k = torch.zeros((64, 8, 16, 128), dtype=torch.bfloat16)
    q, tables = torch.zeros((32, 32, 128), dtype=torch.bfloat16), torch.zeros((32, 8, 64), dtype=torch.int32)
    assert attend_size("ti_sparse_attention_workspace_bytes", 32, 1, 64) == 0
    have = ti.sparse_attention_workspace(BE, q, k, tables)
    for t in range(1, 33):
        assert have.numel() >= attend_size("ti_sparse_attention_workspace_bytes", t, 1, 64)
    have = ti.sparse_attention_workspace(BE, q, k, tables, 4)
    for t in range(1, 33):
        for n in range(1, 5):
            assert have.numel() >= attend_size("ti_sparse_attention_workspace_bytes", t, n, 64)
    assert ti.sparse_attention_workspace(BE, q, k, tables[:, :, :1]) is None      # too short to split


def test_attend_bound_refuses_as_the_call():
    L, size = ti.load_library(), ctypes.c_size_t(7)
    c, a = _lib.KVCache(), _lib.SparseAttentionArgs()
    assert L.ti_sparse_attention_workspace_bound(ctypes.byref(a), ctypes.byref(c), ctypes.byref(size)) == _lib.TI_ERR_INVALID_ARG
    assert size.value == 0
    assert L.ti_sparse_attention_workspace_bound(ctypes.byref(a), ctypes.byref(c), None) == _lib.TI_ERR_INVALID_ARG


def select_size(tokens, stride, seqs=1, n=None, heads=32, kv_heads=8):
    a = _lib.SelectArgs()
    a.dtype, a.q_heads, a.kv_heads, a.head_dim, a.page_size, a.num_pages = 1, heads, kv_heads, 128, 16, 4096
    a.num_seqs, a.max_query_len, a.total_tokens, a.block_table_stride = seqs, tokens if n is None else n, tokens, stride
    a.keep, a.sinks, a.window, a.causal = 8, 1, 2, 1
    a.q = a.bounds.bounds = a.bounds.scale = a.positions = a.block_tables = a.tables = a.lengths = a.query_start_loc = PTR
    size = ctypes.c_size_t(7)
    assert ti.load_library().ti_select_pages_workspace_bytes(ctypes.byref(a), ctypes.byref(size)) == 0
    return size.value


@pytest.mark.parametrize("heads,kv_heads", [(32, 8), (8, 8), (64, 2), (128, 2), (300, 300), (24, 4)])
def test_select_workspace(heads, kv_heads):
    """Bounded (4096 tokens over 8192 table entries of 8 KV heads took 1 GiB), growing with tokens and entries, the
    same for every split of the tokens into sequences, and never less than one token's."""
    size = lambda *a, **kw: select_size(*a, heads=heads, kv_heads=kv_heads, **kw)
    strides = [1, 100, 256, 257, 1032, 2048, 2049, 8192, 8193, 16384, 32768, 40000, 131072, 10 ** 6, 10 ** 7]
    tokens = [1, 2, 3, 15, 31, 32, 33, 127, 255, 256, 512, 4096, 70000]
    for i, w in enumerate(strides):
        one = 4 * kv_heads * w
        for j, t in enumerate(tokens):
            b = size(t, w)
            assert one <= b <= max(128 << 20, 4 * kv_heads * ((w + 255) // 256 * 256))
            assert i == 0 or size(t, strides[i - 1]) <= b
            assert j == 0 or size(tokens[j - 1], w) <= b
            assert size(t, w, seqs=min(t, 9), n=t) == b and size(t, w, seqs=min(t, 9), n=1) == b


def test_select_widest_table():
    """A width is rounded up to 256 entries in 32 bits: one that cannot be is refused (it gave a size near 2^64)."""
    a, size = _lib.SelectArgs(), ctypes.c_size_t(7)
    a.dtype, a.q_heads, a.kv_heads, a.head_dim, a.page_size, a.num_pages = 1, 8, 8, 128, 16, 100
    a.num_seqs, a.max_query_len, a.total_tokens, a.keep, a.sinks, a.window, a.causal = 1, 1, 1, 8, 1, 2, 1
    a.q = a.bounds.bounds = a.bounds.scale = a.positions = a.block_tables = a.tables = a.lengths = PTR
    L = ti.load_library()
    for stride, want in ((2 ** 31 - 256, _lib.TI_OK), (2 ** 31 - 255, _lib.TI_ERR_UNSUPPORTED), (2 ** 31 - 1, _lib.TI_ERR_UNSUPPORTED)):
        a.block_table_stride = stride
        assert L.ti_select_pages_workspace_bytes(ctypes.byref(a), ctypes.byref(size)) == want
        assert size.value == (8 * 4 * stride if want == _lib.TI_OK else 0)
        assert L.ti_select_pages(ctypes.byref(a), None) == (_lib.TI_ERR_WORKSPACE if want == _lib.TI_OK else want)


@pytest.mark.parametrize("P,width", [(1, 2 ** 31 - 1), (1, 2 ** 31 - 255), (2 ** 31 - 1, 1), (2 ** 30 - 1, 2)])
def test_attend_longest_table(P, width):
    """Key counts are 32-bit and rounded up to tiles: a table that holds 2^31 keys but for a few is refused (a full
    one of 2^31 - 1 keys wrapped to none); one of 2^31 - 256 is not."""
    L, size = ti.load_library(), ctypes.c_size_t(7)
    c, a = _lib.KVCache(), _lib.SparseAttentionArgs()
    c.kind, c.head_dim, c.page_size, c.kv_heads, c.num_pages, c.k_pages, c.v_pages = 0, 128, P, 8, 100, PTR, PTR
    a.dtype, a.q_heads, a.total_tokens, a.table_width, a.num_seqs, a.max_query_len, a.scale = 1, 32, 4, width, 4, 1, 0.1
    a.q = a.out = a.tables = a.lengths = PTR
    assert L.ti_sparse_attention(ctypes.byref(a), ctypes.byref(c), None) == _lib.TI_ERR_UNSUPPORTED
    for name in ("bytes", "bound"):
        assert getattr(L, f"ti_sparse_attention_workspace_{name}")(ctypes.byref(a), ctypes.byref(c), ctypes.byref(size)) == _lib.TI_ERR_UNSUPPORTED
        assert size.value == 0
    c.page_size, a.table_width = 1, 2 ** 31 - 256
    assert L.ti_sparse_attention(ctypes.byref(a), ctypes.byref(c), None) == _lib.TI_ERR_WORKSPACE


def test_launches_past_32_bits_of_threads():
    """Work-groups times 256 threads have to fit 32 bits: refused before any HIP call, not a failed launch."""
    L, size = ti.load_library(), ctypes.c_size_t(7)
    c, a = _lib.KVCache(), _lib.SparseAttentionArgs()
    c.kind, c.head_dim, c.page_size, c.kv_heads, c.num_pages, c.k_pages, c.v_pages = 0, 128, 16, 8, 100, PTR, PTR
    a.dtype, a.q_heads, a.table_width, a.num_seqs, a.max_query_len, a.scale = 1, 8, 64, 1, 1, 0.1
    a.q = a.out = a.tables = a.lengths = a.query_start_loc = PTR
    call = lambda: L.ti_sparse_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(c), ctypes.byref(size))
    a.total_tokens = 2 ** 21
    assert call() == _lib.TI_ERR_UNSUPPORTED and L.ti_sparse_attention(ctypes.byref(a), ctypes.byref(c), None) == _lib.TI_ERR_UNSUPPORTED
    a.total_tokens = 2 ** 21 - 1
    assert call() == _lib.TI_OK
    a.total_tokens, a.max_query_len = 2 ** 23 - 1, 2 ** 20     # 16 tokens together
    assert call() == _lib.TI_OK
    kb = _lib.KeyBoundsArgs(PTR, PTR)
    assert L.ti_update_key_bounds(1, ctypes.byref(c), ctypes.byref(kb), PTR, 2 ** 24, PTR, None, 1, 2 ** 28, 2 ** 28, None) \
        == _lib.TI_ERR_UNSUPPORTED
