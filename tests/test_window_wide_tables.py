"""Block tables that hold more positions than the windowed and 8-bit kernels count: refused, where the positions past 2^30 were
read as 2^30 (no GPU)."""
import ctypes

import pytest

from test_window_refusals import OK, UNSUPPORTED, args, cache, window_bytes
from tileinfer_hip import _lib


@pytest.mark.parametrize("dtype", [_lib.TI_F32, _lib.TI_BF16])
@pytest.mark.parametrize("n", [1, 16, 600])
@pytest.mark.parametrize("P,width", [(16, 1 << 26), (64, 1 << 24), (1024, 1 << 20)])
def test_tables_past_2_30_positions(dtype, n, P, width):
    L, size = _lib.load(), ctypes.c_size_t()
    for kind in (_lib.TI_KV_DENSE, _lib.TI_KV_INT8, _lib.TI_KV_FP8):
        c = cache(kind, P=P)
        for w, st in ((width, OK), (width + 1, UNSUPPORTED), (2 ** 31 - 1, UNSUPPORTED)):
            a = args(dtype=dtype, num_seqs=1, max_query_len=n, total_tokens=n, block_table_stride=w)
            assert window_bytes(a, c, 4096, 4)[0] == st
            if st:
                assert L.ti_window_attention(ctypes.byref(a), 4096, 4, ctypes.byref(c), None) == st
            # without a window: 8-bit block caches
            want = st if kind == _lib.TI_KV_FP8 else OK
            assert L.ti_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(c), ctypes.byref(size)) == want
            if want:
                assert L.ti_attention(ctypes.byref(a), ctypes.byref(c), None) == want
                assert L.ti_attention_noalloc(ctypes.byref(a), ctypes.byref(c), None) == want
