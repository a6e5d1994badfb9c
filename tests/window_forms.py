"""Which kernel takes a windowed step of many tokens, asked of the library's own rule on the host (no GPU), steps that reach each
form of the ping-pong prefill kernel with keys that a window hides, and outputs in 64 bits for steps of that size."""
from __future__ import annotations

import ctypes

import numpy as np
import torch

import tileinfer_hip as ti
from tileinfer_hip import _lib

NONE, SHARED, KSPLIT, SOLO = range(4)


class _Window(ctypes.Structure):
    _fields_ = [("size", ctypes.c_int), ("sinks", ctypes.c_int)]


def pick(kv, lens, window, sinks, D, H, G, P):
    """The form of the ping-pong kernel that a step over a bf16, INT8 or 8-bit block cache takes (window 0: none), tables as wide
    as the longest sequence (as window_ref.Step makes them)."""
    f = getattr(ti.load_library(), "_Z18ti_pick_prefill_ppPK17ti_attention_argsPK11ti_kv_cacheib9ti_window")
    f.restype, f.argtypes = ctypes.c_int, [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int, ctypes.c_bool, _Window]
    c = _lib.KVCache()
    c.kind = {"bf16": _lib.TI_KV_DENSE, "int8": _lib.TI_KV_INT8, "fp8": _lib.TI_KV_FP8}[kv]
    c.head_dim, c.page_size, c.kv_heads, c.num_pages = D, P, H, 1000
    a = _lib.AttentionArgs()
    a.dtype, a.q_heads, a.num_seqs, a.max_query_len = _lib.TI_BF16, H * G, len(lens), max(n for _, n in lens)
    a.total_tokens, a.block_table_stride = sum(n for _, n in lens), max(-(-(x + n) // P) for x, n in lens)
    a.scale, a.causal = 1.0, 1
    return f(ctypes.byref(a), ctypes.byref(c), _lib.TI_PATH_AUTO, True, _Window(window, sinks))


# (form, kv, D, lens, H, G, P, window, sinks): each form that a cache's kind has, at both head dims, with pages of 16 and 64
# keys, windows and sinks that end inside tiles, sequences shorter than the window and batches of unequal ones.
FORMS = [
    (SHARED, "bf16", 128, [(1000, 1500)], 8, 4, 16, 425, 37),
    (SHARED, "bf16", 128, [(1000, 700)] * 3, 8, 4, 64, 425, 0),
    (SHARED, "bf16", 128, [(0, 900), (3000, 700), (100, 33), (40, 0), (5, 650)], 8, 4, 16, 300, 70),
    (SHARED, "bf16", 128, [(0, 3000)], 8, 4, 64, 700, 4),
    (SHARED, "bf16", 128, [(200, 2100)], 5, 5, 16, 1, 0),
    (KSPLIT, "bf16", 128, [(1000, 900)], 8, 4, 16, 425, 37),
    (KSPLIT, "bf16", 128, [(333, 500), (900, 450)], 8, 4, 64, 129, 5),
    (KSPLIT, "bf16", 128, [(2000, 100)] * 8, 8, 4, 16, 1450, 100),
    (KSPLIT, "bf16", 64, [(1000, 1500)], 8, 4, 16, 425, 37),
    (KSPLIT, "bf16", 64, [(500, 900)], 8, 4, 64, 77, 0),
    (SOLO, "bf16", 128, [(1000, 150), (0, 20), (300, 130)] * 6, 8, 4, 16, 425, 37),
    (SOLO, "bf16", 64, [(1000, 700)] * 3, 8, 4, 16, 425, 37),
    (SOLO, "bf16", 64, [(700, 300), (0, 250), (90, 180), (0, 1)] * 3, 8, 8, 64, 333, 100),
    (KSPLIT, "int8", 128, [(2000, 1500)], 8, 4, 16, 1449, 37),
    (KSPLIT, "int8", 64, [(2000, 1300)], 8, 4, 64, 1400, 4),
    (SOLO, "int8", 128, [(1000, 700)] * 3, 8, 4, 16, 425, 37),
    (SOLO, "int8", 128, [(0, 2300)], 8, 4, 64, 300, 0),
    (SOLO, "int8", 64, [(1000, 700), (0, 690), (100, 650)], 8, 4, 16, 425, 37),
    (SHARED, "fp8", 128, [(1000, 1500)], 8, 4, 16, 425, 37),
    (SHARED, "fp8", 128, [(0, 900), (3000, 700), (100, 33), (40, 0), (5, 650)], 8, 4, 64, 300, 70),
    (KSPLIT, "fp8", 128, [(1000, 900)], 8, 4, 16, 425, 37),
    (KSPLIT, "fp8", 128, [(333, 500), (900, 450)], 8, 4, 64, 129, 5),
    (KSPLIT, "fp8", 64, [(1000, 1500)], 8, 4, 16, 425, 37),
    (SOLO, "fp8", 128, [(1000, 150), (0, 20), (300, 130)] * 6, 8, 4, 16, 425, 37),
    (SOLO, "fp8", 64, [(1000, 700)] * 3, 8, 4, 64, 425, 37),
]


def want(s):
    """s.want() of a window_ref.Step, causal, by whole sequences, in float64 on the GPU."""
    window = s.window or 1 << 30
    q = s.q.double().cuda()
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    at = 0
    for b, (c, n) in enumerate(s.lens):
        if n == 0:
            continue
        i = np.arange(c + n)
        page, off = np.maximum(s.tables[b][i // s.P].astype(np.int64) - 1, 0), i % s.P
        held = np.zeros(c + n, bool)
        held[s.rows[b]] = True
        key, pos = torch.arange(c + n, device="cuda"), torch.arange(c, c + n, device="cuda")[:, None]
        sees = ((key <= pos) & ((key > pos - window) | (key < s.sinks))).repeat_interleave(s.G, 0)
        for h in range(s.H):
            k, v = (torch.from_numpy(np.where(held[:, None], x[page, h, off], 0.0)).cuda() for x in (s.layer.k, s.layer.v))
            heads = slice(h * s.G, (h + 1) * s.G)
            x = q[at:at + n, heads].reshape(n * s.G, s.D) @ k.T.contiguous() * s.scale
            w = torch.softmax(x.masked_fill(~sees, -torch.inf), 1)
            out[at:at + n, heads] = (w @ v).view(n, s.G, s.D)
            size[at:at + n, heads] = (w @ v.abs()).view(n, s.G, s.D)
        at += n
    return out.cpu().numpy(), size.cpu().numpy()
