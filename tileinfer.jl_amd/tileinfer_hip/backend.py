"""HipBackend: the reference's op interface (src/ops/interface.jl) on the gfx950 kernels.

Each function mirrors one method of the reference for its TileBackend (same name with `!`
spelled as a trailing `_`, same argument order and meaning) and calls one entry point of
libtileinfer_hip.so, from the native call path (_calls.so) where the arguments are plain
ones, else through ctypes after the checks below. torch tensors only carry device memory and
the current stream; all compute is in the HIP library, and there is no fallback: if the
library is missing, the first call raises.

Shapes are C order (the reference's column-major shapes reversed):
q, out [n][heads][D]; k, v [n][kv_heads][D]; dense pools [pages][kv_heads][P][D];
qkv [n][(heads + 2 kv_heads) D]; block_table int32 [>= pages of the sequence], 1-based,
zero-padded; positions int32 [n], 0-based; slots int32 [n], 1-based.
"""
from __future__ import annotations

import contextlib
import ctypes
from typing import Optional

import torch

from . import _lib
from ._lib import (ArgumentError, AttentionArgs, KeyBoundsArgs, KVCache, PagePoolArgs, SelectArgs, SparseAttentionArgs,
                   VerifyArgs, check)
from .kv import Fp8Pages, Int8Pages, KeyBounds, PagePool, fp8_layer_arrays, layer_arrays
from .rope import RotaryTable


def _done(status: int) -> bool:
    """Whether the native call path made a call (raising what it reported): it leaves
    arguments that are not plain ones (-1) to the checks below."""
    if status > 0:
        check(status)
    return status == 0


class HipBackend:
    """Selects the MI355X kernels, as TileBackend selects the cuTile ones
    (src/ops/interface.jl:15-21)."""

    def __repr__(self) -> str:
        return "HipBackend()"


_OPS = {"attention", "attention!", "store_kv!", "rmsnorm", "rmsnorm!", "rope", "rope!", "attention_inputs!",
        "update_key_bounds!", "select_pages", "select_pages!", "sparse_attention", "sparse_attention!", "verify_draft",
        "verify_draft!", "window_attention", "window_attention!", "reserve_pages!", "release_pages!"}


def supports_graphs(be: HipBackend) -> bool:
    """In-place ops neither allocate nor synchronize (src/ops/interface.jl:282-288)."""
    return True


def has_kernel(be: HipBackend, op) -> bool:
    """Whether the backend implements op itself (src/ops/interface.jl:290-295)."""
    name = op if isinstance(op, str) else getattr(op, "__name__", "")
    return name.rstrip("_") in {o.rstrip("!") for o in _OPS} or name in _OPS


def _dtype(t: torch.Tensor) -> int:
    if t.dtype == torch.bfloat16:
        return _lib.TI_BF16
    if t.dtype == torch.float32:
        return _lib.TI_F32
    raise ArgumentError(f"unsupported element type {t.dtype} (bfloat16 or float32)")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _dev(*ts):
    for t in ts:
        if t is not None:
            if not t.is_cuda:
                raise ArgumentError("tensors must be on the GPU")
            if not t.is_contiguous():
                raise ArgumentError("tensors must be contiguous")


def _i32(t: torch.Tensor, name: str):
    if t.dtype != torch.int32:
        raise ArgumentError(f"{name} must be int32")


def _stream(t: torch.Tensor) -> int:
    return torch.cuda.current_stream(t.device).cuda_stream


def kv_cache_struct(k_pages, v_pages, dtype: Optional[torch.dtype] = None) -> KVCache:
    """The ti_kv_cache of a layer: dense pools [pages][H][P][D], an Int8Pages or an Fp8Pages pair."""
    c = KVCache()
    if isinstance(k_pages, Fp8Pages) or isinstance(v_pages, Fp8Pages):
        lq, ls = fp8_layer_arrays(k_pages, v_pages)
        _dev(lq, ls)
        _, pages, H, P, D = lq.shape
        c.kind, c.layer_q, c.layer_scale = _lib.TI_KV_FP8, lq.data_ptr(), ls.data_ptr()
        c.head_dim, c.page_size, c.kv_heads, c.num_pages = D, P, H, pages
        return c
    if isinstance(k_pages, Int8Pages) or isinstance(v_pages, Int8Pages):
        lq, ls, sm = layer_arrays(k_pages, v_pages)
        _dev(lq, ls, sm)
        _, pages, H, P, D = lq.shape
        c.kind, c.layer_q, c.layer_scale, c.smooth = _lib.TI_KV_INT8, lq.data_ptr(), ls.data_ptr(), sm.data_ptr()
    else:
        _dev(k_pages, v_pages)
        if k_pages.shape != v_pages.shape or k_pages.dim() != 4 or k_pages.dtype != v_pages.dtype:
            raise ArgumentError("k_pages and v_pages must be matching [pages][kv_heads][P][D] pools")
        if dtype is not None and k_pages.dtype != dtype:
            raise ArgumentError("pools must have the activations' element type")
        pages, H, P, D = k_pages.shape
        c.kind, c.k_pages, c.v_pages = _lib.TI_KV_DENSE, k_pages.data_ptr(), v_pages.data_ptr()
    c.head_dim, c.page_size, c.kv_heads, c.num_pages = D, P, H, pages
    return c


def _pool_dtype(k_pages, like) -> Optional[torch.dtype]:
    """The element type that dense pools must have."""
    return None if isinstance(k_pages, (Int8Pages, Fp8Pages)) else like.dtype


def _fp8_device(c: KVCache, k_pages, *ts):
    """Where the library launches on an 8-bit block layer: its GPU, that of every tensor ts too. Else the current one."""
    if c.kind != _lib.TI_KV_FP8:
        return contextlib.nullcontext()
    for t in ts:
        if t is not None and t.device != k_pages.layer_q.device:
            raise ArgumentError("tensors must be on one GPU")
    return torch.cuda.device(k_pages.layer_q.device)


def _attention_args(out, q, block_tables, positions, scale, causal, path, num_seqs,
                    max_query_len, query_start_loc, workspace) -> AttentionArgs:
    a = AttentionArgs()
    a.dtype = _dtype(q)
    a.q_heads = q.shape[1]
    a.num_seqs = num_seqs
    a.max_query_len = max_query_len
    a.total_tokens = q.shape[0]
    a.block_table_stride = block_tables.shape[-1]
    a.q, a.out = _ptr(q), _ptr(out)
    a.positions = _ptr(positions)
    a.query_start_loc = _ptr(query_start_loc)
    a.block_tables = _ptr(block_tables)
    a.scale = float(scale)
    a.causal = int(bool(causal))
    a.path = int(path)
    a.workspace = _ptr(workspace)
    a.workspace_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()
    return a


def _shape_only(k_pages) -> KVCache:
    """A ti_kv_cache of the pools' shape and kind, for size queries."""
    c = KVCache()
    if isinstance(k_pages, Int8Pages):
        c.kind, c.layer_q, c.layer_scale, c.smooth = _lib.TI_KV_INT8, 16, 16, 16
    elif isinstance(k_pages, Fp8Pages):
        c.kind, c.layer_q, c.layer_scale = _lib.TI_KV_FP8, 16, 16
    else:
        c.kind, c.k_pages, c.v_pages = _lib.TI_KV_DENSE, 16, 16
    c.num_pages, c.kv_heads, c.page_size, c.head_dim = k_pages.shape
    return c


def workspace_bytes(q, k_pages, num_seqs: int = 1, max_query_len: Optional[int] = None,
                    path: int = _lib.TI_PATH_AUTO) -> int:
    """Bytes of split-KV scratch ti_attention needs for these query shapes (0 for none)."""
    # A shape-only query: the library validates and sizes, it never dereferences pointers.
    c = _shape_only(k_pages)
    n = max_query_len if max_query_len is not None else q.shape[0] // num_seqs
    a = AttentionArgs()
    a.dtype, a.q_heads, a.num_seqs, a.max_query_len = _dtype(q), q.shape[1], num_seqs, n
    a.total_tokens, a.block_table_stride = num_seqs * n, 1
    a.q = a.out = a.positions = a.block_tables = 1
    a.scale, a.causal, a.path = 1.0, 1, int(path)
    size = ctypes.c_size_t(0)
    check(_lib.load().ti_attention_workspace_bytes(ctypes.byref(a), ctypes.byref(c), ctypes.byref(size)))
    return size.value


def attention_workspace(be: HipBackend, q, k_pages, num_seqs: int = 1,
                        max_query_len: Optional[int] = None, path: int = _lib.TI_PATH_AUTO):
    """Scratch for attention_ with queries shaped like q, or None
    (attention_workspace, src/ops/tile/attention.jl:351-352). A byte tensor."""
    n = workspace_bytes(q, k_pages, num_seqs, max_query_len, path)
    return None if n == 0 else torch.empty(n, dtype=torch.uint8, device=q.device)


def paged_attention_(be: HipBackend, out, workspace, q, k_pages, v_pages, block_tables,
                     positions, scale: float, causal: bool = True,
                     query_start_loc: Optional[torch.Tensor] = None,
                     max_query_len: Optional[int] = None, path: int = _lib.TI_PATH_AUTO):
    """Batched attention_: sequence b owns tokens [qsl[b], qsl[b+1]) of q (or equal
    shares when query_start_loc is None) and block table row block_tables[b]."""
    if _done(_lib.native().attention(out, workspace, q, k_pages, v_pages, block_tables, positions, scale, causal,
                                     query_start_loc, max_query_len, path, False)):
        return out
    bts = block_tables if block_tables.dim() == 2 else block_tables.view(1, -1)
    B = bts.shape[0]
    _dev(out, q, bts, positions, query_start_loc, workspace)
    _i32(bts, "block_tables")
    _i32(positions, "positions")
    if q.dim() != 3 or out.shape != q.shape or out.dtype != q.dtype:
        raise ArgumentError("q and out must be matching [n][heads][D] tensors")
    if positions.numel() != q.shape[0]:
        raise ArgumentError("one position per query token")
    c = kv_cache_struct(k_pages, v_pages, _pool_dtype(k_pages, q))
    if q.shape[2] != c.head_dim:
        raise ArgumentError("q's head_dim differs from the pools'")
    if query_start_loc is not None:
        _i32(query_start_loc, "query_start_loc")
        if max_query_len is None:
            raise ArgumentError("max_query_len is required with query_start_loc")
    n = max_query_len if max_query_len is not None else q.shape[0] // B
    a = _attention_args(out, q, bts, positions, scale, causal, path, B, n, query_start_loc,
                        workspace)
    with _fp8_device(c, k_pages, q, out, bts, positions, query_start_loc, workspace):
        check(_lib.load().ti_attention(ctypes.byref(a), ctypes.byref(c), _stream(q)))
    return out


def attention_(be: HipBackend, out, workspace, q, k_pages, v_pages, block_table, positions,
               scale: float, causal: bool = True, path: int = _lib.TI_PATH_AUTO):
    """attention!(::TileBackend, out, workspace, q, k_pages, v_pages, block_table,
    positions, scale; causal) (src/ops/tile/attention.jl:359-366) for one sequence."""
    if _done(_lib.native().attention(out, workspace, q, k_pages, v_pages, block_table, positions, scale, causal,
                                     None, None, path, True)):
        return out
    return paged_attention_(be, out, workspace, q, k_pages, v_pages, block_table.view(1, -1),
                            positions, scale, causal, path=path)


def attention(be: HipBackend, q, k_pages, v_pages, block_table, positions, scale: float,
              causal: bool = True):
    """Allocating attention (src/ops/tile/attention.jl:368-371)."""
    out = torch.empty_like(q)
    return attention_(be, out, attention_workspace(be, q, k_pages), q, k_pages, v_pages,
                      block_table, positions, scale, causal)


def store_kv_(be: HipBackend, k_pages, v_pages, k, v, slots):
    """store_kv!(::TileBackend, k_pages, v_pages, k, v, slots)
    (src/ops/tile/elementwise.jl:133-140, :180-188). Into Fp8Pages a page's rows go from the first on: writing
    row 0 begins the page anew, later rows can only make its scale grow."""
    if _done(_lib.native().store_kv(k_pages, v_pages, k, v, slots)):
        return
    _dev(k, v, slots)
    _i32(slots, "slots")
    if k.shape != v.shape or k.dtype != v.dtype or k.dim() != 3:
        raise ArgumentError("k and v must be matching [n][kv_heads][D] tensors")
    c = kv_cache_struct(k_pages, v_pages, _pool_dtype(k_pages, k))
    if k.shape[1] != c.kv_heads or k.shape[2] != c.head_dim or slots.numel() != k.shape[0]:
        raise ArgumentError("k/v/slots shapes do not match the pools")
    with _fp8_device(c, k_pages, k, v, slots):
        check(_lib.load().ti_store_kv(_dtype(k), ctypes.byref(c), _ptr(k), _ptr(v), _ptr(slots),
                                      k.shape[0], _stream(k)))


def rmsnorm_(be: HipBackend, y, x, w, eps: float):
    """rmsnorm!(::TileBackend, y, x, w, eps) (src/ops/tile/norm.jl:31-38): every row of the
    last dimension of x normalized as rnd(rnd(x inv_rms) w). y may be x."""
    if _done(_lib.native().rmsnorm(y, x, w, eps)):
        return y
    _dev(y, x, w)
    if y.shape != x.shape or y.dtype != x.dtype or w.dtype != x.dtype or w.dim() != 1 \
            or w.shape[0] != x.shape[-1] or not (x.is_contiguous() and y.is_contiguous()):
        raise ArgumentError("rmsnorm shapes/types mismatch")
    H = x.shape[-1]
    check(_lib.load().ti_rmsnorm(_dtype(x), _ptr(y), _ptr(x), _ptr(w), x.numel() // H, H, float(eps),
                                 _stream(x)))
    return y


def rmsnorm(be: HipBackend, x, w, eps: float):
    return rmsnorm_(be, torch.empty_like(x), x, w, eps)


def rope_(be: HipBackend, y, x, cos, sin, positions):
    """rope!(::TileBackend, y, x, cos, sin, positions) (src/ops/tile/elementwise.jl:29-36).
    cos/sin: [max_len][D]."""
    if _done(_lib.native().rope(y, x, cos, sin, positions)):
        return y
    _dev(y, x, cos, sin, positions)
    _i32(positions, "positions")
    if x.dim() != 3 or y.shape != x.shape or y.dtype != x.dtype or cos.dtype != x.dtype \
            or sin.dtype != x.dtype or cos.shape != sin.shape or cos.shape[1] != x.shape[2]:
        raise ArgumentError("rope shapes/types mismatch")
    n, H, D = x.shape
    if positions.numel() != n:
        raise ArgumentError("one position per token")
    check(_lib.load().ti_rope(_dtype(x), _ptr(y), _ptr(x), _ptr(cos), _ptr(sin), cos.shape[0],
                              _ptr(positions), n, H, D, _stream(x)))
    return y


def rope(be: HipBackend, x, cos, sin, positions):
    return rope_(be, torch.empty_like(x), x, cos, sin, positions)


def attention_inputs_(be: HipBackend, q, k_pages, v_pages, qkv, q_norm, k_norm,
                      table: RotaryTable, positions, slots, eps: float):
    """attention_inputs!(::TileBackend, q, k_pages, v_pages, qkv, q_norm, k_norm, table,
    positions, slots, eps) (src/ops/tile/fused.jl:94-130): optional q/k RMSNorm, RoPE,
    queries into q, keys and values into the cache; returns q."""
    if _done(_lib.native().attention_inputs(q, k_pages, v_pages, qkv, q_norm, k_norm, table, positions, slots, eps)):
        return q
    _dev(q, qkv, q_norm, k_norm, table.cos_sin, positions, slots)
    _i32(positions, "positions")
    _i32(slots, "slots")
    n, nq, D = q.shape
    c = kv_cache_struct(k_pages, v_pages, _pool_dtype(k_pages, q))
    if qkv.dtype != q.dtype or qkv.numel() != n * (nq + 2 * c.kv_heads) * D or D != c.head_dim:
        raise ArgumentError("qkv must be [n][(heads + 2 kv_heads) D] in q's element type")
    if table.cos_sin.dtype != q.dtype or table.cos_sin.shape[1:] != (2, D):
        raise ArgumentError("rotary table must be [max_len][2][D] in q's element type")
    if (q_norm is None) != (k_norm is None):
        raise ArgumentError("q_norm and k_norm go together")
    if positions.numel() != n or slots.numel() != n:
        raise ArgumentError("one position and one slot per token")
    with _fp8_device(c, k_pages, q, qkv, q_norm, k_norm, table.cos_sin, positions, slots):
        check(_lib.load().ti_attention_inputs(
            _dtype(q), _ptr(q), ctypes.byref(c), _ptr(qkv), _ptr(q_norm), _ptr(k_norm),
            _ptr(table.cos_sin), table.cos_sin.shape[0], _ptr(positions), _ptr(slots), n, nq,
            float(eps), _stream(q)))
    return q


# ---- attention over chosen pages, and draft verification ---------------------------------------

def _one_device(first: torch.Tensor, *ts):
    """All on the GPU of `first` and contiguous; a context with that GPU as the current one, where the
    library launches."""
    _dev(first, *ts)
    for t in ts:
        if t is not None and t.device != first.device:
            raise ArgumentError("tensors must be on one GPU")
    return torch.cuda.device(first.device)


def _cache_tensors(k_pages, v_pages):
    if isinstance(k_pages, Int8Pages) or isinstance(v_pages, Int8Pages):
        return layer_arrays(k_pages, v_pages)
    if isinstance(k_pages, Fp8Pages) or isinstance(v_pages, Fp8Pages):
        return fp8_layer_arrays(k_pages, v_pages)
    return k_pages, v_pages


def _bounds_struct(b: KeyBounds) -> KeyBoundsArgs:
    if b.channel is not None and (b.channel.dtype != torch.float32 or b.channel.shape != (b.bounds.shape[1], b.bounds.shape[3])):
        raise ArgumentError("channel must be float32 [kv_heads][D]")
    return KeyBoundsArgs(_ptr(b.bounds), _ptr(b.scale), _ptr(b.channel))


def _step(block_tables, positions, query_start_loc, max_query_len):
    """(block tables as rows, sequences, most queries of one) of a step, as paged_attention_ takes it."""
    bts = block_tables if block_tables.dim() == 2 else block_tables.view(1, -1)
    B, T = bts.shape[0], positions.numel()
    _i32(bts, "block_tables")
    _i32(positions, "positions")
    if query_start_loc is not None:
        _i32(query_start_loc, "query_start_loc")
        if max_query_len is None:
            raise ArgumentError("max_query_len is required with query_start_loc")
        if query_start_loc.numel() != B + 1:
            raise ArgumentError("query_start_loc must hold an offset per sequence and the end")
    return bts, B, max_query_len if max_query_len is not None else T // max(B, 1)


def _workspace(size_of, device, *args):
    size = ctypes.c_size_t(0)
    check(size_of(*args, ctypes.byref(size)))
    return None if size.value == 0 else torch.empty(size.value, dtype=torch.uint8, device=device)


def _give_workspace(a, workspace):
    a.workspace = _ptr(workspace)
    a.workspace_bytes = 0 if workspace is None else workspace.numel() * workspace.element_size()


def update_key_bounds_(be: HipBackend, bounds: KeyBounds, k_pages, v_pages, block_tables, positions,
                       query_start_loc: Optional[torch.Tensor] = None, max_query_len: Optional[int] = None):
    """Refresh the bounds of the pages that hold the step's positions, from every key that the cache
    holds in them up to the step's end; the step as paged_attention_ takes it, its keys already
    written. It depends on the cached keys alone: after truncate() and another step on the same
    pages there is nothing else to call. Returns bounds."""
    if _done(_lib.native().update_key_bounds(bounds, k_pages, v_pages, block_tables, positions, query_start_loc, max_query_len)):
        return bounds
    on = _one_device(bounds.bounds, bounds.scale, bounds.channel, *_cache_tensors(k_pages, v_pages), block_tables, positions, query_start_loc)
    bts, B, n = _step(block_tables, positions, query_start_loc, max_query_len)
    c = kv_cache_struct(k_pages, v_pages)
    if bounds.shape != (c.num_pages, c.kv_heads, c.page_size, c.head_dim):
        raise ArgumentError("bounds do not belong to pools of this shape")
    dtype = _lib.TI_BF16 if c.kind != _lib.TI_KV_DENSE else _dtype(k_pages)
    kb = _bounds_struct(bounds)
    with on:
        check(_lib.load().ti_update_key_bounds(
            dtype, ctypes.byref(c), ctypes.byref(kb), _ptr(bts), bts.shape[1], _ptr(positions), _ptr(query_start_loc), B, n,
            positions.numel(), _stream(positions)))
    return bounds


def _select_args(q, bounds: KeyBounds, stride, B, n, keep, sinks, window, causal) -> SelectArgs:
    pages, H, P, D = bounds.shape
    if q.dim() != 3 or q.shape[2] != D or q.shape[1] % H:
        raise ArgumentError("q must be [n][heads][D] with the bounds' head_dim and a multiple of their KV heads")
    a = SelectArgs()
    a.dtype, a.q_heads, a.kv_heads, a.head_dim, a.page_size, a.num_pages = _dtype(q), q.shape[1], H, D, P, pages
    a.num_seqs, a.max_query_len, a.total_tokens, a.block_table_stride = B, n, q.shape[0], stride
    a.keep, a.sinks, a.window, a.causal = keep, sinks, window, int(bool(causal))
    return a


def select_pages_workspace(be: HipBackend, q, bounds: KeyBounds, block_tables):
    """Scratch of select_pages_: a byte tensor, enough for every call with q's heads of at most as many tokens as q
    has and block tables at most as wide (4 bytes per token, KV head and entry, up to 128 MiB or one token's)."""
    a = _select_args(q, bounds, block_tables.shape[-1], 1, q.shape[0], 1, 0, 1, True)
    a.q = a.bounds.bounds = a.bounds.scale = a.positions = a.block_tables = a.tables = a.lengths = 16
    return _workspace(_lib.load().ti_select_pages_workspace_bytes, q.device, ctypes.byref(a))


def select_pages_(be: HipBackend, tables, lengths, workspace, q, bounds: KeyBounds, block_tables, positions,
                  sinks: int = 1, window: int = 1, causal: bool = True,
                  query_start_loc: Optional[torch.Tensor] = None, max_query_len: Optional[int] = None):
    """The tables.shape[2] pages of its sequence that each query token of the step attends to, per KV head,
    by the bounds of their keys; the step as paged_attention_ takes it. tables [n][kv_heads][keep]
    int32: 1-based page ids in order of position, zero-padded; lengths [n][kv_heads] int32: the
    keys they hold, as sparse_attention_ takes both. The first `sinks` and the last `window` visible
    pages are always kept, the others by the largest product that a key inside their bounds could have
    with any of the KV head's queries (rounded to whole numbers); equal ones in order. Bounds and queries are
    rounded to 8 bits per head, which loses pages where a few dimensions are much larger than the rest
    unless the bounds have a channel (KeyBounds). Rows that belong to no sequence are left as they were.
    Returns (tables, lengths)."""
    if _done(_lib.native().select_pages(tables, lengths, workspace, q, bounds, block_tables, positions, sinks, window, causal,
                                        query_start_loc, max_query_len)):
        return tables, lengths
    on = _one_device(q, bounds.bounds, bounds.scale, bounds.channel, block_tables, positions, query_start_loc, tables, lengths, workspace)
    bts, B, n = _step(block_tables, positions, query_start_loc, max_query_len)
    _i32(tables, "tables")
    _i32(lengths, "lengths")
    if positions.numel() != q.shape[0]:
        raise ArgumentError("one position per query token")
    H = bounds.shape[1]
    if tables.dim() != 3 or tables.shape[:2] != (q.shape[0], H) or lengths.shape != (q.shape[0], H):
        raise ArgumentError("tables must be [n][kv_heads][keep] and lengths [n][kv_heads]")
    a = _select_args(q, bounds, bts.shape[1], B, n, tables.shape[2], int(sinks), int(window), causal)
    a.q, a.bounds, a.positions = _ptr(q), _bounds_struct(bounds), _ptr(positions)
    a.query_start_loc, a.block_tables, a.tables, a.lengths = _ptr(query_start_loc), _ptr(bts), _ptr(tables), _ptr(lengths)
    _give_workspace(a, workspace)
    with on:
        check(_lib.load().ti_select_pages(ctypes.byref(a), _stream(q)))
    return tables, lengths


def select_pages(be: HipBackend, q, bounds: KeyBounds, block_tables, positions, keep: int, sinks: int = 1, window: int = 1,
                 causal: bool = True, query_start_loc: Optional[torch.Tensor] = None, max_query_len: Optional[int] = None):
    """Allocating select_pages_: rows that belong to no sequence get empty tables."""
    H = bounds.shape[1]
    tables = torch.zeros((q.shape[0], H, int(keep)), dtype=torch.int32, device=q.device)
    lengths = torch.zeros((q.shape[0], H), dtype=torch.int32, device=q.device)
    return select_pages_(be, tables, lengths, select_pages_workspace(be, q, bounds, block_tables), q, bounds, block_tables,
                         positions, sinks, window, causal, query_start_loc, max_query_len)


def _sparse_args(q, width, B, n, scale) -> SparseAttentionArgs:
    a = SparseAttentionArgs()
    a.dtype, a.q_heads, a.total_tokens, a.table_width, a.num_seqs, a.max_query_len = _dtype(q), q.shape[1], q.shape[0], width, B, n
    a.scale = float(scale)
    return a


def _sparse_step(q, query_start_loc, max_query_len):
    n = int(max_query_len) if max_query_len is not None else 1
    if query_start_loc is None:
        if n <= 0 or q.shape[0] % n:
            raise ArgumentError("without query_start_loc every sequence has max_query_len tokens")
        return q.shape[0] // n, n
    if max_query_len is None:
        raise ArgumentError("max_query_len is required with query_start_loc")
    _i32(query_start_loc, "query_start_loc")
    return query_start_loc.numel() - 1, n


def _sparse_workspace(size_of, q, k_pages, tables, max_query_len):
    c = _shape_only(k_pages)
    a = _sparse_args(q, tables.shape[-1], 1, int(max_query_len), 1.0)
    a.q = a.out = a.tables = a.lengths = a.query_start_loc = 16
    return _workspace(size_of, q.device, ctypes.byref(a), ctypes.byref(c))


def sparse_attention_workspace(be: HipBackend, q, k_pages, tables, max_query_len: int = 1):
    """Scratch of sparse_attention_, or None where no such call needs any: a byte tensor, enough for every call with
    q's heads of at most as many tokens as q has, at most max_query_len of them a sequence and tables at most
    as wide."""
    return _sparse_workspace(_lib.load().ti_sparse_attention_workspace_bound, q, k_pages, tables, max_query_len)


def sparse_attention_(be: HipBackend, out, workspace, q, k_pages, v_pages, tables, lengths, scale: float,
                      query_start_loc: Optional[torch.Tensor] = None, max_query_len: Optional[int] = None):
    """Attention of each query token and KV head over the keys 0 .. lengths - 1 of its own table of pages
    (select_pages_, or any other choice), all of them visible. tables [n][kv_heads][width] int32 1-based
    page ids, lengths [n][kv_heads] int32. A token without keys gets zeros. With query_start_loc, rows
    that belong to no sequence are left as they were. max_query_len (1 without query_start_loc: every
    token a sequence) says that up to so many rows next to each other are one sequence's step, whose
    tables share pages."""
    if _done(_lib.native().sparse_attention(out, workspace, q, k_pages, v_pages, tables, lengths, scale, query_start_loc,
                                            max_query_len)):
        return out
    on = _one_device(q, out, *_cache_tensors(k_pages, v_pages), tables, lengths, query_start_loc, workspace)
    _i32(tables, "tables")
    _i32(lengths, "lengths")
    if q.dim() != 3 or out.shape != q.shape or out.dtype != q.dtype:
        raise ArgumentError("q and out must be matching [n][heads][D] tensors")
    c = kv_cache_struct(k_pages, v_pages, _pool_dtype(k_pages, q))
    if q.shape[2] != c.head_dim:
        raise ArgumentError("q's head_dim differs from the pools'")
    if tables.dim() != 3 or tables.shape[:2] != (q.shape[0], c.kv_heads) or lengths.shape != (q.shape[0], c.kv_heads):
        raise ArgumentError("tables must be [n][kv_heads][width] and lengths [n][kv_heads]")
    B, n = _sparse_step(q, query_start_loc, max_query_len)
    a = _sparse_args(q, tables.shape[2], B, n, scale)
    a.q, a.out, a.tables, a.lengths, a.query_start_loc = _ptr(q), _ptr(out), _ptr(tables), _ptr(lengths), _ptr(query_start_loc)
    _give_workspace(a, workspace)
    with on:
        check(_lib.load().ti_sparse_attention(ctypes.byref(a), ctypes.byref(c), _stream(q)))
    return out


def sparse_attention(be: HipBackend, q, k_pages, v_pages, tables, lengths, scale: float,
                     query_start_loc: Optional[torch.Tensor] = None, max_query_len: Optional[int] = None):
    """Allocating sparse_attention_: rows that belong to no sequence are zero."""
    out = torch.empty_like(q) if query_start_loc is None else torch.zeros_like(q)
    ws = _sparse_workspace(_lib.load().ti_sparse_attention_workspace_bytes, q, k_pages, tables,
                           1 if max_query_len is None else max_query_len)
    return sparse_attention_(be, out, ws, q, k_pages, v_pages, tables, lengths, scale, query_start_loc, max_query_len)


def _verify_args(target) -> VerifyArgs:
    if target.dim() != 3:
        raise ArgumentError("target must be [sequences][drafts + 1][vocabulary]")
    a = VerifyArgs()
    a.dtype, a.num_seqs, a.max_drafts, a.vocab = _dtype(target), target.shape[0], target.shape[1] - 1, target.shape[2]
    return a


def verify_draft_workspace(be: HipBackend, target):
    """Scratch of verify_draft_ for target probabilities of this shape: a byte tensor."""
    a = _verify_args(target)
    a.draft_tokens = a.target = a.uniforms = a.accepted = a.tokens = 16
    return _workspace(_lib.load().ti_verify_draft_workspace_bytes, target.device, ctypes.byref(a))


def verify_draft_(be: HipBackend, accepted, tokens, workspace, draft_tokens, target, draft, uniforms,
                  draft_lens: Optional[torch.Tensor] = None):
    """End of a verify step: how many drafts of each sequence are accepted, and its next tokens.
    draft_tokens [B][N] int32 (0-based), target [B][N + 1][V] probabilities at the positions before
    each draft and after the last, draft [B][N][V] the drafter's (None: it gave its tokens alone),
    uniforms [B][N + 1] float32 in [0, 1), draft_lens [B] int32 (None: N each). Draft i is accepted while
    u_i draft_i(x_i) < target_i(x_i); one token more is drawn with the last uniform, from max(target -
    draft, 0) where a draft was rejected (without the drafter's probabilities: the target's but for the
    draft), else from the target's. accepted [B] int32; tokens [B][N + 1] int32: the accepted drafts, the
    drawn token, -1 behind it. truncate() takes the rejected positions out of the cache. Returns
    (accepted, tokens)."""
    if _done(_lib.native().verify_draft(accepted, tokens, workspace, draft_tokens, target, draft, uniforms, draft_lens)):
        return accepted, tokens
    on = _one_device(target, accepted, tokens, workspace, draft_tokens, draft, uniforms, draft_lens)
    a = _verify_args(target)
    B, N, V = a.num_seqs, a.max_drafts, a.vocab
    for t, name in ((accepted, "accepted"), (tokens, "tokens"), (draft_tokens, "draft_tokens")):
        _i32(t, name)
    if draft_tokens.shape != (B, N) or tokens.shape != (B, N + 1) or accepted.shape != (B,):
        raise ArgumentError("draft_tokens must be [B][N], tokens [B][N + 1] and accepted [B]")
    if draft is not None and (draft.shape != (B, N, V) or draft.dtype != target.dtype):
        raise ArgumentError("draft must be [B][N][V] in target's element type")
    if uniforms.shape != (B, N + 1) or uniforms.dtype != torch.float32:
        raise ArgumentError("uniforms must be float32 [B][N + 1]")
    if draft_lens is not None:
        _i32(draft_lens, "draft_lens")
        if draft_lens.shape != (B,):
            raise ArgumentError("draft_lens must be [B]")
    a.draft_tokens, a.draft_lens, a.target, a.draft = _ptr(draft_tokens), _ptr(draft_lens), _ptr(target), _ptr(draft)
    a.uniforms, a.accepted, a.tokens = _ptr(uniforms), _ptr(accepted), _ptr(tokens)
    _give_workspace(a, workspace)
    with on:
        check(_lib.load().ti_verify_draft(ctypes.byref(a), _stream(target)))
    return accepted, tokens


def verify_draft(be: HipBackend, draft_tokens, target, draft, uniforms, draft_lens: Optional[torch.Tensor] = None):
    """Allocating verify_draft_."""
    B, N1 = target.shape[:2]
    accepted = torch.empty(B, dtype=torch.int32, device=target.device)
    tokens = torch.empty((B, N1), dtype=torch.int32, device=target.device)
    return verify_draft_(be, accepted, tokens, verify_draft_workspace(be, target), draft_tokens, target, draft, uniforms, draft_lens)


# ---- attention with a sliding window, and the page bookkeeping of a step -------------------------

def _window_args(q, window, sinks, B, n):
    a = AttentionArgs()
    a.dtype, a.q_heads, a.num_seqs, a.max_query_len = _dtype(q), q.shape[1], B, n
    a.total_tokens, a.causal, a.path = q.shape[0], 1, _lib.TI_PATH_AUTO
    if isinstance(window, bool) or isinstance(sinks, bool) or int(window) != window or int(sinks) != sinks \
            or not 1 <= window < 1 << 31 or not 0 <= sinks < 1 << 31:
        raise ArgumentError("window must be a whole number from 1 on, sinks from 0 on")
    return a


def window_attention_workspace(be: HipBackend, q, k_pages, window: int, sinks: int = 0, num_seqs: int = 1,
                               max_query_len: Optional[int] = None):
    """Scratch of window_attention_ for steps of these sizes, or None where there is none: a byte tensor."""
    a = _window_args(q, window, sinks, num_seqs, max_query_len if max_query_len is not None else q.shape[0] // max(num_seqs, 1))
    a.block_table_stride, a.scale = 1, 1.0
    a.q = a.out = a.positions = a.block_tables = a.query_start_loc = 16
    c = _shape_only(k_pages)
    return _workspace(_lib.load().ti_window_attention_workspace_bytes, q.device, ctypes.byref(a), int(window), int(sinks), ctypes.byref(c))


def window_attention_(be: HipBackend, out, workspace, q, k_pages, v_pages, block_tables, positions, scale: float, window: int,
                      sinks: int = 0, query_start_loc: Optional[torch.Tensor] = None, max_query_len: Optional[int] = None):
    """Causal attention where the query at position p sees the keys p - window + 1 .. p and the first `sinks`; caches of any
    kind and steps as paged_attention_ takes them. Table entries of pages that hold no visible key are not used
    (release_pages_ gives such pages back), and a key that a query does not see never reaches its output, whatever the
    cache holds there. Rows that belong to no sequence are left as they were."""
    if _done(_lib.native().window_attention(out, workspace, q, k_pages, v_pages, block_tables, positions, scale, window, sinks,
                                            query_start_loc, max_query_len)):
        return out
    on = _one_device(q, out, *_cache_tensors(k_pages, v_pages), block_tables, positions, query_start_loc, workspace)
    bts, B, n = _step(block_tables, positions, query_start_loc, max_query_len)
    if q.dim() != 3 or out.shape != q.shape or out.dtype != q.dtype:
        raise ArgumentError("q and out must be matching [n][heads][D] tensors")
    if positions.numel() != q.shape[0]:
        raise ArgumentError("one position per query token")
    c = kv_cache_struct(k_pages, v_pages, _pool_dtype(k_pages, q))
    if q.shape[2] != c.head_dim:
        raise ArgumentError("q's head_dim differs from the pools'")
    a = _window_args(q, window, sinks, B, n)
    a.block_table_stride, a.scale = bts.shape[1], float(scale)
    a.q, a.out, a.positions, a.query_start_loc, a.block_tables = _ptr(q), _ptr(out), _ptr(positions), _ptr(query_start_loc), _ptr(bts)
    _give_workspace(a, workspace)
    with on:
        check(_lib.load().ti_window_attention(ctypes.byref(a), int(window), int(sinks), ctypes.byref(c), _stream(q)))
    return out


def window_attention(be: HipBackend, q, k_pages, v_pages, block_tables, positions, scale: float, window: int, sinks: int = 0,
                     query_start_loc: Optional[torch.Tensor] = None, max_query_len: Optional[int] = None):
    """Allocating window_attention_: rows that belong to no sequence are zero."""
    out = torch.empty_like(q) if query_start_loc is None else torch.zeros_like(q)
    B = block_tables.shape[0] if block_tables.dim() == 2 else 1
    return window_attention_(be, out, window_attention_workspace(be, q, k_pages, window, sinks, B, max_query_len), q, k_pages, v_pages,
                             block_tables, positions, scale, window, sinks, query_start_loc, max_query_len)


def _pool_args(pool: PagePool, *ts):
    """The ti_page_pool and a context with its GPU as the current one; ts on it too."""
    state = (pool.free_count, pool.tables, pool.lengths, pool.behind, pool.ticket)
    on = _one_device(pool.free, *state, *ts)
    for t in (pool.free, *state, *ts):
        if t is not None:
            _i32(t, "a pool's and a step's tensors")
    S, W = pool.tables.shape
    if pool.free_count.numel() != 1 or pool.lengths.shape != (S,) or (pool.behind is not None and pool.behind.shape != (S,)):
        raise ArgumentError("a pool has one length per sequence")
    a = PagePoolArgs(pool.free.numel(), pool.page_size, S, W, pool.window, pool.sinks, _ptr(pool.free), _ptr(pool.free_count),
                     _ptr(pool.tables), _ptr(pool.lengths), _ptr(pool.behind), _ptr(pool.ticket))
    return a, on


def reserve_pages_(be: HipBackend, pool: PagePool, counts, positions, slots, query_start_loc, short):
    """reserve and slots (src/kv/block_manager.jl:58-65, 97-100) for every sequence of a step, on the GPU: counts [sequences]
    int32 more positions each. Writes the step's query_start_loc [sequences + 1], and the positions and slots [tokens] of
    its tokens, 0 behind them (slot 0 writes nothing); pool.tables and pool.lengths then hold the step. short [1] int32: 0,
    or the pages that were missing, or -1 where a sequence would outgrow its table or the step the token arrays: then
    nothing is reserved and the step is empty. Calls on one pool must not overlap. Returns (positions, slots, query_start_loc, short)."""
    if _done(_lib.native().reserve_pages(pool, counts, positions, slots, query_start_loc, short)):
        return positions, slots, query_start_loc, short
    a, on = _pool_args(pool, counts, positions, slots, query_start_loc, short)
    S = pool.tables.shape[0]
    if counts.shape != (S,) or query_start_loc.shape != (S + 1,) or short.numel() != 1 or positions.dim() != 1 or slots.shape != positions.shape:
        raise ArgumentError("counts must be [sequences], query_start_loc [sequences + 1], positions and slots [tokens], short [1]")
    with on:
        check(_lib.load().ti_reserve_pages(ctypes.byref(a), _ptr(counts), positions.numel(), _ptr(positions), _ptr(slots),
                                           _ptr(query_start_loc), _ptr(short), _stream(pool.free)))
    return positions, slots, query_start_loc, short


def release_pages_(be: HipBackend, pool: PagePool, lengths):
    """truncate (src/kv/block_manager.jl:74-81) for every sequence, on the GPU: sequence b keeps its first lengths[b]
    positions (all, where that is more), unused pages go back, and with a window those that no query at a kept
    position's successor or later sees. The stack gets them in the opposite order to that in which reserve_pages_ takes them: a
    step taken back whole leaves the pool as it was. Calls on one pool must not overlap. Returns pool."""
    if _done(_lib.native().release_pages(pool, lengths)):
        return pool
    a, on = _pool_args(pool, lengths)
    if lengths.shape != pool.lengths.shape:
        raise ArgumentError("lengths must be [sequences]")
    with on:
        check(_lib.load().ti_release_pages(ctypes.byref(a), _ptr(lengths), _stream(pool.free)))
    return pool
