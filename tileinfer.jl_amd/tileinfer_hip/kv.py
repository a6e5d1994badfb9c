"""Paged KV cache: host-side page allocation and the device page pools.

Mirrors src/kv/block_manager.jl (BlockManager, Sequence, reserve!, truncate!, release!,
slots, OutOfPagesError), src/kv/paged_cache.jl (PagedKVCache) and the INT8 cache types of
src/ops/quant.jl:56-135 (Int8Pages, int8_kv_pools, key_smoothing, layer_arrays).

Pools are torch tensors in C order, the reference's column-major shapes reversed:
dense (head_dim, page_size, kv_heads, pages) -> [pages][kv_heads][page_size][head_dim];
an INT8 layer's values `layer_q` (D, P, H, pages, 2) -> [2][pages][H][P][D] (keys first)
and scales `layer_scale` (P, H, pages, 2) -> [2][pages][H][P]. Page ids and slots are
1-based, as in the reference, so block tables and slots pass through unchanged. Fp8Pages (8-bit pages
with one scale per page and KV head) and PagePool (the bookkeeping of the pages on the GPU) have no
counterpart there.
"""
from __future__ import annotations

from dataclasses import dataclass, field
from typing import List, Optional

import torch

from ._lib import ArgumentError

DEFAULT_PAGE_SIZE = 64  # src/kv/paged_cache.jl:7


class OutOfPagesError(Exception):
    """Raised by reserve when the pool has fewer free pages than a step needs
    (src/kv/block_manager.jl:26-32)."""

    def __init__(self, needed: int, free: int):
        super().__init__(f"KV cache full: need {needed} more pages, {free} free")
        self.needed, self.free = needed, free


@dataclass
class Sequence:
    """A sequence's block table (1-based page ids) and cached token ids
    (src/kv/block_manager.jl:13-18)."""
    block_table: List[int] = field(default_factory=list)
    tokens: List[int] = field(default_factory=list)

    def __len__(self) -> int:
        return len(self.tokens)


class BlockManager:
    """Hands out the pages of a pool of num_pages pages of page_size positions
    (src/kv/block_manager.jl:39-50). The free list is a stack, reversed so pages are
    handed out in increasing order."""

    def __init__(self, num_pages: int, page_size: int):
        self.num_pages, self.page_size = int(num_pages), int(page_size)
        self.free: List[int] = list(range(self.num_pages, 0, -1))

    def num_free_pages(self) -> int:
        return len(self.free)


def _cld(a: int, b: int) -> int:
    return -(-a // b)


def reserve(b: BlockManager, seq: Sequence, n: int) -> Sequence:
    """Pages for n more positions of seq; raises OutOfPagesError before changing anything
    (src/kv/block_manager.jl:58-65)."""
    needed = _cld(len(seq) + n, b.page_size) - len(seq.block_table)
    if needed > b.num_free_pages():
        raise OutOfPagesError(needed, b.num_free_pages())
    for _ in range(max(needed, 0)):
        seq.block_table.append(b.free.pop())
    return seq


def truncate(b: BlockManager, seq: Sequence, n: int) -> Sequence:
    """Keep the first n cached positions; unused pages go back to the pool
    (src/kv/block_manager.jl:74-81)."""
    if not 0 <= n <= len(seq):
        raise ArgumentError(f"cannot truncate a sequence of length {len(seq)} to {n}")
    del seq.tokens[n:]
    keep = _cld(n, b.page_size)
    b.free.extend(reversed(seq.block_table[keep:]))
    del seq.block_table[keep:]
    return seq


def release(b: BlockManager, seq: Sequence) -> Sequence:
    """Return all pages of seq (src/kv/block_manager.jl:88)."""
    return truncate(b, seq, 0)


def slots(b: BlockManager, seq: Sequence, start: int, n: int) -> List[int]:
    """1-based cache slots of positions start .. start+n-1: (page - 1) P + offset + 1
    (src/kv/block_manager.jl:97-100)."""
    P = b.page_size
    return [(seq.block_table[p // P] - 1) * P + p % P + 1 for p in range(start, start + n)]


class Int8Pages:
    """One half (keys or values) of an INT8 layer (src/ops/quant.jl:86-92): `q`
    [pages][H][P][D] int8 and `scale` [pages][H][P] f32 are views of the layer arrays
    `layer_q` [2][pages][H][P][D] and `layer_scale` [2][pages][H][P]; `smooth` [D] holds
    the keys' smoothing factors (ones for values)."""

    def __init__(self, layer_q: torch.Tensor, layer_scale: torch.Tensor, smooth: torch.Tensor,
                 half: int):
        self.layer_q, self.layer_scale, self.smooth, self.half = layer_q, layer_scale, smooth, half
        self.q = layer_q[half]
        self.scale = layer_scale[half]

    @property
    def shape(self):
        return tuple(self.q.shape)

    def size(self, d: Optional[int] = None):
        return self.q.size() if d is None else self.q.size(d)


def int8_kv_pools(head_dim: int, page_size: int, kv_heads: int, num_pages: int,
                  key_smoothing: Optional[torch.Tensor] = None, device="cuda"):
    """The zeroed key and value Int8Pages of one layer (src/ops/quant.jl:104-109)."""
    q = torch.zeros((2, num_pages, kv_heads, page_size, head_dim), dtype=torch.int8, device=device)
    s = torch.zeros((2, num_pages, kv_heads, page_size), dtype=torch.float32, device=device)
    ks = (key_smoothing.to(device=device, dtype=torch.float32).contiguous() if key_smoothing is not None
          else torch.ones(head_dim, dtype=torch.float32, device=device))
    return Int8Pages(q, s, ks, 0), Int8Pages(q, s, torch.ones(head_dim, dtype=torch.float32, device=device), 1)


def key_smoothing(k_norm: torch.Tensor) -> torch.Tensor:
    """max(|w_i|, |w_j|) for each rotary pair (i, j = i + D/2), 1 where both are zero
    (src/ops/quant.jl:118-124)."""
    w = k_norm.float().abs()
    half = w.numel() // 2
    c = torch.maximum(w[:half], w[half:2 * half])
    c = torch.where(c > 0, c, torch.ones_like(c))
    return torch.cat([c, c])


def layer_arrays(k: Int8Pages, v: Int8Pages):
    """The layer arrays behind a key/value pair; both must be the halves of one layer
    made by int8_kv_pools (src/ops/quant.jl:131-135)."""
    if not (isinstance(k, Int8Pages) and isinstance(v, Int8Pages) and k.layer_q is v.layer_q
            and k.half == 0 and v.half == 1):
        raise ArgumentError("keys and values must be the halves of one layer's pools (int8_kv_pools)")
    return k.layer_q, k.layer_scale, k.smooth


class Fp8Pages:
    """One half (keys or values) of an 8-bit block layer: e4m3 values with one scale for each block, the rows
    of a page and KV head. `q` [pages][H][P][D] torch.float8_e4m3fn and `scale` [pages][H] f32 (powers of two) are
    views of the layer arrays `layer_q` [2][pages][H][P][D] (uint8 or float8_e4m3fn; keys first) and `layer_scale`
    [2][pages][H]. head_dim 64 or 128, pages of 2^k rows from 16 to 1024. store_kv_ and attention_inputs_
    write them, page by page from the first row on; attention_, paged_attention_ and window_attention_ read them."""

    def __init__(self, layer_q: torch.Tensor, layer_scale: torch.Tensor, half: int):
        if layer_q.dim() != 5 or layer_q.shape[0] != 2 or layer_q.dtype not in (torch.uint8, torch.float8_e4m3fn) \
                or layer_scale.dtype != torch.float32 or layer_scale.shape != layer_q.shape[:3] or half not in (0, 1):
            raise ArgumentError("layer_q must be e4m3 [2][pages][kv_heads][P][D] and layer_scale float32 [2][pages][kv_heads]")
        self.layer_q, self.layer_scale, self.half = layer_q, layer_scale, half
        self.q = layer_q[half].view(torch.float8_e4m3fn)
        self.scale = layer_scale[half]

    @property
    def shape(self):
        return tuple(self.q.shape)

    def size(self, d: Optional[int] = None):
        return self.q.size() if d is None else self.q.size(d)

    def values(self) -> torch.Tensor:
        """What the pages stand for, in Float32."""
        return self.q.float() * self.scale[..., None, None]


def fp8_kv_pools(head_dim: int, page_size: int, kv_heads: int, num_pages: int, device="cuda"):
    """The zeroed key and value Fp8Pages of one layer."""
    q = torch.zeros((2, num_pages, kv_heads, page_size, head_dim), dtype=torch.uint8, device=device)
    s = torch.zeros((2, num_pages, kv_heads), dtype=torch.float32, device=device)
    return Fp8Pages(q, s, 0), Fp8Pages(q, s, 1)


def fp8_layer_arrays(k: Fp8Pages, v: Fp8Pages):
    """The layer arrays behind a key/value pair; both must be the halves of one layer (fp8_kv_pools)."""
    if not (isinstance(k, Fp8Pages) and isinstance(v, Fp8Pages) and k.layer_q.data_ptr() == v.layer_q.data_ptr()
            and k.layer_scale.data_ptr() == v.layer_scale.data_ptr() and k.layer_q.shape == v.layer_q.shape
            and k.half == 0 and v.half == 1):
        raise ArgumentError("keys and values must be the halves of one layer's pools (fp8_kv_pools)")
    return k.layer_q, k.layer_scale


class PagePool:
    """The pages of a cache and the sequences that hold them, on the GPU: what BlockManager and Sequence keep on the
    host. `free` [num_pages] int32 is the stack of free page ids (1-based), `free_count` [1] its height, `tables`
    [sequences][width] int32 the sequences' pages (0: none), `lengths` [sequences] int32 their positions.
    reserve_pages_ and release_pages_ change them in place.

    window, sinks: of the attention over the cache (window_attention_); release_pages_ then gives back the pages that no later
    query sees. `behind` [sequences] int32 counts a sequence's pages up to the first that it still holds past its sinks: where
    it is not given, it is taken from the tables, whose entries of pages that went back before are 0."""

    def __init__(self, free: torch.Tensor, free_count: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor, page_size: int,
                 window: int = 0, sinks: int = 0, behind: Optional[torch.Tensor] = None):
        if any(t.dtype != torch.int32 for t in (free, free_count, tables, lengths)) or free.dim() != 1 or free_count.numel() != 1 \
                or tables.dim() != 2 or lengths.shape != tables.shape[:1]:
            raise ArgumentError("free, free_count, tables and lengths must be int32 [pages], [1], [sequences][width] and [sequences]")
        if any(isinstance(x, bool) or int(x) != x or not low <= x < 1 << 31 for x, low in ((page_size, 1), (window, 0), (sinks, 0))):
            raise ArgumentError("page_size must be a whole number from 1 on, window and sinks from 0 on")
        self.free, self.free_count, self.tables, self.lengths = free, free_count, tables, lengths
        self.page_size, self.window, self.sinks = int(page_size), int(window), int(sinks)
        if behind is not None and (not window or behind.dtype != torch.int32 or behind.shape != lengths.shape):
            raise ArgumentError("behind must be int32 [sequences], of a pool with a window")
        self.behind = self._behind() if window and behind is None else behind
        self.ticket = torch.zeros(1, dtype=torch.int32, device=free.device)

    def _behind(self) -> torch.Tensor:
        first = -(-self.sinks // self.page_size)            # pages of sinks
        none = torch.full_like(self.lengths, first)
        if first >= self.tables.shape[1]:
            return none
        held = self.tables[:, first:] > 0
        # no page held past the sinks: all that the length reaches into went back
        all_back = torch.maximum(none, ((self.lengths.long() + (self.page_size - 1)) // self.page_size).to(torch.int32))
        return torch.where(held.any(1), first + held.int().argmax(1).to(torch.int32), all_back)


def page_pool(num_pages: int, page_size: int, num_seqs: int, max_pages: int, window: int = 0, sinks: int = 0, device="cuda") -> PagePool:
    """A PagePool whose pages are all free, handed out in increasing order as a new BlockManager's, for num_seqs
    sequences of at most max_pages pages."""
    i32 = dict(dtype=torch.int32, device=device)
    return PagePool(torch.arange(num_pages, 0, -1, **i32), torch.full((1,), num_pages, **i32),
                    torch.zeros((num_seqs, max_pages), **i32), torch.zeros(num_seqs, **i32), page_size, window, sinks)


class KeyBounds:
    """Bounds of the keys of a layer's pages, beside its pools of either kind: for each page and KV
    head the keys' largest and smallest element in each dimension as whole multiples of the page's
    power of two. `bounds` [pages][H][2][D] int8 (largest first), `scale` [pages][H] f32;
    update_key_bounds_ writes them, select_pages_ scores pages by them.

    channel: what keys of each dimension are about as large as ([D] or [H][D], positive), rounded here to powers
    of two between 2^-30 and 2^30: keys are divided by them before they are bounded, queries multiplied, so that
    dimensions with large keys do not take the others' precision. Good values are the largest |k| of each dimension over
    sample keys, or key_smoothing(k_norm); None where keys are about alike. Kept as `channel` [H][D] f32 or None."""

    def __init__(self, bounds: torch.Tensor, scale: torch.Tensor, page_size: int, channel: Optional[torch.Tensor] = None):
        if bounds.dtype != torch.int8 or scale.dtype != torch.float32 or bounds.dim() != 4 or bounds.shape[2] != 2 \
                or scale.shape != bounds.shape[:2] or page_size <= 0:
            raise ArgumentError("bounds must be int8 [pages][kv_heads][2][D] and scale float32 [pages][kv_heads]")
        self.bounds, self.scale, self.page_size = bounds, scale, int(page_size)
        self.channel = None if channel is None else _channel(channel, bounds)

    @property
    def shape(self):
        """(pages, kv_heads, page_size, D), as the pools the bounds belong to."""
        pages, H, _, D = self.bounds.shape
        return (pages, H, self.page_size, D)


def _channel(channel: torch.Tensor, bounds: torch.Tensor) -> torch.Tensor:
    """The nearest powers of two (by ratio), [H][D] on the bounds' device."""
    H, D = bounds.shape[1], bounds.shape[3]
    if channel.shape not in ((D,), (H, D)):
        raise ArgumentError("channel must be [D] or [kv_heads][D]")
    c = channel.detach().double().cpu()
    if not bool(((c > 0) & torch.isfinite(c)).all()):
        raise ArgumentError("channel must be positive and finite")
    e = torch.log2(c).round().clamp(-30, 30)
    return torch.exp2(e).float().expand(H, D).contiguous().to(bounds.device)


def key_bounds(head_dim: int, page_size: int, kv_heads: int, num_pages: int, device="cuda",
               channel: Optional[torch.Tensor] = None) -> KeyBounds:
    """The zeroed KeyBounds of one layer."""
    return KeyBounds(torch.zeros((num_pages, kv_heads, 2, head_dim), dtype=torch.int8, device=device),
                     torch.zeros((num_pages, kv_heads), dtype=torch.float32, device=device), page_size, channel)


class PagedKVCache:
    """Key/value pools for every layer and their page allocator (src/kv/paged_cache.jl:18-36).
    quantize=None: pools in `dtype`; "int8": Int8Pages pairs; "fp8": Fp8Pages pairs. bounds=True: a KeyBounds
    for every layer in `bounds`, for attention over chosen pages; bounds_channel: the channel of each layer's."""

    def __init__(self, num_layers: int, head_dim: int, kv_heads: int, num_pages: int,
                 page_size: int = DEFAULT_PAGE_SIZE, dtype=torch.bfloat16, quantize=None,
                 key_smoothing=None, device="cuda", bounds: bool = False, bounds_channel=None):
        self.blocks = BlockManager(num_pages, page_size)
        self.quantize = quantize
        self.bounds = [key_bounds(head_dim, page_size, kv_heads, num_pages, device,
                                  None if bounds_channel is None else bounds_channel[l])
                       for l in range(num_layers)] if bounds else None
        if quantize is None:
            shape = (num_pages, kv_heads, page_size, head_dim)
            self.k = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)]
            self.v = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        elif quantize == "int8":
            pairs = [int8_kv_pools(head_dim, page_size, kv_heads, num_pages,
                                   None if key_smoothing is None else key_smoothing[l], device)
                     for l in range(num_layers)]
            self.k = [p[0] for p in pairs]
            self.v = [p[1] for p in pairs]
        elif quantize == "fp8":
            if bounds:
                raise ArgumentError("page bounds are of dense and INT8 caches")
            pairs = [fp8_kv_pools(head_dim, page_size, kv_heads, num_pages, device) for _ in range(num_layers)]
            self.k = [p[0] for p in pairs]
            self.v = [p[1] for p in pairs]
        else:
            raise ArgumentError(f"unsupported KV cache quantization {quantize} (only 'int8' and 'fp8')")

    def page_size(self) -> int:
        return self.blocks.page_size

    def num_pages(self) -> int:
        return self.blocks.num_pages

    def new_sequence(self) -> Sequence:
        return Sequence()


def bytes_per_token(num_layers: int, kv_heads: int, head_dim: int, elt_bytes: int = 2,
                    quantize=None) -> int:
    """Cache bytes per cached position (src/kv/paged_cache.jl:43-47), without KeyBounds (2 head_dim + 4
    bytes a page, layer and KV head) and the scales of Fp8Pages (8 bytes a page, layer and KV head)."""
    if quantize == "fp8":
        return 2 * num_layers * kv_heads * head_dim
    if quantize == "int8":
        return 2 * num_layers * kv_heads * (head_dim + 4)
    return 2 * num_layers * kv_heads * head_dim * elt_bytes
