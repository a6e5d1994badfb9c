"""tileinfer_hip: TileInfer.jl's paged flash-attention path on MI355X (gfx950).

Host-side mirror of the reference's op interface (src/ops/interface.jl) and KV layout
(src/kv/), driving the HIP kernels of libtileinfer_hip.so through its C ABI.
"""
from ._lib import (ArgumentError, TileInferError, WorkspaceError, TI_PATH_AUTO, TI_PATH_DECODE,
                   TI_PATH_PREFILL, TI_PATH_PREFILL_STAGED, TI_PATH_PREFILL_DIRECT,
                   TI_PATH_PREFILL_PINGPONG, TI_PATH_PREFILL_PAIRED, TI_PATH_PREFILL_PAIRED16, EXPORTS, LIB_PATH, load as load_library)
from .backend import (HipBackend, attention, attention_, attention_inputs_, attention_workspace,
                      has_kernel, kv_cache_struct, paged_attention_, release_pages_, reserve_pages_, rmsnorm, rmsnorm_, rope, rope_, select_pages,
                      select_pages_, select_pages_workspace, sparse_attention, sparse_attention_,
                      sparse_attention_workspace, store_kv_, supports_graphs, update_key_bounds_, verify_draft,
                      verify_draft_, verify_draft_workspace, window_attention, window_attention_, window_attention_workspace, workspace_bytes)
from .kv import (DEFAULT_PAGE_SIZE, BlockManager, Fp8Pages, Int8Pages, KeyBounds, OutOfPagesError, PagedKVCache, PagePool,
                 Sequence, bytes_per_token, fp8_kv_pools, fp8_layer_arrays, int8_kv_pools, key_bounds, key_smoothing,
                 layer_arrays, page_pool, release, reserve, slots, truncate)
from .rope import Llama3RopeScaling, RotaryTable, inverse_frequencies, llama3_scaled

__version__ = "0.1.0"
