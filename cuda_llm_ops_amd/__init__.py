"""MI355X-native flash grouped-query attention (decode incl. paged/fp8/int8 KV caches, their writing, eviction and forking, causal, sliding-window, MLA and sparse-index prefill, the causal, sliding-window and MLA prefill backward, and norm and rotation of queries and keys).

The kernels live in libfgqa.so (HIP, gfx950); ``flash_gqa`` is the Python host
interface over its C ABI (include/fgqa.h), ``kv_cache`` that of the paged
cache's operators (include/fgqa_kv.h, include/fgqa_pages.h) and ``qk_rope`` that of the norm and rotation
of queries and keys (include/fgqa_rope.h).
"""
from ._lib import FgqaError, LIB_PATH, lib, native, status_string  # noqa: F401
from .flash_gqa import (  # noqa: F401
    backward_workspace_bytes,
    decode_flash_gqa_bshd,
    decode_flash_gqa_paged,
    decode_workspace_bytes,
    flash_gqa_backward_bshd,
    flash_gqa_forward_bshd,
    launch_decode_flash_gqa_bf16_kernel,
    launch_flash_gqa_backward_bf16_kernel,
    launch_flash_gqa_forward_bf16_kernel,
    launch_flash_swa_backward_bf16_kernel,
    launch_flash_swa_forward_bf16_kernel,
    launch_flash_mla_backward_bf16_kernel,
    launch_flash_mla_forward_bf16_kernel,
    launch_flash_sgqa_forward_bf16_kernel,
    flash_sgqa_forward_bshd,
    prepare_sparse_prefill,
    PREFILL_HEAD_DIMS,
    BACKWARD_HEAD_DIMS,
    paged_decode_workspace_bytes,
    prepare_backward,
    prepare_decode,
    prepare_decode_paged,
    prefill_kernel_choice,
    prefill_kernel_name,
    prepare_prefill,
    PreparedLaunch,
)
from .kv_cache import (  # noqa: F401
    accumulate_kv_weights_paged,
    append_kv_paged,
    compact_kv_paged,
    decode_flash_gqa_paged_shared,
    evict_kv_paged,
    fork_kv_paged,
)
from .qk_rope import (  # noqa: F401
    qk_norm_rope,
    qk_norm_rope_backward,
)

__version__ = "0.1.0"
