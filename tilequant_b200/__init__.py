"""tilequant_b200 -- B200 (sm_100a) mixed-precision 64x64 tile GEMM path.

Drop-in for the Triton path of HanzhiZhang-Ulrica/TileQuant (src/kernels/triton/,
src/kernels/quant_utils.py, src/kernels/pack.py, src/models/mixed_linear.py): the
same Python API over hand-written CUDA kernels reached through the C ABI in
``include/tilequant_b200.h`` (``libtilequant_b200.so``).
"""

from .gemm import gemm_int8_partials, gemm_mixed_fused_quant, gemm_mixed_rows_splitk, select_split_k
from .mixed_linear import (
    MixedLinear,
    MixedLinearGroup,
    MixedLinearSlice,
    fuse_projection_groups,
    reset_projection_groups,
)
from .pack import Pack, concat_packs_along_rows, is_row_major_pack, pack_weight, pack_weight_from_tile_ids
from .paged_cache import KVPages, PagePool, StepPlan, attn_paged, cache_write, plan_step, read_pages, release_requests
from .peer import PeerExchange, gemm_mixed_peer_sum
from .quant_utils import (
    activation_tile_absmax_scales,
    pad_to_multiple,
    quantize_activation_tile_absmax,
    quantize_activation_tile_with_scales,
)
from .sampling import Sampling, sample_pick, sample_tokens

__all__ = [
    "KVPages", "MixedLinear", "MixedLinearGroup", "MixedLinearSlice", "Pack", "PagePool", "PeerExchange", "Sampling", "StepPlan",
    "activation_tile_absmax_scales", "attn_paged", "cache_write", "concat_packs_along_rows", "fuse_projection_groups",
    "gemm_int8_partials", "gemm_mixed_fused_quant", "gemm_mixed_peer_sum", "gemm_mixed_rows_splitk",
    "is_row_major_pack", "pack_weight", "pack_weight_from_tile_ids", "pad_to_multiple", "plan_step",
    "quantize_activation_tile_absmax", "quantize_activation_tile_with_scales", "read_pages", "release_requests",
    "reset_projection_groups", "sample_pick", "sample_tokens", "select_split_k",
]
