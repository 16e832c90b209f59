"""MI355X (gfx950) implementation of the rgd-triton operator set: hand-written HIP kernels behind the
reference's torch.nn.Module / autograd.Function API.  No Triton, no CPU fallback."""
from .ops import (CachableModule, FlashAttention, FusedHeadLayerNorm, FusedL2Normalize2, FusedLNRoPE, FusedLNRoPECacheAppend,
                  FusedRMSNorm, FusedRMSNorm2, L2Normalize, PagedDecodeAttention, RelativePositionBias, RoPE, RoPECacheAppend)
from .functional import (clear_bias_classes_cache, flash_attn_func, paged_decode_attn_func, relative_position_bias_fn,
                         rope_cache_append_fn, set_attention_backward, triton_fused_ln_func_fn, triton_fused_ln_rope_fn, triton_fused_norm_func_fn,
                         triton_fused_rms_func_fn, triton_norm_func_fn, triton_rms_func_fn, triton_rope_fn)

__version__ = "0.1.0"
