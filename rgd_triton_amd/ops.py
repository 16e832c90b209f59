"""torch.nn.Module API: the same classes, constructor arguments, forward signatures, parameter names
and cache behaviour as the reference's rgd_triton/ops.py, backed by the gfx950 HIP kernels.

Reference: rgd_triton/ops.py:12-249.  Two defects of the reference are not reproduced: its
FlashAttention module imports a module that does not exist (ops.py:37), and its RoPE module rotates
query and key in place because the cache object lands in the in_place argument
(rope/head_rope_cached.py:326-327); here FlashAttention works and RoPE is out of place.

Beyond the reference: the learned relative position bias that FlashAttention takes (RelativePositionBias), and what the same
model needs to run token by token (RoPECacheAppend / FusedLNRoPECacheAppend, PagedDecodeAttention).
"""
import torch
import torch.nn as nn

from . import functional as F_

__all__ = ["CachableModule", "FlashAttention", "L2Normalize", "FusedL2Normalize2", "FusedHeadLayerNorm",
           "FusedRMSNorm", "FusedRMSNorm2", "RoPE", "FusedLNRoPE", "RelativePositionBias", "RoPECacheAppend",
           "FusedLNRoPECacheAppend", "PagedDecodeAttention"]


class CachableModule(nn.Module):
    """nn.Module with a per-module launch cache: an object whose attributes are the given field
    names, all None until the first launch (ops.py:12-24).  enable_cache(False) sets it to None."""

    def __init__(self, cache_fields=None):
        super().__init__()
        self._cache_fields = cache_fields or []
        self.cache = self._make_cache()

    def _make_cache(self):
        fields = {name: None for name in self._cache_fields}
        return type("DynamicCache", (), fields)()

    def enable_cache(self, enable=True):
        self.cache = self._make_cache() if enable else None


class FlashAttention(CachableModule):
    def __init__(self):
        super().__init__(cache_fields=("fwd", "bwd_odot", "bwd"))
        self._triton_fn = F_.flash_attn_func

    def forward(self, q, k, v, bias=None, causal=False, softmax_scale=None):
        return self._triton_fn(q=q, k=k, v=v, bias=bias, causal=causal, softmax_scale=softmax_scale,
                               kernel_cache=self.cache)


class L2Normalize(CachableModule):
    def __init__(self):
        super().__init__(cache_fields=("fwd", "bwd"))
        self._triton_fn = F_.triton_norm_func_fn

    def forward(self, x, eps=1e-6):
        return self._triton_fn(x=x, norm_eps=eps, kernel_cache=self.cache)


class FusedL2Normalize2(CachableModule):
    def __init__(self):
        super().__init__(cache_fields=("fwd", "bwd"))
        self._triton_fn = F_.triton_fused_norm_func_fn

    def forward(self, x1, x2, eps=1e-6):
        return self._triton_fn(x1=x1, x2=x2, norm_eps=eps, kernel_cache=self.cache)


class FusedHeadLayerNorm(CachableModule):
    def __init__(self):
        super().__init__(cache_fields=("fwd", "bwd"))
        self._triton_fn = F_.triton_fused_ln_func_fn

    def forward(self, query, key, heads_second=True, eps=1e-6):
        return self._triton_fn(query=query, key=key, heads_second=heads_second, norm_eps=eps,
                               kernel_cache=self.cache)


class FusedRMSNorm(CachableModule):
    def __init__(self, normalized_shape, eps=1e-6, elementwise_affine=True, device=None, dtype=None):
        super().__init__(cache_fields=("fwd", "bwd", "bwd_dw"))
        assert isinstance(normalized_shape, int), "Fused RMSNorm only supports int dims"
        self.normalized_shape = (normalized_shape,)
        self.eps = eps
        self.elementwise_affine = elementwise_affine
        if self.elementwise_affine:
            factory_kwargs = {"device": device, "dtype": dtype}
            self.weight = nn.Parameter(torch.empty(self.normalized_shape, **factory_kwargs))
        else:
            self.register_parameter("weight", None)
        self.reset_parameters()
        self._triton_fn = F_.triton_rms_func_fn

    def reset_parameters(self) -> None:
        if self.elementwise_affine:
            torch.nn.init.ones_(self.weight)

    def forward(self, x, weight=None):
        if self.elementwise_affine:
            weight = self.weight  # the module's own weight wins
        else:
            assert weight is not None, "Must pass in a weight tensor if not using element-wise affine"
        return self._triton_fn(x=x, w=weight, norm_eps=self.eps, kernel_cache=self.cache)


class FusedRMSNorm2(CachableModule):
    def __init__(self, normalized_shape, eps=1e-6, elementwise_affine=True, device=None, dtype=None):
        super().__init__(cache_fields=("fwd", "bwd", "bwd_dw"))
        assert isinstance(normalized_shape, (tuple, list)) and len(normalized_shape) == 2, \
            "Fused RMSNorm2 requires 2 int dims"
        self.normalized_shape1 = (normalized_shape[0],)
        self.normalized_shape2 = (normalized_shape[1],)
        self.eps = eps
        self.elementwise_affine = elementwise_affine
        if self.elementwise_affine:
            factory_kwargs = {"device": device, "dtype": dtype}
            self.weight1 = nn.Parameter(torch.empty(self.normalized_shape1, **factory_kwargs))
            self.weight2 = nn.Parameter(torch.empty(self.normalized_shape2, **factory_kwargs))
        else:
            self.register_parameter("weight1", None)
            self.register_parameter("weight2", None)
        self.reset_parameters()
        self._triton_fn = F_.triton_fused_rms_func_fn

    def reset_parameters(self) -> None:
        if self.elementwise_affine:
            torch.nn.init.ones_(self.weight1)
            torch.nn.init.ones_(self.weight2)

    def forward(self, x1, x2, weight1=None, weight2=None):
        if self.elementwise_affine:
            weight1 = self.weight1
            weight2 = self.weight2
        else:
            assert (weight1 is not None) and (weight2 is not None), \
                "Must pass in a weight tensor if not using element-wise affine"
        return self._triton_fn(x1=x1, x2=x2, w1=weight1, w2=weight2, norm_eps=self.eps, kernel_cache=self.cache)


class RoPE(CachableModule):
    def __init__(self):
        super().__init__(cache_fields=("fwd", "bwd"))
        self._triton_fn = F_.triton_rope_fn

    def forward(self, query, key, pos_emb, seq_cutoff=None, heads_second=True):
        return self._triton_fn(query=query, key=key, pos_emb=pos_emb, seq_cutoff=seq_cutoff,
                               heads_second=heads_second, kernel_cache=self.cache)


class FusedLNRoPE(CachableModule):
    def __init__(self):
        super().__init__(cache_fields=("fwd", "bwd"))
        self._triton_fn = F_.triton_fused_ln_rope_fn

    def forward(self, query, key, pos_emb, seq_cutoff=None, heads_second=True, eps=1e-6):
        return self._triton_fn(query=query, key=key, pos_emb=pos_emb, seq_cutoff=seq_cutoff,
                               heads_second=heads_second, norm_eps=eps, kernel_cache=self.cache)


class RelativePositionBias(CachableModule):
    """Learned relative position bias: forward gives the (1, nheads, seqlen_q, seqlen_k) bias that FlashAttention takes."""

    def __init__(self, num_buckets, nheads, max_distance=128, bidirectional=True, device=None, dtype=None):
        super().__init__(cache_fields=("fwd", "bwd"))
        self.max_distance = max_distance
        self.bidirectional = bool(bidirectional)
        F_.relative_ranges(num_buckets, max_distance, self.bidirectional)  # refuses impossible buckets
        self.weight = nn.Parameter(torch.empty((num_buckets, nheads), device=device, dtype=dtype))
        self.reset_parameters()
        self._fn = F_.relative_position_bias_fn

    def reset_parameters(self) -> None:
        torch.nn.init.zeros_(self.weight)

    def forward(self, seqlen_q, seqlen_k, q_offset=0, dtype=None):
        return self._fn(self.weight, seqlen_q, seqlen_k, max_distance=self.max_distance, bidirectional=self.bidirectional,
                        q_offset=q_offset, dtype=dtype, kernel_cache=self.cache)


class RoPECacheAppend(CachableModule):
    def __init__(self):
        super().__init__(cache_fields=("fwd",))
        self._fn = F_.rope_cache_append_fn

    def forward(self, query, key, value, pos_emb, k_cache, v_cache, page_table, cache_lens, new_lens=None, seq_cutoff=None,
                heads_second=True):
        return self._fn(query, key, value, pos_emb, k_cache, v_cache, page_table, cache_lens, new_lens=new_lens,
                        seq_cutoff=seq_cutoff, heads_second=heads_second, kernel_cache=self.cache)


class FusedLNRoPECacheAppend(CachableModule):
    def __init__(self):
        super().__init__(cache_fields=("fwd",))
        self._fn = F_.rope_cache_append_fn

    def forward(self, query, key, value, pos_emb, k_cache, v_cache, page_table, cache_lens, new_lens=None, seq_cutoff=None,
                heads_second=True, eps=1e-6):
        return self._fn(query, key, value, pos_emb, k_cache, v_cache, page_table, cache_lens, new_lens=new_lens,
                        seq_cutoff=seq_cutoff, heads_second=heads_second, norm_eps=eps, kernel_cache=self.cache)


class PagedDecodeAttention(CachableModule):
    def __init__(self):
        super().__init__(cache_fields=("fwd",))
        self._fn = F_.paged_decode_attn_func

    def forward(self, q, k_cache, v_cache, page_table, seq_lens, rel_bias=None, softmax_scale=None):
        """rel_bias: the RelativePositionBias the model was trained with, or None."""
        rel = {} if rel_bias is None else dict(rel_weight=rel_bias.weight, max_distance=rel_bias.max_distance,
                                               bidirectional=rel_bias.bidirectional)
        return self._fn(q, k_cache, v_cache, page_table, seq_lens, softmax_scale=softmax_scale, kernel_cache=self.cache, **rel)
