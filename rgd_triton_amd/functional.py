"""torch.autograd.Function layer: the same functions, argument order and error behaviour as the
reference's `*_cached.py` modules, launching the gfx950 HIP kernels of librgd_hip.so through ctypes.

Reference entry points mirrored here (paths relative to rgd_triton/triton/):
    flash_attn_func            flash_attn/flash_attn_triton_cached.py:1079-1133
    triton_rms_func_fn         normalization/rmsnorm_cached.py:572-629
    triton_fused_rms_func_fn   normalization/fused_rmsnorm_cached.py:725-802
    triton_fused_ln_func_fn    normalization/head_layernorm_cached.py:416-457
    triton_norm_func_fn        normalization/l2normalize_cached.py:402-437
    triton_fused_norm_func_fn  normalization/fused_l2normalize_cached.py:464-507
    triton_rope_fn             rope/head_rope_cached.py:277-327
    triton_fused_ln_rope_fn    rope/fused_ln_rope_cached.py:649-696

Differences from the reference, all deliberate:
  * row statistics (rrms, mean/rstd, rlen) are recomputed in the backward instead of being saved;
  * dw of a shared RMSNorm weight is reduced in fp32 inside the kernel and rounded once;
  * `kernel_cache` objects keep their field names; a field holds the set of validated call
    signatures instead of a compiled-kernel handle, so a change of shape, dtype or bias kind after
    the first call can never reuse a stale specialisation.
"""
import ctypes
import functools
import math
import os

import torch
from torch.autograd import forward_ad

from . import _hip
from ._hip import t3, t4

__all__ = [
    "flash_attn_func", "triton_rms_func_fn", "triton_fused_rms_func_fn", "triton_fused_ln_func_fn",
    "triton_norm_func_fn", "triton_fused_norm_func_fn", "triton_rope_fn", "triton_fused_ln_rope_fn",
    "set_attention_backward", "rope_cache_append_fn", "paged_decode_attn_func", "relative_position_bias_fn",
]

_FLOATS = (torch.float16, torch.bfloat16, torch.float32)


def _lastdim_contig(*ts):
    return [t if (t is None or t.stride(-1) == 1) else t.contiguous() for t in ts]


def _seen(cache, field, key):
    """True if a call with this signature has passed every check with this cache object."""
    if cache is None:
        return False
    plans = getattr(cache, field, None)
    return plans is not None and key in plans


_MOST_SIGNATURES = 1024  # of a cache field: with more (prompts of every length) it starts anew, a check costs microseconds


def _remember(cache, field, key):
    """Keeps the signature of a call that has passed every check: a refused one has to be refused again."""
    if cache is None:
        return
    plans = getattr(cache, field, None)
    if plans is None:
        plans = set()
        setattr(cache, field, plans)
    elif len(plans) >= _MOST_SIGNATURES:
        plans.clear()
    plans.add(key)


def _no_capture(what):
    """Every backward starts here.  Recording an autograd backward of these operators into a HIP graph ended in a
    crash inside the runtime's end-of-capture call on the one occasion it was tried (the backward nodes run on
    autograd's worker thread), and its cause was never established, so the combination is refused with an error
    instead: record the backward through direct C-ABI calls (tests/test_graph_capture.py does) or keep autograd
    outside the graph.  The forward functions can be captured."""
    if torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: an autograd backward cannot be recorded into a HIP graph with this package; "
                           "record direct calls of the C ABI instead")


def _no_tangent(what, *ts):
    """For what goes round autograd: a forward-mode derivative is refused, as autograd functions without one refuse it."""
    if forward_ad._current_level >= 0:
        for t in ts:
            assert t is None or forward_ad.unpack_dual(t).tangent is None, f"{what} has no forward-mode derivative"


def _sig(*ts):
    """What the checks of a call look at: its tensors' sizes, types, strides and the device of every one of them."""
    return tuple((t.shape, t.dtype, t.stride(), t.get_device()) if t is not None else None for t in ts)


# ----------------------------------------------------------------------------------------------
# RMSNorm
# ----------------------------------------------------------------------------------------------


def _w_layout(w, x):
    """Weight broadcast rule of the reference (rmsnorm_cached.py:582-589): returns (shared, stride_b)."""
    if w.ndim == 1:
        assert w.shape[0] == x.shape[-1], f"{x.shape=}, {w.shape=}"
        return True, 0
    assert w.ndim == 3 and w.shape[1] == 1 and w.shape[2] == x.shape[-1], f"{x.shape=}, {w.shape=}"
    if w.shape[0] == 1:
        return True, 0
    assert w.shape[0] == x.shape[0], f"{x.shape=}, {w.shape=}"
    return False, w.stride(0)


def _check_rows(x):
    assert x.ndim == 3, f"{x.shape=}"
    assert x.dtype in _FLOATS, "Only support fp16, bf16, and fp32"
    assert x.is_cuda, "rgd_triton_amd operators run on the GPU only"


def _rms_scratch(x1, x2):
    B = x1.shape[0]
    T2, C2 = (x2.shape[1], x2.shape[2]) if x2 is not None else (0, 0)
    nbytes = _hip.lib().rgd_rms_bwd_workspace(B, x1.shape[1], x1.shape[2], T2, C2)
    return _hip.workspace(x1.device, nbytes), nbytes


class RMS_Func(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, norm_eps=1e-6, kernel_cache=None):
        x, w = _lastdim_contig(x, w)
        key = _sig(x, w)
        if not _seen(kernel_cache, "fwd", key):
            _check_rows(x)
            assert w.is_cuda and w.dtype in _FLOATS, "Only support fp16, bf16, and fp32"
            _remember(kernel_cache, "fwd", key)
        shared, w_sb = _w_layout(w, x)
        B, T, C = x.shape
        y = torch.empty_like(x)
        lib = _hip.lib()
        _hip.check(lib.rgd_rms_fwd(B, T, C, t3(x), t3(w, w_sb), t3(y), _hip.dtype_code(x.dtype),
                                   _hip.dtype_code(w.dtype), float(norm_eps), _hip.stream_ptr(x.device)), "rgd_rms_fwd")
        ctx.kernel_cache = kernel_cache
        ctx.save_for_backward(x, w)
        ctx.norm_eps = float(norm_eps)
        ctx.w_layout = (shared, w_sb)
        return y

    @staticmethod
    def backward(ctx, dy):
        _no_capture("RMS_Func.backward")
        (dy,) = _lastdim_contig(dy)
        x, w = ctx.saved_tensors
        shared, w_sb = ctx.w_layout
        B, T, C = x.shape
        _remember(ctx.kernel_cache, "bwd", _sig(x, w, dy))
        _remember(ctx.kernel_cache, "bwd_dw", _sig(w))
        dx = torch.empty_like(x)
        dw = torch.empty(w.shape, dtype=w.dtype, device=w.device)
        if B * T == 0:
            dw.zero_()
            return dx, dw, None, None
        wbuf, wsz = _rms_scratch(x, None)
        lib = _hip.lib()
        _hip.check(lib.rgd_rms_bwd(B, T, C, t3(dy), t3(x), t3(w, w_sb), t3(dx), t3(dw, 0 if shared else dw.stride(0)),
                                   int(shared), _hip.dtype_code(x.dtype), _hip.dtype_code(w.dtype), ctx.norm_eps,
                                   wbuf.data_ptr(), wsz, _hip.stream_ptr(x.device)), "rgd_rms_bwd")
        return dx, dw, None, None


def triton_rms_func_fn(x, w, norm_eps=1e-6, kernel_cache=None):
    return RMS_Func.apply(x, w, norm_eps, kernel_cache)


class Fused_RMS_Func(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x1, x2, w1, w2, norm_eps=1e-6, kernel_cache=None):
        x1, x2, w1, w2 = _lastdim_contig(x1, x2, w1, w2)
        key = _sig(x1, x2, w1, w2)
        if not _seen(kernel_cache, "fwd", key):
            _check_rows(x1)
            _check_rows(x2)
            assert x1.dtype == x2.dtype, "All tensors must have the same type"
            assert x1.shape[0] == x2.shape[0], f"{x1.shape=}, {x2.shape=}"
            assert w1.is_cuda and w2.is_cuda and w1.dtype in _FLOATS and w2.dtype in _FLOATS
            _remember(kernel_cache, "fwd", key)
        l1, l2 = _w_layout(w1, x1), _w_layout(w2, x2)
        B, T1, C1 = x1.shape
        _, T2, C2 = x2.shape
        y1, y2 = torch.empty_like(x1), torch.empty_like(x2)
        lib = _hip.lib()
        _hip.check(lib.rgd_fused_rms_fwd(B, T1, C1, T2, C2, t3(x1), t3(w1, l1[1]), t3(y1), t3(x2), t3(w2, l2[1]), t3(y2),
                                         _hip.dtype_code(x1.dtype), _hip.dtype_code(w1.dtype), _hip.dtype_code(w2.dtype),
                                         float(norm_eps), _hip.stream_ptr(x1.device)), "rgd_fused_rms_fwd")
        ctx.kernel_cache = kernel_cache
        ctx.save_for_backward(x1, x2, w1, w2)
        ctx.norm_eps = float(norm_eps)
        ctx.layouts = (l1, l2)
        return y1, y2

    @staticmethod
    def backward(ctx, dy1, dy2):
        _no_capture("Fused_RMS_Func.backward")
        dy1, dy2 = _lastdim_contig(dy1, dy2)
        x1, x2, w1, w2 = ctx.saved_tensors
        (s1, sb1), (s2, sb2) = ctx.layouts
        B, T1, C1 = x1.shape
        _, T2, C2 = x2.shape
        _remember(ctx.kernel_cache, "bwd", _sig(x1, x2, w1, w2, dy1, dy2))
        _remember(ctx.kernel_cache, "bwd_dw", _sig(w1, w2))
        dx1, dx2 = torch.empty_like(x1), torch.empty_like(x2)
        dw1 = torch.empty(w1.shape, dtype=w1.dtype, device=w1.device)
        dw2 = torch.empty(w2.shape, dtype=w2.dtype, device=w2.device)
        if B * T1 == 0:
            dw1.zero_()
        if B * T2 == 0:
            dw2.zero_()
        wbuf, wsz = _rms_scratch(x1, x2)
        lib = _hip.lib()
        _hip.check(lib.rgd_fused_rms_bwd(
            B, T1, C1, T2, C2,
            t3(dy1), t3(x1), t3(w1, sb1), t3(dx1), t3(dw1, 0 if s1 else dw1.stride(0)), int(s1),
            t3(dy2), t3(x2), t3(w2, sb2), t3(dx2), t3(dw2, 0 if s2 else dw2.stride(0)), int(s2),
            _hip.dtype_code(x1.dtype), _hip.dtype_code(w1.dtype), _hip.dtype_code(w2.dtype), ctx.norm_eps,
            wbuf.data_ptr(), wsz, _hip.stream_ptr(x1.device)), "rgd_fused_rms_bwd")
        return dx1, dx2, dw1, dw2, None, None


def triton_fused_rms_func_fn(x1, x2, w1, w2, norm_eps=1e-6, kernel_cache=None):
    return Fused_RMS_Func.apply(x1, x2, w1, w2, norm_eps, kernel_cache)


# ----------------------------------------------------------------------------------------------
# L2 normalize
# ----------------------------------------------------------------------------------------------


class Norm_Func(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, norm_eps=1e-6, use_ptx=False, kernel_cache=None):
        (x,) = _lastdim_contig(x)
        key = _sig(x)
        if not _seen(kernel_cache, "fwd", key):
            _check_rows(x)
            _remember(kernel_cache, "fwd", key)
        B, T, C = x.shape
        y = torch.empty_like(x)
        lib = _hip.lib()
        _hip.check(lib.rgd_l2_fwd(B, T, C, t3(x), t3(y), _hip.dtype_code(x.dtype), float(norm_eps),
                                  _hip.stream_ptr(x.device)), "rgd_l2_fwd")
        ctx.kernel_cache = kernel_cache
        ctx.save_for_backward(x)
        ctx.norm_eps = float(norm_eps)
        return y

    @staticmethod
    def backward(ctx, dy):
        _no_capture("Norm_Func.backward")
        (dy,) = _lastdim_contig(dy)
        (x,) = ctx.saved_tensors
        B, T, C = x.shape
        _remember(ctx.kernel_cache, "bwd", _sig(x, dy))
        dx = torch.empty_like(x)
        lib = _hip.lib()
        _hip.check(lib.rgd_l2_bwd(B, T, C, t3(dy), t3(x), t3(dx), _hip.dtype_code(x.dtype), ctx.norm_eps,
                                  _hip.stream_ptr(x.device)), "rgd_l2_bwd")
        return dx, None, None, None


def triton_norm_func_fn(x, norm_eps=1e-6, use_ptx=False, kernel_cache=None):
    # use_ptx selected an NVIDIA inline-PTX reciprocal in the reference
    # (l2normalize_cached.py:79-98); it has no meaning here and is ignored
    return Norm_Func.apply(x, norm_eps, use_ptx, kernel_cache)


class Fused_Norm_Func(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x1, x2, norm_eps=1e-6, kernel_cache=None):
        x1, x2 = _lastdim_contig(x1, x2)
        key = _sig(x1, x2)
        if not _seen(kernel_cache, "fwd", key):
            _check_rows(x1)
            _check_rows(x2)
            assert x1.dtype == x2.dtype, "All tensors must have the same type"
            assert x1.shape[0] == x2.shape[0], f"{x1.shape=}, {x2.shape=}"
            _remember(kernel_cache, "fwd", key)
        B, T1, C1 = x1.shape
        _, T2, C2 = x2.shape
        y1, y2 = torch.empty_like(x1), torch.empty_like(x2)
        lib = _hip.lib()
        _hip.check(lib.rgd_fused_l2_fwd(B, T1, C1, T2, C2, t3(x1), t3(y1), t3(x2), t3(y2), _hip.dtype_code(x1.dtype),
                                        float(norm_eps), _hip.stream_ptr(x1.device)), "rgd_fused_l2_fwd")
        ctx.kernel_cache = kernel_cache
        ctx.save_for_backward(x1, x2)
        ctx.norm_eps = float(norm_eps)
        return y1, y2

    @staticmethod
    def backward(ctx, dy1, dy2):
        _no_capture("Fused_Norm_Func.backward")
        dy1, dy2 = _lastdim_contig(dy1, dy2)
        x1, x2 = ctx.saved_tensors
        B, T1, C1 = x1.shape
        _, T2, C2 = x2.shape
        _remember(ctx.kernel_cache, "bwd", _sig(x1, x2, dy1, dy2))
        dx1, dx2 = torch.empty_like(x1), torch.empty_like(x2)
        lib = _hip.lib()
        _hip.check(lib.rgd_fused_l2_bwd(B, T1, C1, T2, C2, t3(dy1), t3(x1), t3(dx1), t3(dy2), t3(x2), t3(dx2),
                                        _hip.dtype_code(x1.dtype), ctx.norm_eps, _hip.stream_ptr(x1.device)),
                   "rgd_fused_l2_bwd")
        return dx1, dx2, None, None


def triton_fused_norm_func_fn(x1, x2, norm_eps=1e-6, kernel_cache=None):
    return Fused_Norm_Func.apply(x1, x2, norm_eps, kernel_cache)


# ----------------------------------------------------------------------------------------------
# per-head operators on (query, key)
# ----------------------------------------------------------------------------------------------


def _qk_dims(q, k, heads_second, max_d, what):
    assert q.ndim == k.ndim == 4
    assert q.dtype == k.dtype, "All tensors must have the same type"
    assert q.dtype in _FLOATS, "Only support fp16, bf16, and fp32"
    assert q.is_cuda and k.is_cuda, "rgd_triton_amd operators run on the GPU only"
    if heads_second:
        bq, hq, tq, dq = q.shape
        bk, hk, tk, dk = k.shape
    else:
        bq, tq, hq, dq = q.shape
        bk, tk, hk, dk = k.shape
    assert (bq, hq, dq) == (bk, hk, dk)
    assert dq <= max_d, f"Only supports head dimensions up to {max_d}"
    return bq, hq, tq, tk, dq


def _cutoffs(seq_cutoff, tq, tk):
    # head_rope_cached.py:193-201
    if seq_cutoff is None:
        return tq, tk
    if isinstance(seq_cutoff, (tuple, list)):
        return int(seq_cutoff[0]), int(seq_cutoff[1])
    return int(seq_cutoff), int(seq_cutoff)


def _table_for(pos_emb, x):
    """A rotary table the kernels can read next to tensors of x.dtype: same dtype, or fp32."""
    if pos_emb.dtype == x.dtype or pos_emb.dtype == torch.float32:
        return pos_emb
    return pos_emb.float()  # e.g. an fp16 table with bf16 tensors: exact upcast, tiny tensor


def _pos_emb_args(pos_emb, tq, tk):
    """pos_emb (2, P, R) -> C arguments.  The kernels read a table in the tensors' dtype or in fp32; the
    caller has already converted any other combination (see _table_for)."""
    assert pos_emb.ndim == 3 and pos_emb.shape[0] == 2, f"{pos_emb.shape=}"
    assert pos_emb.is_cuda and pos_emb.dtype in _FLOATS
    _, P, R = pos_emb.shape
    assert tq < P
    assert tk < P
    return (ctypes.c_void_p(pos_emb.data_ptr()), P, R, pos_emb.stride(0), pos_emb.stride(1),
            _hip.dtype_code(pos_emb.dtype))


class Fused_LNQK_Func(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, heads_second=True, norm_eps=1e-6, kernel_cache=None):
        q, k = _lastdim_contig(q, k)
        B, H, Tq, Tk, D = _qk_dims(q, k, heads_second, 256, "head LayerNorm")
        _remember(kernel_cache, "fwd", _sig(q, k) + (heads_second,))
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        lib = _hip.lib()
        _hip.check(lib.rgd_ln_qk_fwd(B, H, Tq, Tk, D, t4(q, heads_second), t4(k, heads_second), t4(qo, heads_second),
                                     t4(ko, heads_second), _hip.dtype_code(q.dtype), float(norm_eps),
                                     _hip.stream_ptr(q.device)), "rgd_ln_qk_fwd")
        ctx.kernel_cache = kernel_cache
        ctx.save_for_backward(q, k)
        ctx.heads_second = heads_second
        ctx.norm_eps = float(norm_eps)
        ctx.dims = (B, H, Tq, Tk, D)
        return qo, ko

    @staticmethod
    def backward(ctx, doq, dok):
        _no_capture("Fused_LNQK_Func.backward")
        q, k = ctx.saved_tensors
        hs = ctx.heads_second
        doq, dok = _lastdim_contig(doq, dok)
        _remember(ctx.kernel_cache, "bwd", _sig(q, k, doq, dok) + (hs,))
        B, H, Tq, Tk, D = ctx.dims
        dq, dk = torch.empty_like(q), torch.empty_like(k)
        lib = _hip.lib()
        _hip.check(lib.rgd_ln_qk_bwd(B, H, Tq, Tk, D, t4(q, hs), t4(k, hs), t4(doq, hs), t4(dok, hs), t4(dq, hs),
                                     t4(dk, hs), _hip.dtype_code(q.dtype), ctx.norm_eps, _hip.stream_ptr(q.device)),
                   "rgd_ln_qk_bwd")
        return dq, dk, None, None, None


def triton_fused_ln_func_fn(query, key, heads_second=True, norm_eps=1e-6, kernel_cache=None):
    return Fused_LNQK_Func.apply(query, key, heads_second, norm_eps, kernel_cache)


class CombinedRoPEFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos_emb, seq_cutoff=None, heads_second=True, in_place=False, kernel_cache=None):
        if in_place:
            assert q.stride(-1) == 1 and k.stride(-1) == 1, "in_place RoPE needs unit-stride head dims"
        q, k, pos_emb = _lastdim_contig(q, k, _table_for(pos_emb, q))
        B, H, Tq, Tk, D = _qk_dims(q, k, heads_second, 128, "RoPE")
        pe = _pos_emb_args(pos_emb, Tq, Tk)
        _remember(kernel_cache, "fwd", _sig(q, k, pos_emb) + (heads_second,))
        cq, ck = _cutoffs(seq_cutoff, Tq, Tk)
        if in_place:
            qo, ko = q, k
            ctx.mark_dirty(q, k)
        else:
            qo, ko = torch.empty_like(q), torch.empty_like(k)
        lib = _hip.lib()
        _hip.check(lib.rgd_rope_qk(B, H, Tq, Tk, D, t4(q, heads_second), t4(k, heads_second), t4(qo, heads_second),
                                   t4(ko, heads_second), *pe, cq, ck, 0, _hip.dtype_code(q.dtype),
                                   _hip.stream_ptr(q.device)), "rgd_rope_qk")
        ctx.kernel_cache = kernel_cache
        ctx.save_for_backward(pos_emb)
        ctx.seq_cutoff = (cq, ck)
        ctx.heads_second = heads_second
        ctx.dims = (B, H, Tq, Tk, D)
        return qo, ko

    @staticmethod
    def backward(ctx, doq, dok):
        _no_capture("CombinedRoPEFunc.backward")
        (pos_emb,) = ctx.saved_tensors
        assert not ctx.needs_input_grad[2], "CombinedRoPE does not support gradients in position embeddings"
        hs = ctx.heads_second
        doq, dok = _lastdim_contig(doq, dok)
        _remember(ctx.kernel_cache, "bwd", _sig(doq, dok, pos_emb) + (hs,))
        B, H, Tq, Tk, D = ctx.dims
        pe = _pos_emb_args(pos_emb, Tq, Tk)
        cq, ck = ctx.seq_cutoff
        dq, dk = torch.empty_like(doq), torch.empty_like(dok)
        lib = _hip.lib()
        _hip.check(lib.rgd_rope_qk(B, H, Tq, Tk, D, t4(doq, hs), t4(dok, hs), t4(dq, hs), t4(dk, hs), *pe, cq, ck, 1,
                                   _hip.dtype_code(doq.dtype), _hip.stream_ptr(doq.device)), "rgd_rope_qk")
        return dq, dk, None, None, None, None, None


def triton_rope_fn(query, key, pos_emb, seq_cutoff=None, heads_second=True, fused_ln=False, kernel_cache=None,
                   in_place=False):
    """Out of place unless in_place=True.  (The reference passes kernel_cache into the in_place slot,
    head_rope_cached.py:326-327, so its Module rotated q and k in place and never cached; `fused_ln`
    is ignored there as here.)"""
    return CombinedRoPEFunc.apply(query, key, pos_emb, seq_cutoff, heads_second, in_place, kernel_cache)


class FusedRoPEFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, pos_emb, seq_cutoff=None, heads_second=True, norm_eps=1e-6, kernel_cache=None):
        q, k, pos_emb = _lastdim_contig(q, k, _table_for(pos_emb, q))
        B, H, Tq, Tk, D = _qk_dims(q, k, heads_second, 128, "LayerNorm+RoPE")
        pe = _pos_emb_args(pos_emb, Tq, Tk)
        _remember(kernel_cache, "fwd", _sig(q, k, pos_emb) + (heads_second,))
        cq, ck = _cutoffs(seq_cutoff, Tq, Tk)
        qo, ko = torch.empty_like(q), torch.empty_like(k)
        lib = _hip.lib()
        _hip.check(lib.rgd_ln_rope_qk_fwd(B, H, Tq, Tk, D, t4(q, heads_second), t4(k, heads_second),
                                          t4(qo, heads_second), t4(ko, heads_second), *pe, cq, ck,
                                          _hip.dtype_code(q.dtype), float(norm_eps), _hip.stream_ptr(q.device)),
                   "rgd_ln_rope_qk_fwd")
        ctx.kernel_cache = kernel_cache
        ctx.save_for_backward(q, k, pos_emb)
        ctx.seq_cutoff = (cq, ck)
        ctx.heads_second = heads_second
        ctx.norm_eps = float(norm_eps)
        ctx.dims = (B, H, Tq, Tk, D)
        return qo, ko

    @staticmethod
    def backward(ctx, doq, dok):
        _no_capture("FusedRoPEFunc.backward")
        q, k, pos_emb = ctx.saved_tensors
        assert not ctx.needs_input_grad[2], "CombinedRoPE does not support gradients in position embeddings"
        hs = ctx.heads_second
        doq, dok = _lastdim_contig(doq, dok)
        _remember(ctx.kernel_cache, "bwd", _sig(q, k, doq, dok, pos_emb) + (hs,))
        B, H, Tq, Tk, D = ctx.dims
        pe = _pos_emb_args(pos_emb, Tq, Tk)
        cq, ck = ctx.seq_cutoff
        dq, dk = torch.empty_like(q), torch.empty_like(k)
        lib = _hip.lib()
        _hip.check(lib.rgd_ln_rope_qk_bwd(B, H, Tq, Tk, D, t4(q, hs), t4(k, hs), t4(doq, hs), t4(dok, hs), t4(dq, hs),
                                          t4(dk, hs), *pe, cq, ck, _hip.dtype_code(q.dtype), ctx.norm_eps,
                                          _hip.stream_ptr(q.device)), "rgd_ln_rope_qk_bwd")
        return dq, dk, None, None, None, None, None


def triton_fused_ln_rope_fn(query, key, pos_emb, seq_cutoff=None, heads_second=True, norm_eps=1e-6, kernel_cache=None):
    return FusedRoPEFunc.apply(query, key, pos_emb, seq_cutoff, heads_second, norm_eps, kernel_cache)


# ----------------------------------------------------------------------------------------------
# attention
# ----------------------------------------------------------------------------------------------


def _bias_args(bias, q, seqlen_q, seqlen_k, batch, nheads):
    """Bias classification of the reference (flash_attn_triton_cached.py:771-788): 4-D, dtype of q or
    fp32, last two dims (1, Tk) = "vector" or (Tq, Tk) = "matrix", leading dims broadcast."""
    if bias is None:
        return _hip.Tensor4(None, 0, 0, 0), _hip.BIAS_NONE, _hip.RGD_F32
    assert bias.dtype in [q.dtype, torch.float]
    assert bias.is_cuda
    assert bias.dim() == 4
    assert bias.stride(-1) == 1
    if bias.shape[2:] == (1, seqlen_k):
        kind = _hip.BIAS_VECTOR
    elif bias.shape[2:] == (seqlen_q, seqlen_k):
        kind = _hip.BIAS_MATRIX
    else:
        raise RuntimeError("Last 2 dimensions of bias must be (1, seqlen_k)" " or (seqlen_q, seqlen_k)")
    bias = bias.expand(batch, nheads, seqlen_q, seqlen_k)
    desc = _hip.Tensor4(bias.data_ptr(), bias.stride(0), bias.stride(1), bias.stride(2))
    return desc, kind, _hip.dtype_code(bias.dtype)


# The classes of the last head-shared bias seen on each device.  The layers of a model usually share one mask: the first
# attention call of a step classifies it, the others find the classes here.  An entry names the bias by its storage,
# view and version counter (in-place writes through any view bump it) and holds the storage, so that its address cannot
# be given to another tensor while the entry lives; one entry per device, replaced by the next bias.
# Writes that bypass the counter (through `.data`, or by a kernel that was handed the raw pointer) are not seen: call
# clear_bias_classes_cache() after them, or set RGD_CLASSES_CACHE=0.
_classes_cache = {}
_classes_cache_on = os.environ.get("RGD_CLASSES_CACHE", "1") != "0"


def clear_bias_classes_cache():
    """Forgets the tile classes kept for the last head-shared attention bias of every device."""
    _classes_cache.clear()


def _bias_classes(bias, bdesc, bkind, bdtype, dims):
    """Tile classes of a bias matrix that the heads share (rgd_attn_bias_classify): one pass over the bias, made in the
    forward and kept for the backward.  None when the library has no use for them (any other bias, head dims above 64)."""
    if bias is None:
        return None
    lib = _hip.lib()
    nbytes = lib.rgd_attn_bias_classes_bytes(*dims, bdesc, bkind, bdtype)
    if nbytes == 0:
        return None
    # under stream capture the classification must be part of the graph (a replay may find new values in the bias)
    cacheable = _classes_cache_on and not torch.cuda.is_current_stream_capturing()
    storage = bias.untyped_storage()
    # (the stream too: the classes are ready for work queued behind them on the stream that wrote them)
    key = (storage.data_ptr(), bias.storage_offset(), tuple(bias.shape), tuple(bias.stride()), bias.dtype, bias._version, dims,
           torch.cuda.current_stream(bias.device).cuda_stream)
    if cacheable:
        hit = _classes_cache.get(bias.device)
        if hit is not None and hit[0] == key:
            return hit[2]
    classes = torch.empty(nbytes // 8, dtype=torch.int64, device=bias.device)
    _hip.check(lib.rgd_attn_bias_classify(*dims, bdesc, bkind, bdtype, classes.data_ptr(), nbytes, _hip.stream_ptr(bias.device)),
               "rgd_attn_bias_classify")
    if cacheable:
        _classes_cache[bias.device] = (key, storage, classes)
    return classes


def _flash_attn_forward(q, k, v, bias=None, causal=False, softmax_scale=None, kernel_cache=None, return_classes=False):
    batch, seqlen_q, nheads, d = q.shape
    _, seqlen_k, _, _ = k.shape
    key = _sig(q, k, v, bias) + (bool(causal),)
    if not _seen(kernel_cache, "fwd", key):
        assert k.shape == (batch, seqlen_k, nheads, d)
        assert v.shape == (batch, seqlen_k, nheads, d)
        assert d <= 128, "FlashAttention only support head dimensions up to 128"
        assert q.dtype == k.dtype == v.dtype, f"All tensors must have the same type {q.dtype=}, {k.dtype=}, {v.dtype=}"
        assert q.dtype in [torch.float16, torch.bfloat16], "Only support fp16 and bf16"
        assert q.is_cuda and k.is_cuda and v.is_cuda
        _remember(kernel_cache, "fwd", key)
    softmax_scale = softmax_scale or 1.0 / math.sqrt(d)
    if bias is not None and bias.stride(-1) != 1:
        bias = bias.contiguous()
    bdesc, bkind, bdtype = _bias_args(bias, q, seqlen_q, seqlen_k, batch, nheads)
    lib = _hip.lib()
    seqlen_q_rounded = lib.rgd_attn_seqlen_q_rounded(seqlen_q)
    lse = torch.empty((batch, nheads, seqlen_q_rounded), device=q.device, dtype=torch.float32)
    o = torch.empty_like(q)
    ws = _hip.workspace(q.device, lib.rgd_attn_fwd_workspace(batch, nheads, seqlen_q, seqlen_k, d))
    classes = _bias_classes(bias, bdesc, bkind, bdtype, (batch, nheads, seqlen_q, seqlen_k, d))
    _hip.check(lib.rgd_attn_fwd(batch, nheads, seqlen_q, seqlen_k, d, t4(q, False), t4(k, False), t4(v, False),
                                bdesc, bkind, bdtype, t4(o, False), ctypes.c_void_p(lse.data_ptr()),
                                _hip.dtype_code(q.dtype), int(bool(causal)), float(softmax_scale),
                                classes.data_ptr() if classes is not None else None,
                                ctypes.c_void_p(ws.data_ptr()), ws.numel(), _hip.stream_ptr(q.device)), "rgd_attn_fwd")
    if return_classes:
        return o, lse, softmax_scale, classes
    return o, lse, softmax_scale


_ATTN_BWD_MODES = {"auto": _hip.ATTN_BWD_AUTO, "two_kernel": _hip.ATTN_BWD_TWO_KERNEL, "one_pass": _hip.ATTN_BWD_ONE_PASS}
_attn_bwd_mode = os.environ.get("RGD_ATTN_BWD", "auto")
assert _attn_bwd_mode in _ATTN_BWD_MODES, f"RGD_ATTN_BWD must be one of {sorted(_ATTN_BWD_MODES)}"


def set_attention_backward(mode):
    """Form of the attention backward: "two_kernel" (every gradient reproducible bit for bit), "one_pass" (head dims up
    to 64: one kernel, dQ accumulated with fp32 atomics, so its last bits differ from run to run; dK and dV do not;
    wider heads run the two-kernel form) or "auto" (the library's choice).  `torch.use_deterministic_algorithms(True)`
    overrides it with "two_kernel".  Returns the previous setting."""
    global _attn_bwd_mode
    assert mode in _ATTN_BWD_MODES, f"mode must be one of {sorted(_ATTN_BWD_MODES)}"
    prev, _attn_bwd_mode = _attn_bwd_mode, mode
    return prev


def _bwd_mode(d):
    if torch.are_deterministic_algorithms_enabled():
        return _hip.ATTN_BWD_TWO_KERNEL
    if _attn_bwd_mode == "one_pass" and d > 64:
        return _hip.ATTN_BWD_TWO_KERNEL
    return _ATTN_BWD_MODES[_attn_bwd_mode]


# bytes of the buffer that receives dS of every (query, key) pair when a bias gradient is asked for; a bias that
# broadcasts over heads (or the batch) is served in chunks of heads (or batch elements) that fit it
_DBIAS_CHUNK_BYTES = int(os.environ.get("RGD_DBIAS_CHUNK_MB", "256")) << 20


def _attn_bwd_call(do, q, k, v, o, lse, dq, dk, dv, bias, causal, softmax_scale, mode, dfull, bias_classes):
    """One rgd_attn_bwd launch sequence on (B, T, H, D) tensors or views of them; lse is contiguous (B, H, Tq_rounded)."""
    batch, seqlen_q, nheads, d = q.shape
    seqlen_k = k.shape[1]
    lib = _hip.lib()
    bdesc, bkind, bdtype = _bias_args(bias, q, seqlen_q, seqlen_k, batch, nheads)
    ddesc = None
    if dfull is not None:
        ddesc = _hip.Tensor4(dfull.data_ptr(), dfull.stride(0), dfull.stride(1), dfull.stride(2))
    nbytes = lib.rgd_attn_bwd_workspace(batch, nheads, seqlen_q, seqlen_k, d, mode)
    ws = _hip.workspace(q.device, nbytes)
    _hip.check(lib.rgd_attn_bwd(batch, nheads, seqlen_q, seqlen_k, d, t4(do, False), t4(q, False), t4(k, False),
                                t4(v, False), t4(o, False), ctypes.c_void_p(lse.data_ptr()), bdesc, bkind, bdtype,
                                t4(dq, False), t4(dk, False), t4(dv, False), ddesc, _hip.dtype_code(q.dtype),
                                int(bool(causal)), float(softmax_scale), mode,
                                bias_classes.data_ptr() if bias_classes is not None else None, ws.data_ptr(), nbytes,
                                _hip.stream_ptr(q.device)), "rgd_attn_bwd")


def _flash_attn_backward(do, q, k, v, o, lse, dq, dk, dv, bias=None, causal=False, softmax_scale=None,
                         kernel_cache=None, bias_grad=False, bias_classes=None):
    """Returns None, or with bias_grad the gradient of `bias` in its own shape and dtype (beyond the reference, which
    refuses it, flash_attn_triton_cached.py:1107): the dQ kernel leaves dS of every (query, key) pair, rounded to the
    bias dtype, in a (B, H, Tq, Tk) buffer and the dimensions the bias broadcasts are summed here in fp32.  A bias
    that broadcasts over the heads (else: over the batch) is served in chunks of heads (batch elements), so that the
    buffer stays within RGD_DBIAS_CHUNK_MB (256) MiB where one head (batch element) fits that."""
    if do.stride(-1) != 1:
        do = do.contiguous()
    batch, seqlen_q, nheads, d = q.shape
    _, seqlen_k, _, _ = k.shape
    lib = _hip.lib()
    seqlen_q_rounded = lib.rgd_attn_seqlen_q_rounded(seqlen_q)
    key = _sig(q, k, v, bias, do) + (bool(causal),)
    if not _seen(kernel_cache, "bwd", key):
        assert d <= 128
        assert lse.shape == (batch, nheads, seqlen_q_rounded)
        assert q.stride(-1) == k.stride(-1) == v.stride(-1) == o.stride(-1) == 1
        assert dq.stride(-1) == dk.stride(-1) == dv.stride(-1) == 1
        _remember(kernel_cache, "bwd", key)
    _remember(kernel_cache, "bwd_odot", _sig(o, do))
    softmax_scale = softmax_scale or 1.0 / math.sqrt(d)
    if not bias_grad:
        _attn_bwd_call(do, q, k, v, o, lse, dq, dk, dv, bias, causal, softmax_scale, _bwd_mode(d), None, bias_classes)
        return None

    mode = _hip.ATTN_BWD_TWO_KERNEL  # the dQ kernel writes the bias gradient
    tk_pad = (seqlen_k + 63) // 64 * 64  # rows of whole 64-key tiles
    alloc = torch.zeros if causal else torch.empty  # key tiles past the causal diagonal are not visited
    over_heads = bias.shape[1] == 1 and nheads > 1
    over_batch = bias.shape[0] == 1 and batch > 1
    pair_bytes = seqlen_q * tk_pad * bias.element_size()
    hc, bc = nheads, batch
    if over_heads:
        hc = max(1, min(nheads, _DBIAS_CHUNK_BYTES // max(1, batch * pair_bytes)))
    elif over_batch:
        bc = max(1, min(batch, _DBIAS_CHUNK_BYTES // max(1, nheads * pair_bytes)))
    if hc == nheads and bc == batch:
        dfull = alloc((batch, nheads, seqlen_q, tk_pad), dtype=bias.dtype, device=q.device)
        _attn_bwd_call(do, q, k, v, o, lse, dq, dk, dv, bias, causal, softmax_scale, mode, dfull, None)
        dfull = dfull[..., :seqlen_k]
        dims = [i for i in range(4) if bias.shape[i] == 1 and dfull.shape[i] != 1]
        if dims:
            return dfull.sum(dim=dims, keepdim=True, dtype=torch.float32).to(bias.dtype)
        return dfull.contiguous()

    acc = torch.zeros(bias.shape, dtype=torch.float32, device=q.device)
    buf = alloc((bc, hc, seqlen_q, tk_pad), dtype=bias.dtype, device=q.device)
    for b0 in range(0, batch, bc):
        for h0 in range(0, nheads, hc):
            bs, hs = slice(b0, min(batch, b0 + bc)), slice(h0, min(nheads, h0 + hc))
            part = buf[: bs.stop - bs.start, : hs.stop - hs.start]
            if causal and (b0 or h0):
                part.zero_()
            bias_part = bias[bs if bias.shape[0] > 1 else slice(None), hs if bias.shape[1] > 1 else slice(None)]
            _attn_bwd_call(do[bs, :, hs], q[bs, :, hs], k[bs, :, hs], v[bs, :, hs], o[bs, :, hs], lse[bs, hs].contiguous(),
                           dq[bs, :, hs], dk[bs, :, hs], dv[bs, :, hs], bias_part, causal, softmax_scale, mode, part, None)
            got = part[..., :seqlen_k]
            dims = [i for i in range(4) if bias.shape[i] == 1 and got.shape[i] != 1]
            got = got.sum(dim=dims, keepdim=True, dtype=torch.float32) if dims else got.float()
            acc[bs if bias.shape[0] > 1 else slice(None), hs if bias.shape[1] > 1 else slice(None)] += got
    return acc.to(bias.dtype)


class FlashAttnFunc(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, bias=None, causal=False, softmax_scale=None, kernel_cache=None):
        """
        q: (batch_size, seqlen_q, nheads, headdim)
        k, v: (batch_size, seqlen_k, nheads, headdim)
        bias: optional, shape broadcastible to (batch, nheads, seqlen_q, seqlen_k).
        """
        q, k, v, bias = _lastdim_contig(q, k, v, bias)
        o, lse, ctx.softmax_scale, ctx.bias_classes = _flash_attn_forward(
            q, k, v, bias=bias, causal=causal, softmax_scale=softmax_scale, kernel_cache=kernel_cache, return_classes=True)
        ctx.kernel_cache = kernel_cache
        ctx.save_for_backward(q, k, v, o, lse, bias)
        ctx.causal = causal
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    def backward(ctx, do, dlse):
        _no_capture("FlashAttnFunc.backward")
        q, k, v, o, lse, bias = ctx.saved_tensors
        # the reference stops here with "FlashAttention does not support bias gradient yet"
        # (flash_attn_triton_cached.py:1107); this implementation provides it
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        dbias = _flash_attn_backward(do, q, k, v, o, lse, dq, dk, dv, bias=bias, causal=ctx.causal,
                                     softmax_scale=ctx.softmax_scale, kernel_cache=ctx.kernel_cache,
                                     bias_grad=bias is not None and ctx.needs_input_grad[3], bias_classes=ctx.bias_classes)
        return dq, dk, dv, dbias, None, None, None


def flash_attn_func(q, k, v, bias=None, causal=False, softmax_scale=None, return_lse=False, kernel_cache=None):
    o, lse = FlashAttnFunc.apply(q, k, v, bias, causal, softmax_scale, kernel_cache)
    return (o, lse) if return_lse else o


# ----------------------------------------------------------------------------------------------
# learned relative position bias (no counterpart in the reference)
# ----------------------------------------------------------------------------------------------


class _RelativeRanges:
    """The buckets as ranges of d = key position - query position, ascending (what the C ABI takes)."""

    def __init__(self, starts, buckets):
        self.starts, self.buckets, self.n, self.most = starts, buckets, len(starts), max(buckets)
        self.c_starts = (ctypes.c_int32 * self.n)(*starts)
        self.c_buckets = (ctypes.c_int32 * self.n)(*buckets)
        self.starts_at, self.buckets_at = ctypes.addressof(self.c_starts), ctypes.addressof(self.c_buckets)


@functools.lru_cache(maxsize=64, typed=True)
def relative_ranges(num_buckets, max_distance, bidirectional):
    """Buckets of a learned relative position bias, n = query position - key position.  Causal (bidirectional False):
    n < 0 counts as 0, and with e = num_buckets // 2 the distances n < e have a bucket each, the others
    e + floor(log(n / e) / log(max_distance / e) * (num_buckets - e)), at most the last bucket.  Bidirectional: the same
    with half of the buckets for n >= 0, and the other half, after them, for the keys behind the query with |n|.
    The borders are found in whole numbers: bucket e + k begins at the smallest n with n^m >= max_distance^k e^(m - k), m the
    number of logarithmic buckets, so no rounding of a logarithm decides a bucket."""
    assert isinstance(num_buckets, int) and 2 <= num_buckets <= 256, f"{num_buckets=}: 2 to 256 buckets"
    assert not bidirectional or (num_buckets % 2 == 0 and num_buckets >= 4), f"{num_buckets=}: bidirectional buckets are even, at least 4"
    side = num_buckets // 2 if bidirectional else num_buckets
    e = side // 2
    assert isinstance(max_distance, int) and e < max_distance < 2**30, f"{max_distance=}: more than {e}, less than 2^30"
    m = side - e
    begin = list(range(e + 1))  # smallest n of buckets 0 .. e
    for k in range(1, m):
        bar = max_distance**k * e ** (m - k)
        lo, hi = begin[-1], max_distance
        while lo < hi:  # smallest n with n^m >= bar
            mid = (lo + hi) // 2
            lo, hi = (lo, mid) if mid**m >= bar else (mid + 1, hi)
        begin.append(lo)
    # a bucket that begins where the next one does holds nothing
    held = [b for b in range(side) if b + 1 == side or begin[b] < begin[b + 1]]
    starts, buckets = [], []
    for b in reversed(held):  # keys in front of the query, farthest first: n from begin[b] on, d = -n up to -begin[b]
        end = [begin[c] for c in held if c > b]
        starts.append(1 - end[0] if end else -(2**31))
        buckets.append(b)
    if bidirectional:
        for b in held:
            if b > 0:
                starts.append(begin[b])
                buckets.append(side + b)
    return _RelativeRanges(tuple(starts), tuple(buckets))


# The functions below are called once per token, or between short kernels, where their host time is what a user waits for: tensor
# attributes are read once, arguments are packed bytes, the stream is asked for as a number.
_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream
_desc4 = _hip.desc4


@functools.lru_cache(maxsize=256)
def _bias_workspaces(nheads, seqlen_q, seqlen_k, num_buckets, code):
    lib = _hip.lib()
    return (lib.rgd_rel_bias_fwd_workspace(nheads, seqlen_q, seqlen_k, code),
            lib.rgd_rel_bias_bwd_workspace(nheads, seqlen_q, seqlen_k, num_buckets))


def _relative_bias(weight, seqlen_q, seqlen_k, ranges, q_offset, dtype, kernel_cache):
    wstride = weight.stride()
    device = weight.device
    # (lengths and offsets are not kept: a model that reads on in chunks has others with every call)
    assert seqlen_q >= 0 and seqlen_k >= 0, f"{seqlen_q=}, {seqlen_k=}"
    key = kernel_cache and (weight.shape, wstride, weight.dtype, device, dtype, ranges.most)
    if not _seen(kernel_cache, "fwd", key):
        assert weight.is_cuda, "rgd_triton_amd operators run on the GPU only"
        assert weight.dtype in _FLOATS and dtype in _FLOATS, "Only support fp16, bf16, and fp32"
        assert weight.ndim == 2 and ranges.most < weight.shape[0], f"{weight.shape=}"
        _remember(kernel_cache, "fwd", key)
    index = device.index
    if index != _current_device():  # kernels are launched on the tensors' device, whichever is current
        with torch.cuda.device(index):
            return _relative_bias(weight, seqlen_q, seqlen_k, ranges, q_offset, dtype, None)
    num_buckets, nheads = weight.shape
    bias = torch.empty((1, nheads, seqlen_q, seqlen_k), dtype=dtype, device=device)
    lib, code = _hip.lib(), _hip.dtype_code(dtype)
    nbytes = _bias_workspaces(nheads, seqlen_q, seqlen_k, num_buckets, code)[0]  # 0 for all but large matrices
    ws = _hip.workspace(device, nbytes) if nbytes else None
    rc = lib.rgd_rel_bias_fwd(nheads, seqlen_q, seqlen_k, weight.data_ptr(), wstride[0], num_buckets, _hip.dtype_code(weight.dtype),
                              ranges.n, ranges.c_starts, ranges.c_buckets, q_offset,
                              _desc4(bias.data_ptr(), 0, seqlen_q * seqlen_k, seqlen_k), code, ws.data_ptr() if nbytes else None, nbytes,
                              _raw_stream(index))
    if rc:
        _hip.check(rc, "rgd_rel_bias_fwd")
    return bias


def _relative_bias_grad(dbias, num_buckets, nheads, seqlen_q, seqlen_k, ranges, q_offset, wdtype):
    stride = dbias.stride()
    if stride[3] != 1:
        dbias = dbias.contiguous()
        stride = dbias.stride()
    device = dbias.device
    index = device.index
    if index != _current_device():
        with torch.cuda.device(index):
            return _relative_bias_grad(dbias, num_buckets, nheads, seqlen_q, seqlen_k, ranges, q_offset, wdtype)
    dw = torch.empty((num_buckets, nheads), dtype=wdtype, device=device)
    lib = _hip.lib()
    code = _hip.dtype_code(dbias.dtype)
    nbytes = _bias_workspaces(nheads, seqlen_q, seqlen_k, num_buckets, code)[1]
    ws = _hip.workspace(device, nbytes)
    rc = lib.rgd_rel_bias_bwd(nheads, seqlen_q, seqlen_k, _desc4(dbias.data_ptr(), 0, stride[1], stride[2]),
                              code, ranges.n, ranges.c_starts, ranges.c_buckets, q_offset, dw.data_ptr(),
                              nheads, num_buckets, _hip.dtype_code(wdtype), ws.data_ptr(), nbytes, _raw_stream(index))
    if rc:
        _hip.check(rc, "rgd_rel_bias_bwd")
    return dw


class Relative_Bias_Func(torch.autograd.Function):
    @staticmethod
    def forward(ctx, weight, call):
        ctx.weight, ctx.call = (*weight.shape, weight.dtype), call
        return _relative_bias(weight, *call)

    @staticmethod
    def backward(ctx, dbias):
        # (once_differentiable costs 5 us, so only what could be differentiated again passes through it)
        if torch.is_grad_enabled() and dbias.requires_grad:
            return _relative_bias_once(ctx, dbias)
        return _relative_bias_backward(ctx, dbias)


def _relative_bias_backward(ctx, dbias):
    _no_capture("Relative_Bias_Func.backward")
    num_buckets, nheads, wdtype = ctx.weight
    seqlen_q, seqlen_k, ranges, q_offset, _, kernel_cache = ctx.call
    if kernel_cache is not None:
        _remember(kernel_cache, "bwd", _sig(dbias))
    return _relative_bias_grad(dbias, num_buckets, nheads, seqlen_q, seqlen_k, ranges, q_offset, wdtype), None


_relative_bias_once = torch.autograd.function.once_differentiable(_relative_bias_backward)


def relative_position_bias_fn(weight, seqlen_q, seqlen_k, max_distance=128, bidirectional=True, q_offset=0, dtype=None,
                              kernel_cache=None):
    """Learned relative position bias for flash_attn_func(bias=...): (1, nheads, seqlen_q, seqlen_k) with
    bias[0, h, i, j] = weight[bucket of key j for query i + q_offset, h], weight (num_buckets, nheads); the buckets are
    relative_ranges'.  dtype: of the bias (the weight's by default; attention takes its own tensors' or fp32).  The
    gradient of the weight is summed in fp32 and rounded once."""
    if weight.stride(-1) != 1:
        weight = weight.contiguous()
    ranges = relative_ranges(weight.shape[0], max_distance, bool(bidirectional))
    _no_tangent("relative_position_bias", weight)
    if torch.is_grad_enabled() and weight.requires_grad:
        return Relative_Bias_Func.apply(weight, (seqlen_q, seqlen_k, ranges, q_offset, dtype or weight.dtype, kernel_cache))
    return _relative_bias(weight, seqlen_q, seqlen_k, ranges, q_offset, dtype or weight.dtype, kernel_cache)


# ----------------------------------------------------------------------------------------------
# paged key/value cache (no counterpart in the reference)
# ----------------------------------------------------------------------------------------------


def _no_grad(what, *ts):
    for t in ts:
        assert t is None or not t.requires_grad, f"{what} is for serving and has no gradient: call it under torch.no_grad()"


def _check_cache(what, k_cache, v_cache, page_table, lens, batch, dtype, head_dim):
    shape = k_cache.shape
    assert len(shape) == 4 and shape == v_cache.shape, f"{k_cache.shape=}, {v_cache.shape=}"
    assert k_cache.stride(-1) == v_cache.stride(-1) == 1, f"{what}: the caches need unit-stride head dims"
    assert k_cache.dtype == v_cache.dtype == dtype, f"All tensors must have the same type {dtype=}, {k_cache.dtype=}, {v_cache.dtype=}"
    assert dtype in (torch.float16, torch.bfloat16), "Only support fp16 and bf16"
    assert shape[3] == head_dim <= 128, f"{what} only supports head dimensions up to 128, the cache's the same: {head_dim=}"
    assert shape[1] >= 1, f"{k_cache.shape=}: page size must be positive"
    table = page_table.shape
    assert page_table.dtype == torch.int32 and len(table) == 2 and table[0] == batch, \
        f"page_table is (batch, pages) int32: {page_table.dtype}, {page_table.shape}"
    assert table[1] <= 1 or page_table.stride(1) == 1, "page_table rows need unit stride"
    _check_lens(lens, batch)


def _check_lens(lens, batch):
    assert lens.dtype == torch.int32 and lens.shape == (batch,) and (batch <= 1 or lens.stride(0) == 1), \
        f"lengths are (batch,) int32, contiguous: {lens.dtype}, {lens.shape}"


def _check_device(what, index, *ts):
    """index: get_device() of the operator's first tensor, -1 for one that is not on a GPU"""
    assert index >= 0, "rgd_triton_amd operators run on the GPU only"
    for t in ts:
        assert t is None or t.get_device() == index, f"{what}: a tensor on {t.device}, another on cuda:{index}"


def rope_cache_append_fn(query, key, value, pos_emb, k_cache, v_cache, page_table, cache_lens, new_lens=None, seq_cutoff=None,
                         heads_second=True, norm_eps=None, kernel_cache=None):
    """Appends the new tokens of every sequence to a paged cache, rotating query and key at their positions on the way;
    returns the rotated query, writes k_cache and v_cache in place.

    query (B, Hq, T, D), key and value (B, Hkv, T, D) with heads_second, else (B, T, H, D); k_cache, v_cache
    (num_pages, page_size, Hkv, D), any strides with a unit last one (head-major storage is passed as a transposed view);
    page_table (B, pages) int32; cache_lens (B,) int32, the tokens already there: token t gets position cache_lens[b] + t, page
    page_table[b, position // page_size].  new_lens (B,) int32: how many of the T tokens are real, the rest is padding (nothing
    stored, query rows zero).  pos_emb as in triton_rope_fn, with a row for every position the page table covers; None: no
    rotation.  Positions from seq_cutoff on (an int, or one for query and one for key) are not rotated.  norm_eps: LayerNorm over
    the head dim in front of the rotation, as triton_fused_ln_rope_fn has it; None: none.  A token whose page number is outside
    the cache is not stored; one whose position is outside the page table is padding.  Two tokens of a call must not fall on one slot
    (a page twice in the table), and the two caches must not share memory.  cache_lens is the caller's to advance."""
    what = "rope_cache_append"
    query, key, value = _lastdim_contig(query, key, value)
    if pos_emb is not None:
        (pos_emb,) = _lastdim_contig(_table_for(pos_emb, query))
    if torch.is_grad_enabled():
        _no_grad(what, query, key, value, pos_emb, k_cache, v_cache)
    _no_tangent(what, query, key, value, pos_emb, k_cache, v_cache)
    head, tok = (1, 2) if heads_second else (2, 1)
    shape, kshape, cshape = query.shape, key.shape, k_cache.shape
    index = query.get_device()
    dtype = query.dtype
    sig = kernel_cache and _sig(query, key, value, pos_emb, k_cache, v_cache, page_table, cache_lens, new_lens) + (bool(heads_second),)
    if not _seen(kernel_cache, "fwd", sig):
        assert len(shape) == len(kshape) == 4
        assert dtype == key.dtype == value.dtype, "All tensors must have the same type"
        assert kshape == value.shape and kshape[0] == shape[0] and kshape[tok] == shape[tok] and kshape[3] == shape[3], \
            f"{query.shape=}, {key.shape=}, {value.shape=}"
        _check_cache(what, k_cache, v_cache, page_table, cache_lens, shape[0], dtype, shape[3])
        assert cshape[2] == kshape[head], f"{k_cache.shape=}, {key.shape=}"
        if new_lens is not None:
            _check_lens(new_lens, shape[0])
        if pos_emb is not None:
            assert pos_emb.ndim == 3 and pos_emb.shape[0] == 2 and pos_emb.dtype in _FLOATS, f"{pos_emb.shape=}"
            assert pos_emb.shape[2] <= shape[3] and pos_emb.shape[2] % 2 == 0, f"{pos_emb.shape=}: an even rotary dim, at most {shape[3]}"
            assert pos_emb.shape[1] >= page_table.shape[1] * cshape[1], \
                f"{pos_emb.shape=}: a row for every position of {page_table.shape[1]} pages of {cshape[1]}"
        _check_device(what, index, key, value, pos_emb, k_cache, v_cache, page_table, cache_lens, new_lens)
        _remember(kernel_cache, "fwd", sig)
    if index != _current_device():
        with torch.cuda.device(index):
            return rope_cache_append_fn(query, key, value, pos_emb, k_cache, v_cache, page_table, cache_lens, new_lens, seq_cutoff,
                                        heads_second, norm_eps)
    if pos_emb is None:
        table, P, R, ss, sn, table_code = 0, 0, 0, 0, 0, _hip.RGD_F32
    else:
        _, P, R = pos_emb.shape
        ss, sn, _ = pos_emb.stride()
        table, table_code = pos_emb.data_ptr(), _hip.dtype_code(pos_emb.dtype)
    cq, ck = _cutoffs(seq_cutoff, 2**31 - 1, 2**31 - 1)
    qo = torch.empty_like(query)
    sq, sk, sv, so = query.stride(), key.stride(), value.stride(), qo.stride()
    kcp, kcs, kch, _ = k_cache.stride()
    vcp, vcs, vch, _ = v_cache.stride()
    args = _hip.append_args(
        shape[0], shape[tok], shape[head], kshape[head], shape[3], query.data_ptr(), sq[0], sq[head], sq[tok], key.data_ptr(), sk[0], sk[head], sk[tok],
        value.data_ptr(), sv[0], sv[head], sv[tok], qo.data_ptr(), so[0], so[head], so[tok], k_cache.data_ptr(), kcp, kch, kcs, v_cache.data_ptr(), vcp,
        vch, vcs, cshape[0], cshape[1], page_table.data_ptr(), page_table.shape[1], page_table.stride(0), cache_lens.data_ptr(),
        0 if new_lens is None else new_lens.data_ptr(), table, P, R, ss, sn, cq, ck, table_code, norm_eps is not None,
        _hip.dtype_code(dtype), norm_eps or 0.0)
    rc = _hip.lib().rgd_rope_cache_append(args, _raw_stream(index))
    if rc:
        _hip.check(rc, "rgd_rope_cache_append")
    if k_cache.is_inference() or v_cache.is_inference():  # (tensors made in inference mode have no version)
        for cache in (k_cache, v_cache):
            if not cache.is_inference():
                torch.autograd.graph.increment_version(cache)
    else:
        torch.autograd.graph.increment_version((k_cache, v_cache))
    return qo


_NO_BIAS = (0, 0, 0, 0, 0, 0)


@functools.lru_cache(maxsize=256)
def _decode_workspace(B, Hq, Hkv, D):
    return _hip.lib().rgd_paged_decode_workspace(B, Hq, Hkv, D)


def paged_decode_attn_func(q, k_cache, v_cache, page_table, seq_lens, rel_weight=None, max_distance=128, bidirectional=True,
                           softmax_scale=None, return_lse=False, kernel_cache=None):
    """Attention of one new token per sequence over a paged cache.

    q (B, 1, Hq, D); k_cache, v_cache (num_pages, page_size, Hkv, D), Hq a multiple of Hkv (query head h reads key head
    h // (Hq // Hkv)); page_table (B, pages) int32; seq_lens (B,) int32: keys 0 .. seq_lens[b] - 1 are seen, the new token's own
    key among them.  rel_weight (num_buckets, Hq): the learned bias of relative_position_bias_fn for a query at position
    seq_lens[b] - 1.  Returns o (B, 1, Hq, D), with return_lse also the logsumexp (B, Hq) in fp32.  A sequence without keys gives
    o = 0, lse = -inf.  Keys on a page number outside the cache are not seen; lengths beyond the page table end there."""
    what = "paged_decode_attn"
    sq = q.stride()
    if sq[-1] != 1:
        q = q.contiguous()
        sq = q.stride()
    if rel_weight is not None and rel_weight.stride(-1) != 1:
        rel_weight = rel_weight.contiguous()
    if torch.is_grad_enabled():
        _no_grad(what, q, k_cache, v_cache, rel_weight)
    _no_tangent(what, q, k_cache, v_cache, rel_weight)
    shape, cache = q.shape, k_cache.shape
    index = q.get_device()
    dtype = q.dtype
    sig = kernel_cache and _sig(q, k_cache, v_cache, page_table, seq_lens, rel_weight)
    if not _seen(kernel_cache, "fwd", sig):
        assert len(shape) == 4 and shape[1] == 1, f"{q.shape=}: one new token per sequence"
        _check_cache(what, k_cache, v_cache, page_table, seq_lens, shape[0], dtype, shape[3])
        assert cache[2] >= 1 and shape[2] % cache[2] == 0, f"{q.shape=}, {k_cache.shape=}: query heads in groups"
        if rel_weight is not None:
            assert rel_weight.ndim == 2 and rel_weight.shape[1] == shape[2] and rel_weight.dtype in _FLOATS, f"{rel_weight.shape=}"
        _check_device(what, index, k_cache, v_cache, page_table, seq_lens, rel_weight)
        _remember(kernel_cache, "fwd", sig)
    if index != _current_device():
        with torch.cuda.device(index):
            return paged_decode_attn_func(q, k_cache, v_cache, page_table, seq_lens, rel_weight, max_distance, bidirectional,
                                          softmax_scale, return_lse)
    B, _, Hq, D = shape
    rel, rel_code = _NO_BIAS, _hip.RGD_F32
    if rel_weight is not None:
        r = relative_ranges(rel_weight.shape[0], max_distance, bool(bidirectional))
        rel = (rel_weight.data_ptr(), rel_weight.stride(0), rel_weight.shape[0], r.n, r.starts_at, r.buckets_at)
        rel_code = _hip.dtype_code(rel_weight.dtype)
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = torch.empty((B, Hq), dtype=torch.float32, device=q.device) if return_lse else None
    nbytes = _decode_workspace(B, Hq, cache[2], D)
    ws = _hip.workspace(q.device, nbytes)
    kcp, kcs, kch, _ = k_cache.stride()
    vcp, vcs, vch, _ = v_cache.stride()
    args = _hip.decode_args(
        B, Hq, cache[2], D, q.data_ptr(), sq[0], sq[2], sq[1], k_cache.data_ptr(), kcp, kch, kcs, v_cache.data_ptr(), vcp, vch, vcs,
        o.data_ptr(), Hq * D, D, 0, cache[0], cache[1], page_table.data_ptr(), page_table.shape[1], page_table.stride(0),
        seq_lens.data_ptr(), *rel, 0 if lse is None else lse.data_ptr(), ws.data_ptr(), nbytes, rel_code, _hip.dtype_code(dtype),
        1.0 / math.sqrt(D) if softmax_scale is None else softmax_scale)
    rc = _hip.lib().rgd_paged_decode(args, _raw_stream(index))
    if rc:
        _hip.check(rc, "rgd_paged_decode")
    return (o, lse) if return_lse else o
