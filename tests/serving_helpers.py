"""Inputs and tolerances of the cache, decode and relative-bias tests."""
import math
import os
import sys

import torch

from helpers import ROOT, dev, gen, randn

sys.path.insert(0, os.path.join(ROOT, "oracle"))
import serving_oracle  # noqa: E402,F401


def half_step(dtype):
    """largest rounding error relative to the value"""
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """half a step at the bottom of the type's range (subnormal numbers)"""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def pages_for(g, B, cap, size, spare=3):
    """(page count, page table (B, ceil(cap / size)) int32): the sequences' pages in no order among spare ones"""
    each = -(-cap // size)
    total = B * each + spare
    return total, torch.randperm(total, generator=g)[: B * each].to(torch.int32).reshape(B, each)


def rounded_once(actual, ref, bound, name=""):
    """|actual - ref| within half a step of the type, of the value, plus the 32-bit error bound of its computation"""
    a, r = actual.detach().cpu().double(), ref
    tol = half_step(actual.dtype) * (r.abs() + bound) + bound + smallest(actual.dtype)
    assert torch.equal(torch.isnan(a), torch.isnan(r)), f"{name}: NaN pattern differs"
    bad = (a - r).abs() > tol
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {((a - r).abs() / tol).max():.3g} of the tolerance"


def check_decode(o, lse, ref, length, D, name=""):
    """o and lse against the oracle's.  In 32 bits a logit's product is off by at most d = (D + 4) 2^-24 reach (D products of
    16-bit values, exact, and their sums; the scale), the logit itself by 2 roundings of its value (bias, difference to the
    maximum), the exponential by 4 2^-24 relative: every p by r = d + 2^-22 |logit| + 2^-22 relative, numerator and denominator
    both; p is split into two 16-bit parts, the first within 2^-8 of (1 - 2^-7) p (bf16), so that the second is at most
    (2^-7 + 2^-8) p = 0.0118 p and its own rounding at most 2^-8 0.0118 p < 2^-14 p; sums over the keys add length 2^-24.  The output is then
    rounded once."""
    ro, rlse, weighted, reach = ref
    span = reach.max().item() + rlse[torch.isfinite(rlse)].abs().max().item() if torch.isfinite(rlse).any() else 0.0
    r = (D + 4) * 2.0**-24 * reach + 2.0**-22 * (span + 1)
    sums = (length + 16) * 2.0**-24
    rounded_once(o, ro, (2 * r + 2 * sums + 2.0**-14)[:, None, :, None] * weighted, f"{name} o")
    if lse is not None:
        a = lse.cpu().double()
        fin = torch.isfinite(rlse)
        assert torch.equal(a[~fin], rlse[~fin]), f"{name}: lse of empty rows"
        off = ((a - rlse).abs() - (r + sums + 2.0**-22 * (rlse.abs() + 1)))[fin]
        assert (off <= 0).all(), f"{name}: lse off by {off.max()} more than allowed"


def rotary(positions, R, dtype=torch.float32):
    rate = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))
    ang = torch.arange(positions, dtype=torch.float64)[:, None] * rate
    return torch.stack([ang.sin(), ang.cos()]).repeat_interleave(2, dim=-1).to(dtype)


def spread(t, dims):
    """The values of t in a larger buffer: a view with gaps after every listed dimension (NaN in the gaps on the GPU)."""
    shape = list(t.shape)
    big = torch.zeros([n + (8 if i in dims else 0) for i, n in enumerate(shape)], dtype=t.dtype)
    v = big[tuple(slice(0, n) for n in shape)]
    v.copy_(t)
    return v


__all__ = ["dev", "gen", "randn", "math", "half_step", "smallest", "pages_for", "rounded_once", "check_decode", "rotary", "spread",
           "serving_oracle"]
