"""PagedDecodeAttention at the ends of its ranges: keys that weigh next to nothing each and something together, infinite values under
small weights, logits so large that neighbouring numbers are far apart, thousands of sequences."""
import math

import pytest
import torch

from serving_helpers import gen, half_step, randn, serving_oracle

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("D", [64, 32, 80, 128])
@pytest.mark.parametrize("drop", [25, 20, 30])
def test_many_keys_far_below_one(D, dtype, drop):
    """one key, then 32767 equal ones 2^-drop of it, for as many key heads in all as wavefronts are resident (12 a compute unit up to
    D = 64, else 8), so that a wavefront walks the whole length behind the one key.  All sequences read the same two pages."""
    from rgd_triton_amd import paged_decode_attn_func

    n, size, H = 32768, 128, 2
    B = 1536 if D <= 64 else 1024
    k, v = torch.zeros(2, size, H, D), torch.ones(2, size, H, D)
    k[0, 0, :, 0] = 1.0
    v[0, 0], v[0, 0, :, 1] = 0.0, 1.0
    k, v = k.to(dtype), v.to(dtype)
    table = torch.ones(1, n // size, dtype=torch.int32)
    table[0, 0] = 0
    q = torch.zeros(1, 1, H, D)
    q[..., 0] = 16.0
    q, scale = q.to(dtype), drop * math.log(2) / 16.0
    lens = torch.full((1,), n, dtype=torch.int32)
    o, lse = paged_decode_attn_func(q.expand(B, 1, H, D).cuda(), k.cuda(), v.cuda(), table.expand(B, -1).cuda(), lens.expand(B).contiguous().cuda(),
                                    softmax_scale=scale, return_lse=True)
    ref, rlse, _, reach = serving_oracle.decode(q, k, v, table, lens, scale)
    # the logit by 2^-22 of itself and the sums by length 2^-24, relative (check_decode), the parts of a probability by 2^-14 of it and in
    # fp16 by 2^-33 of the largest; values are 0 and 1; one rounding
    p = torch.cat([torch.ones(1), torch.full((n - 1,), 2.0**-drop)]).double()
    p /= p.sum()
    rel = 2 * 2.0**-22 * (reach.max().item() + rlse.max().item() + 1) + 2 * (n + 16) * 2.0**-24 + 2.0**-14
    floor = n * 2.0**-33 * p[0].item() if dtype == HF else 0.0
    bound = rel * ref + floor
    tol = half_step(dtype) * (ref + bound) + bound + (2.0**-25 if dtype == HF else 0.0)
    assert ((o.double().cpu() - ref).abs() <= tol).all(), ((o.double().cpu() - ref).abs() / tol).max()
    assert ((lse.double().cpu() - rlse).abs() <= 2.0**-22 * (drop + 12) + (n + 16) * 2.0**-24).all()


@pytest.mark.parametrize("drop,dtype", [(5, HF), (20, HF), (25, HF), (25, BF), (60, BF)])
def test_infinite_values_under_small_weights(drop, dtype):
    """an infinite value stays infinite, and alone, under a weight 2^-drop of the largest; before and behind the largest, also where the
    pieces of a sequence are joined"""
    from rgd_triton_amd import paged_decode_attn_func

    size, D = 16, 64
    for n in (40, 3000):
        g = gen(620)
        pages = -(-n // size)
        k, v = torch.zeros(pages, size, 1, D, dtype=dtype), randn(g, pages, size, 1, D, dtype=dtype)
        q = torch.zeros(1, 1, 2, D, dtype=dtype)
        q[..., 0] = 16.0
        at = lambda j: (j // size, j % size, 0)  # noqa: E731
        k[at(n // 2)][0] = 1.0  # the largest
        for j, c, value in ((3, 5, math.inf), (n - 1, 6, -math.inf), (n // 2, 7, math.inf)):
            v[at(j)][c] = value
        o = paged_decode_attn_func(q.cuda(), k.cuda(), v.cuda(), torch.arange(pages, dtype=torch.int32)[None].cuda(),
                                   torch.tensor([n], dtype=torch.int32).cuda(), softmax_scale=drop * math.log(2) / 16.0).cpu()
        for h in range(2):
            assert o[0, 0, h, 5] == math.inf and o[0, 0, h, 6] == -math.inf and o[0, 0, h, 7] == math.inf, o[0, 0, h, 5:8]
            assert torch.isfinite(o[0, 0, h].float()).sum() == D - 3


@pytest.mark.parametrize("dtype", [HF, BF])
@pytest.mark.parametrize("top", [2.0**16, 2.0**20, 2.0**23, 2.0**24, 2.0**26])
def test_logits_so_large_that_steps_are_whole(top, dtype):
    """logits `top` + 0, 1, 2, .. rounded to what 32 bits hold there, rising and falling: exact in 32 bits, so the weights are
    those of the rounded logits"""
    from rgd_triton_amd import paged_decode_attn_func

    n, size, D = 96, 16, 64
    g = gen(630)
    step = max(1.0, top * 2.0**-23)
    j = torch.arange(n)
    rise = torch.stack([j % 32, 31 - j % 32, (7 * j) % 32]).float() * step  # per key head
    # q = (64, 1, 0, ..), k = (top / 64 split over channels, rise): products and their sums are whole numbers of the step
    q = torch.zeros(1, 1, 3, D)
    q[..., 0], q[..., 1] = 256.0, step
    k = torch.zeros(n, 3, D)
    high = top / 256.0
    if high > 32768:  # fp16 ends at 65504: the rest by a larger factor
        q[..., 0], high = 16384.0, top / 16384.0
    k[..., 0], k[..., 1] = high, (rise / step).t()
    v = randn(g, n, 3, D, shift=0.5)
    q, k, v = q.to(dtype), k.to(dtype), v.to(dtype)
    pages = n // size
    o, lse = paged_decode_attn_func(q.cuda(), k.reshape(pages, size, 3, D).cuda(), v.reshape(pages, size, 3, D).cuda(),
                                    torch.arange(pages, dtype=torch.int32)[None].cuda(), torch.tensor([n], dtype=torch.int32).cuda(),
                                    softmax_scale=1.0, return_lse=True)
    s = (q[0, 0].double()[:, None] * k.double().transpose(0, 1)).sum(-1)  # (heads, keys)
    assert torch.equal(s, s.float().double())
    p = torch.softmax(s, -1)
    ref, mag = ((p[:, None] @ x.transpose(0, 1))[:, 0] for x in (v.double(), v.double().abs()))
    # the differences of logits are exact; a product with log2(e) and an exponential of at most 45 in front: 2^-17; parts 2^-14
    bound = (2.0**-17 + 2.0**-13 + 112 * 2.0**-23) * mag
    assert ((o[0, 0].double().cpu() - ref).abs() <= half_step(dtype) * (ref.abs() + bound) + bound).all()
    assert ((lse[0].double().cpu() - torch.logsumexp(s, -1)).abs() <= 2.0**-23 * top + 2.0**-18).all()


@pytest.mark.parametrize("Hq,Hkv,D,size,most,dtype", [(2, 1, 64, 4, 9, BF), (3, 3, 40, 16, 70, HF)])
def test_thousands_of_sequences(Hq, Hkv, D, size, most, dtype):
    """6000 sequences, a third of them empty: a wavefront finds its run behind 94 looks at the lengths.  Checked on the GPU in 64 bits"""
    from rgd_triton_amd import paged_decode_attn_func

    B, g = 6000, gen(640)
    each = -(-most // size)
    pages = torch.randperm(B * each, generator=g).to(torch.int32).reshape(B, each).cuda()
    lens = torch.randint(0, most + 1, (B,), generator=g, dtype=torch.int32)
    lens[::3] = 0
    lens = lens.cuda()
    q = randn(g, B, 1, Hq, D, dtype=dtype).cuda()
    k, v = (randn(g, B * each, size, Hkv, D, dtype=dtype, shift=0.2).cuda() for _ in range(2))
    o, lse = paged_decode_attn_func(q, k, v, pages, lens, return_lse=True)
    kk, vv = (c[pages.long()].reshape(B, each * size, Hkv, D).double().repeat_interleave(Hq // Hkv, 2) for c in (k, v))
    s = (kk * q.double()).sum(-1) * D**-0.5  # (B, keys, Hq)
    reach = ((kk * q.double()).abs().sum(-1) * D**-0.5).max().item()
    s = s.masked_fill((torch.arange(each * size, device="cuda") >= lens[:, None])[..., None], -math.inf)
    p = torch.softmax(s, 1).nan_to_num(0.0)
    ref, mag = ((p[..., None] * x).sum(1)[:, None] for x in (vv, vv.abs()))
    # as check_decode has it: products and sums of a logit, the exponential, the parts of a probability, sums over the keys
    bound = (2 * ((D + 4) * 2.0**-24 * reach + 2.0**-22 * (reach + 10)) + 2 * (most + 16) * 2.0**-24 + 2.0**-14) * mag
    assert ((o.double() - ref).abs() <= half_step(dtype) * (ref.abs() + bound) + bound + 2.0**-25).all()
    rlse = torch.logsumexp(s, 1)
    assert torch.equal(lse[lens == 0], torch.full_like(lse[lens == 0], -math.inf)) and torch.isfinite(lse[lens > 0]).all()
    seen = lens > 0
    assert ((lse[seen].double() - rlse[seen]).abs() <= (D + 4) * 2.0**-24 * reach + 2.0**-21 * (reach + 10)).all()
