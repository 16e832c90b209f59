"""PagedDecodeAttention against the definition in 64 bits.  Every slot of the cache that no key of a sequence stands in holds NaN, so
a read beyond a length or a page shows in the output."""
import math

import pytest
import torch

from serving_helpers import check_decode, dev, gen, pages_for, randn, serving_oracle, spread

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
CASES = [  # Hq, Hkv, D, page, lengths, dtype, buckets
    (1, 1, 64, 16, [1], BF, 0),
    (4, 4, 64, 16, [0, 1, 15, 16, 17, 33, 200], BF, 0),
    (8, 2, 128, 16, [31, 32, 33, 127, 128, 129, 0, 1000], BF, 0),
    (8, 1, 128, 64, [700, 5], HF, 0),
    (32, 1, 128, 16, [65, 300], BF, 0),
    (40, 2, 64, 32, [90, 257], HF, 0),
    (17, 1, 32, 16, [40, 1], BF, 0),
    (6, 6, 80, 5, [0, 4, 5, 6, 64, 333], HF, 32),
    (6, 3, 96, 48, [47, 48, 49, 500], BF, 32),
    (4, 2, 59, 7, [0, 13, 14, 15, 222], BF, 0),
    (3, 3, 111, 1, [1, 2, 130], HF, 8),
    (4, 1, 16, 3, [3, 100, 70], BF, 8),
    (2, 2, 8, 8, [9, 64, 65], HF, 0),
    (2, 1, 1, 4, [5, 33], HF, 0),
    (2, 2, 128, 128, [127, 128, 129, 2000], HF, 32),
    (16, 16, 64, 24, [513] * 40, BF, 32),
    (2, 2, 64, 16, [5000], BF, 32),
]


def _inputs(case, seed, extra=3):
    Hq, Hkv, D, size, lens, dtype, nb = case
    g = gen(seed)
    B, cap = len(lens), max(max(lens), 1) + extra
    total, pt = pages_for(g, B, cap, size)
    s = dict(q=randn(g, B, 1, Hq, D, dtype=dtype), k=randn(g, total, size, Hkv, D, dtype=dtype),
             v=randn(g, total, size, Hkv, D, dtype=dtype, shift=0.3), pages=pt, lens=torch.tensor(lens, dtype=torch.int32),
             w=randn(g, nb, Hq) if nb else None)
    held = torch.zeros(total, size, dtype=torch.bool)
    for b, n in enumerate(lens):
        for j in range(n):
            held[pt[b, j // size], j % size] = True
    s["k"][~held], s["v"][~held] = float("nan"), float("nan")
    return s


def _run(s, gpu=None, scale=None, md=40, both=False):
    from rgd_triton_amd import paged_decode_attn_func

    gpu = gpu or {}
    a = {n: gpu[n] if n in gpu else (None if t is None else dev(t)) for n, t in s.items()}
    return paged_decode_attn_func(a["q"], a["k"], a["v"], a["pages"], a["lens"], rel_weight=a["w"], max_distance=md, bidirectional=both,
                                  softmax_scale=scale, return_lse=True)


def _ref(s, scale=None, md=40, both=False):
    scale = scale or s["q"].shape[3] ** -0.5
    return serving_oracle.decode(s["q"], s["k"], s["v"], s["pages"], s["lens"], scale, s["w"], md, both)


@pytest.mark.parametrize("case", CASES)
def test_decode_matches_definition(case):
    s = _inputs(case, 300 + CASES.index(case))
    o, lse = _run(s)
    assert o.shape == s["q"].shape and o.dtype == case[5] and lse.dtype == torch.float32
    check_decode(o, lse, _ref(s), max(case[4]), case[2])
    empty = s["lens"] == 0
    assert (o.cpu()[empty] == 0).all() and (lse.cpu()[empty] == -math.inf).all()


LENGTHS = [0, 1, 31, 32, 33, 64, 65, 100, 127, 128, 129, 200, 255, 256, 300, 330]
BUNDLES = [  # 2, 4 and 8 key heads whose rows end on a 128-byte line together, and fewer where the head count ends earlier
    (40, 2, 32, 16, LENGTHS, BF, 8),
    (4, 4, 16, 4, LENGTHS * 2, HF, 0),
    (8, 8, 80, 16, LENGTHS, HF, 32),
    (8, 8, 112, 48, LENGTHS, BF, 0),
    (16, 8, 59, 8, LENGTHS, BF, 0),
    (8, 8, 40, 5, LENGTHS, HF, 16),
    (12, 12, 80, 16, LENGTHS, BF, 0),
    (6, 6, 5, 16, LENGTHS, BF, 0),
    (8, 8, 40, 16, [4000, 1, 3999, 0, 2500, 3000, 4000, 3500], BF, 16),
]


@pytest.mark.parametrize("case", BUNDLES)
def test_decode_heads_that_share_lines(case):
    s = _inputs(case, 370 + BUNDLES.index(case))
    o, lse = _run(s)
    check_decode(o, lse, _ref(s), max(case[4]), case[2])


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("nb,md,wdtype", [(32, 128, FP), (64, 600, BF), (8, 5, HF), (256, 300, FP)])
def test_decode_relative_bias(nb, md, wdtype, both):
    """all distances around the borders of the buckets, lengths inside and beyond max_distance"""
    case = (6, 2, 64, 16, [1, 4, 33, 129, 130, 601, 1500], BF, nb)
    s = _inputs(case, 330)
    s["w"] = (2 * s["w"]).to(wdtype)
    o, lse = _run(s, md=md, both=both)
    check_decode(o, lse, _ref(s, md=md, both=both), 1500, 64)


@pytest.mark.parametrize("scale", [0.3, -0.2, 2.5])
def test_decode_softmax_scale(scale):
    s = _inputs((4, 2, 64, 16, [70, 300], BF, 8), 340)
    o, lse = _run(s, scale=scale)
    check_decode(o, lse, _ref(s, scale=scale), 300, 64)


@pytest.mark.parametrize("D", [64, 128, 80])
def test_decode_layouts(D):
    """head-major caches, gaps, keys and values side by side, unaligned starts, a wider page table, q from a packed buffer"""
    case = (4, 2, D, 16, [70, 15, 0, 290], HF, 8)
    s = _inputs(case, 350)
    ref = _ref(s)
    head_major = lambda t: dev(t.transpose(1, 2).contiguous()).transpose(1, 2)  # noqa: E731
    pair = dev(torch.stack([s["k"], s["v"]], dim=1))
    odd = lambda t: dev(torch.nn.functional.pad(t, (3, 2), value=float("nan")))[..., 3:-2]  # noqa: E731
    packed = dev(torch.cat([s["q"], s["q"], s["q"]], dim=2))
    for name, gpu in {
        "head major": dict(k=head_major(s["k"]), v=head_major(s["v"])),
        "gaps": dict(k=dev(spread(s["k"], (1, 2))), v=dev(spread(s["v"], (3,)))),
        "side by side": dict(k=pair[:, 0], v=pair[:, 1]),
        "odd keys": dict(k=odd(s["k"])),
        "odd values": dict(v=odd(s["v"])),
        "odd query": dict(q=odd(s["q"])),
        "packed query": dict(q=packed[:, :, 4:8]),
        "wide table": dict(pages=dev(torch.nn.functional.pad(s["pages"], (1, 4), value=-7))[:, 1:-4]),
        "weight view": dict(w=dev(spread(s["w"], (1,)))),
    }.items():
        o, lse = _run(s, gpu)
        check_decode(o, lse, ref, 290, D, name)


def test_decode_bad_pages_and_lengths():
    """pages that do not exist hold no keys; lengths below zero are zero, lengths beyond the table end there (the kernel checks
    both before it forms an address)"""
    case = (4, 2, 64, 4, [50, 50, 50, 50, 50], BF, 8)
    s = _inputs(case, 360, extra=2)
    s["pages"][0, 3] = -1
    s["pages"][0, 5] = s["k"].shape[0]
    s["pages"][1, :] = -1
    s["pages"][2, 0] = 2**31 - 1
    s["pages"][2, 12] = -(2**31)
    s["lens"] = torch.tensor([50, 50, 50, -1, 50], dtype=torch.int32)
    check_decode(*_run(s), _ref(s), 50, 64)
    s["lens"] = torch.tensor([49, 0, -(2**31), 2**31 - 1, 1], dtype=torch.int32)
    for page in s["pages"][3]:
        s["k"][page], s["v"][page] = 0.5, 0.25  # the whole table is seen
    check_decode(*_run(s), _ref(s), 52, 64)


def test_decode_masked_rows():
    """-inf and the type's lowest value as bias: single keys, every key but one, every key of a row"""
    case = (4, 4, 64, 16, [1, 3, 40, 200], BF, 8)
    s = _inputs(case, 370)
    low = torch.finfo(FP).min
    w = s["w"]
    w[0, 0] = -math.inf  # the newest key hidden: with one key nothing is left
    w[:, 1] = -math.inf  # every key hidden
    w[:, 2] = low  # every key equally low: the logits vanish beside it, all keys weigh the same
    w[7, 3] = low  # the far ones as good as hidden
    o, lse = _run(s)
    assert not torch.isnan(o.float()).any() and not torch.isnan(lse).any()
    ref = _ref(s)
    assert (o.cpu()[:, 0, 1] == 0).all() and (lse.cpu()[:, 1] == -math.inf).all()
    assert (o.cpu()[0, 0, 0] == 0).all() and lse[0, 0].item() == -math.inf
    # head 2: in 64 bits the logits still differ beside -3.4e38, in 32 bits they do not; the mean over the keys it is
    for b, n in enumerate(case[4]):
        page, slot = s["pages"][b, torch.arange(n) // 16].long(), torch.arange(n) % 16
        mean = s["v"][page, slot, 2].double().mean(0)
        tol = 2.0**-8 * mean.abs() + 2.0**-14 * s["v"][page, slot, 2].double().abs().mean(0)
        assert ((o[b, 0, 2].cpu().double() - mean).abs() <= tol).all()
    keep = [0, 1, 3]
    check_decode(o[:, :, keep], lse[:, keep], (ref[0][:, :, keep], ref[1][:, keep], ref[2][:, :, keep], ref[3][:, keep]), 200, 64)


def test_decode_infinities_and_nan():
    """NaN in a seen key makes its sequence's heads NaN and no others; NaN in a seen value its channel; +inf as a value is +inf;
    a key of -inf weighs nothing"""
    case = (2, 2, 64, 16, [40, 40, 40, 33], HF, 0)
    s = _inputs(case, 380)
    at = lambda b, j: (int(s["pages"][b, j // 16]), j % 16)  # noqa: E731
    s["k"][at(0, 7) + (0, 3)] = float("nan")
    s["v"][at(1, 39) + (1, 5)] = float("nan")
    s["v"][at(3, 32) + (0, 9)] = float("inf")  # the last key, alone in the last tile of 32
    s["q"][2, 0, 0, 4] = 1.0
    s["k"][at(2, 11) + (0, 4)] = -float("inf")
    s["v"][at(2, 11) + (0,)] = 1000.0
    o, _ = _run(s)
    o = o.cpu()
    assert torch.isnan(o[0, 0, 0]).all() and not torch.isnan(o[0, 0, 1]).any()
    assert torch.isnan(o[1, 0, 1, 5]) and torch.isnan(o[1].float()).sum() == 1
    assert o[3, 0, 0, 9] == math.inf and torch.isfinite(o[3].float()).sum() == 127
    ref = _ref(s)
    check_decode(o[2:3], None, tuple(t[2:3] for t in ref), 40, 64)


def test_decode_large_logits():
    """a maximum that moves late and far: the running maximum is raised in the last keys, and falls behind in the first"""
    case = (2, 1, 128, 16, [900, 901], HF, 0)
    s = _inputs(case, 390)
    for b, j in ((0, 899), (1, 0)):
        page, slot = int(s["pages"][b, j // 16]), j % 16
        s["k"][page, slot, 0] = 8 * s["q"][b, 0, 0]
    o, lse = _run(s)
    check_decode(o, lse, _ref(s), 901, 128)


@pytest.mark.parametrize("B,Hq,pages", [(0, 4, 3), (3, 0, 3), (3, 4, 0)])
def test_decode_empty(B, Hq, pages):
    from rgd_triton_amd import paged_decode_attn_func

    q, k = torch.randn(B, 1, Hq, 64, device="cuda").to(BF), torch.randn(pages, 16, 2, 64, device="cuda").to(BF)
    table = torch.zeros(B, 2 if pages else 0, dtype=torch.int32, device="cuda")
    o, lse = paged_decode_attn_func(q, k, k, table, torch.full((B,), 5, dtype=torch.int32, device="cuda"), return_lse=True)
    assert o.shape == q.shape and lse.shape == (B, Hq)
    if pages == 0:
        assert (o == 0).all() and (lse == -math.inf).all()


def test_decode_reproducible_and_on_streams():
    """many lengths, so that sequences share workgroups and workgroups sequences: the same bits every time, also from two streams
    at once"""
    lens = [int(n) for n in torch.randint(0, 900, (64,), generator=gen(5))]
    s = {n: (None if t is None else t.cuda()) for n, t in _inputs((8, 2, 64, 16, lens, BF, 0), 400).items()}
    first = _run(s, s)
    other = {n: (None if t is None else t.cuda()) for n, t in _inputs((4, 4, 128, 8, lens[:20], HF, 8), 401).items()}
    second = _run(other, other)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(20):
        with torch.cuda.stream(a):
            outs.append((_run(s, s), first))
        with torch.cuda.stream(b):
            outs.append((_run(other, other), second))
    torch.cuda.synchronize()
    for got, want in outs:
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_decode_cache_beyond_32_bits():
    """pages whose elements start behind 2^31 and bytes behind 2^32"""
    from rgd_triton_amd import paged_decode_attn_func

    size, Hkv, D, B, n = 64, 4, 128, 2, 150
    total = (2**31 + 2**26) // (size * Hkv * D)
    g = gen(410)
    k, v = (torch.empty(total, size, Hkv, D, dtype=BF, device="cuda") for _ in range(2))
    table = torch.tensor([[total - 1, 3, total - 2], [total // 2, total - 3, 0]], dtype=torch.int32)
    for page in table.flatten().tolist():
        k[page], v[page] = randn(g, size, Hkv, D, dtype=BF).cuda(), randn(g, size, Hkv, D, dtype=BF).cuda()
    q = randn(g, B, 1, 8, D, dtype=BF)
    lens = torch.tensor([n, n - 1], dtype=torch.int32)
    o, lse = paged_decode_attn_func(q.cuda(), k, v, table.cuda(), lens.cuda(), return_lse=True)
    order = table.flatten().long()
    small = torch.arange(6, dtype=torch.int32).reshape(2, 3)
    ref = serving_oracle.decode(q, k[order.cuda()].cpu(), v[order.cuda()].cpu(), small, lens, D**-0.5)
    check_decode(o, lse, ref, n, D)
