"""RoPECacheAppend / FusedLNRoPECacheAppend against the definition in 64 bits: the rotated query, the slots of the new tokens, and
every other slot of the cache left as it was, bit for bit."""
import pytest
import torch

from serving_helpers import dev, gen, pages_for, randn, rotary, rounded_once, serving_oracle, spread

pytestmark = pytest.mark.gpu

BF, HF, FP = torch.bfloat16, torch.float16, torch.float32
CASES = [  # B, T, Hq, Hkv, D, R, page, dtype, table, layer norm, ragged, heads_second
    (1, 1, 1, 1, 64, 64, 16, BF, FP, False, False, False),
    (3, 1, 8, 2, 128, 128, 16, BF, BF, False, False, False),
    (3, 1, 8, 2, 128, 64, 16, HF, HF, True, False, True),
    (2, 37, 4, 4, 64, 32, 16, BF, FP, False, True, True),
    (2, 37, 4, 4, 64, 32, 5, HF, FP, True, True, False),
    (4, 19, 3, 1, 59, 30, 7, BF, BF, False, True, False),
    (2, 9, 3, 3, 59, 58, 1, HF, FP, True, False, True),
    (1, 300, 2, 1, 32, 32, 64, BF, BF, True, False, False),
    (5, 3, 5, 5, 80, 40, 48, HF, FP, False, True, False),
    (2, 6, 2, 2, 8, 8, 3, BF, FP, True, False, False),
    (2, 6, 2, 2, 2, 2, 3, BF, FP, False, False, True),
    (2, 6, 2, 1, 1, 0, 3, BF, FP, False, False, False),
    (3, 11, 6, 2, 96, 0, 16, HF, FP, True, False, False),
    (3, 11, 6, 2, 112, 20, 8, BF, BF, False, False, False),
    (2, 5, 5, 3, 100, 50, 8, BF, BF, True, False, True),
    (2, 5, 3, 3, 127, 126, 8, HF, FP, True, False, False),
    (2, 5, 3, 1, 9, 8, 8, BF, FP, False, False, False),
    (2, 5, 3, 1, 33, 2, 8, HF, HF, True, False, False),
    (1, 5, 1, 1, 7, 6, 8, BF, FP, True, False, True),
    (2, 5, 7, 2, 122, 122, 8, HF, FP, False, True, True),
]


def _inputs(case, seed, cap=None):
    B, T, Hq, Hkv, D, R, size, dtype, table, ln, ragged, hs = case
    g = gen(seed)
    cap = cap or T + 2 * size + 5
    total, pt = pages_for(g, B, cap, size)
    s = dict(q=randn(g, B, Hq, T, D, dtype=dtype, shift=0.2), k=randn(g, B, Hkv, T, D, dtype=dtype, shift=-0.1),
             v=randn(g, B, Hkv, T, D, dtype=dtype), k_cache=randn(g, total, size, Hkv, D, dtype=dtype),
             v_cache=randn(g, total, size, Hkv, D, dtype=dtype), pages=pt,
             lens=torch.randint(0, cap - T + 1, (B,), generator=g, dtype=torch.int32),
             new=torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32) if ragged else None,
             table=rotary(pt.shape[1] * size, R, table) if R else None)
    return s


def _check(case, s, gpu=None, cutoff=None, eps=1e-6):
    from rgd_triton_amd import rope_cache_append_fn

    dtype, ln, hs = case[7], case[9], case[11]
    gpu = gpu or {}
    place = lambda n: gpu[n] if n in gpu else (None if s[n] is None else dev(s[n]))  # noqa: E731
    layout = lambda n: gpu[n] if n in gpu else dev(s[n] if hs else s[n].transpose(1, 2).contiguous())  # noqa: E731
    kc, vc = place("k_cache"), place("v_cache")
    q = layout("q")
    got = rope_cache_append_fn(q, layout("k"), layout("v"), place("table"), kc, vc, place("pages"), place("lens"),
                               new_lens=place("new"), seq_cutoff=cutoff, heads_second=hs, norm_eps=eps if ln else None)
    assert got.shape == q.shape and got.dtype == dtype
    got = got if hs else got.transpose(1, 2)
    qo, rk, rv, written = serving_oracle.append(s["q"], s["k"], s["v"], s["table"], s["k_cache"], s["v_cache"], s["pages"], s["lens"],
                                                s["new"], cutoff, eps if ln else None)
    # 32-bit arithmetic in front of the one rounding: the norm's D-term sums and a few operations, the pair's two products;
    # relative to the largest element that enters (a normalised element is at most sqrt(D) long)
    D = case[4]
    size = lambda x: (D**0.5 if ln else 1.0) * (1.0 if ln else x.double().abs().max().item())  # noqa: E731
    steps = (2 * D + 16 if ln else 4) * 2.0**-24
    rounded_once(got, qo, torch.full_like(qo, 2 * steps * size(s["q"])), "q")
    rounded_once(kc, rk, (2 * steps * size(s["k"]) * written.double())[:, :, None, None].expand_as(rk), "k cache")
    for name, now in (("k_cache", kc), ("v_cache", vc)):
        assert torch.equal(now.cpu()[~written], s[name][~written]), f"{name}: a slot of no new token changed"
    assert torch.equal(vc.cpu().double(), rv), "v cache"
    if case[5] == 0 and not ln:
        assert torch.equal(kc.cpu().double(), rk)
    return written


@pytest.mark.parametrize("case", CASES)
def test_append_matches_definition(case):
    written = _check(case, _inputs(case, 200 + CASES.index(case)))
    assert case[10] or int(written.sum()) == case[0] * case[1]


@pytest.mark.parametrize("cutoff", [0, 9, (4, 20)])
def test_append_cutoff(cutoff):
    case = (3, 12, 4, 2, 64, 32, 8, BF, FP, False, False, True)
    _check(case, _inputs(case, 230), cutoff=cutoff)


@pytest.mark.parametrize("ln", [False, True])
@pytest.mark.parametrize("hs", [False, True])
def test_append_layouts(hs, ln):
    """inputs with gaps between rows, head-major and gapped caches, a wider page table, an odd start, a table with gaps"""
    case = (2, 13, 4, 2, 64, 32, 16, BF, BF, ln, True, hs)
    s = _inputs(case, 240)
    lay = lambda t: t if hs else t.transpose(1, 2).contiguous()  # noqa: E731
    packed = torch.cat([lay(s["q"]), lay(s["k"]), lay(s["v"])], dim=1 if hs else 2)  # one buffer for q, k and v
    pk = dev(packed)
    cut = lambda a, b: pk[:, a:b] if hs else pk[:, :, a:b]  # noqa: E731
    _check(case, s, dict(q=cut(0, 4), k=cut(4, 6), v=cut(6, 8)))
    head_major = lambda t: dev(t.transpose(1, 2).contiguous()).transpose(1, 2)  # noqa: E731
    _check(case, s, dict(k_cache=head_major(s["k_cache"]), v_cache=dev(spread(s["v_cache"], (1, 2)))))
    _check(case, s, dict(k_cache=dev(spread(s["k_cache"], (3,))), v_cache=dev(torch.nn.functional.pad(s["v_cache"], (3, 2)))[..., 3:-2]))
    both = torch.stack([s["k_cache"], s["v_cache"]], dim=1)  # keys and values of a page side by side
    bg = dev(both)
    wide = dev(torch.nn.functional.pad(s["pages"], (1, 4), value=-1))[:, 1:-4]
    _check(case, s, dict(k_cache=bg[:, 0], v_cache=bg[:, 1], pages=wide, table=dev(spread(s["table"], (1, 2)))))
    odd = torch.nn.functional.pad(lay(s["q"]), (1, 0))
    _check(case, s, dict(q=dev(odd)[..., 1:]))


def test_append_bad_pages_and_positions():
    """pages that do not exist, lengths below zero and beyond the table, more new tokens than there are: dropped, nothing else
    touched (bounds that the host oracle states; the kernel checks them before it forms an address)"""
    case = (6, 9, 4, 2, 64, 64, 4, BF, FP, False, True, False)
    s = _inputs(case, 250, cap=24)
    s["lens"] = torch.tensor([0, -3, 20, 24, 2**31 - 1, -(2**31)], dtype=torch.int32)
    s["new"] = torch.tensor([9, 99, 9, 2**31 - 1, 9, -5], dtype=torch.int32)
    s["pages"][0, 1] = -1
    s["pages"][0, 2] = s["k_cache"].shape[0]
    s["pages"][2, 5] = 2**31 - 1
    s["pages"][1, 0] = -(2**31)
    _check(case, s)


def test_append_in_place_query_and_version():
    """the C ABI allows the rotated query in the query's own place, also where lanes of a row overlap"""
    from rgd_triton_amd import RoPECacheAppend, _hip, rope_cache_append_fn

    for D, R in ((64, 64), (100, 60), (59, 58)):
        case = (2, 3, 3, 4, D, R, 16, BF, FP, True, False, True)
        s = {n: (None if t is None else t.cuda()) for n, t in _inputs(case, 260).items()}
        want = rope_cache_append_fn(s["q"], s["k"], s["v"], s["table"], s["k_cache"], s["v_cache"], s["pages"], s["lens"], norm_eps=1e-6)
        d4 = lambda t, h, n: (t.data_ptr(), t.stride(0), t.stride(h), t.stride(n))  # noqa: E731
        args = _hip.append_args(
            2, 3, 3, 4, D, *d4(s["q"], 1, 2), *d4(s["k"], 1, 2), *d4(s["v"], 1, 2), *d4(s["q"], 1, 2), *d4(s["k_cache"], 2, 1),
            *d4(s["v_cache"], 2, 1), s["k_cache"].shape[0], 16, s["pages"].data_ptr(), s["pages"].shape[1], s["pages"].stride(0),
            s["lens"].data_ptr(), 0, s["table"].data_ptr(), s["table"].shape[1], R, s["table"].stride(0), s["table"].stride(1), 2**31 - 1,
            2**31 - 1, 0, 1, 2, 1e-6)
        rc = _hip.lib().rgd_rope_cache_append(args, _hip.stream_ptr(s["q"].device))
        assert rc == 0 and torch.equal(s["q"], want)
    case = (2, 3, 4, 4, 64, 64, 16, BF, FP, False, False, True)
    s = {n: (None if t is None else t.cuda()) for n, t in _inputs(case, 260).items()}
    before = s["k_cache"]._version
    RoPECacheAppend()(s["q"], s["k"], s["v"], s["table"], s["k_cache"], s["v_cache"], s["pages"], s["lens"])
    assert s["k_cache"]._version > before and s["v_cache"]._version > 0  # an in-place write that autograd can see


@pytest.mark.parametrize("B,T,Hq,Hkv", [(0, 3, 2, 2), (2, 0, 2, 2), (2, 3, 0, 2), (2, 3, 2, 0)])
def test_append_empty(B, T, Hq, Hkv):
    case = (B, T, Hq, Hkv, 64, 32, 16, BF, FP, False, False, True)
    g = gen(270)
    s = dict(q=randn(g, B, Hq, T, 64, dtype=BF), k=randn(g, B, Hkv, T, 64, dtype=BF), v=randn(g, B, Hkv, T, 64, dtype=BF),
             k_cache=randn(g, 9, 16, Hkv, 64, dtype=BF), v_cache=randn(g, 9, 16, Hkv, 64, dtype=BF),
             pages=torch.arange(B * 2, dtype=torch.int32).reshape(B, 2), lens=torch.full((B,), 3, dtype=torch.int32), new=None,
             table=rotary(32, 32))
    from rgd_triton_amd import rope_cache_append_fn

    d = {n: (None if t is None else t.cuda()) for n, t in s.items()}
    out = rope_cache_append_fn(d["q"], d["k"], d["v"], d["table"], d["k_cache"], d["v_cache"], d["pages"], d["lens"])
    torch.cuda.synchronize()
    assert out.shape == s["q"].shape
    if s["q"].numel() and Hkv == 0:
        qo = serving_oracle.append(s["q"], s["k"], s["v"], s["table"], s["k_cache"], s["v_cache"], s["pages"], s["lens"])[0]
        rounded_once(out, qo, torch.full_like(qo, 2.0**-20), "q")
    if T == 0 or B == 0:
        assert torch.equal(d["k_cache"].cpu(), s["k_cache"])


def test_append_special_values():
    """infinities and NaN in a row stay in that row (no norm) and reach the cache as torch arithmetic has them"""
    case = (1, 4, 2, 2, 64, 0, 4, HF, FP, False, False, True)
    s = _inputs(case, 280)
    s["k"][0, 0, 1, 5], s["v"][0, 1, 2, 7], s["q"][0, 0, 3, 0] = float("inf"), float("nan"), float("-inf")
    from rgd_triton_amd import rope_cache_append_fn

    d = {n: (None if t is None else t.cuda()) for n, t in s.items()}
    out = rope_cache_append_fn(d["q"], d["k"], d["v"], None, d["k_cache"], d["v_cache"], d["pages"], d["lens"])
    assert torch.equal(out.cpu(), s["q"])
    for t in range(4):
        pos = int(s["lens"][0]) + t
        page, slot = int(s["pages"][0, pos // 4]), pos % 4
        assert torch.equal(d["k_cache"][page, slot].cpu(), s["k"][0, :, t])
        assert torch.equal(d["v_cache"][page, slot].cpu().view(torch.int16), s["v"][0, :, t].contiguous().view(torch.int16))
