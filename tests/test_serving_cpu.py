"""CPU side of the cache, decode and relative-bias operators: the oracle against independent formulas, the buckets, and everything
that is refused before a kernel is launched."""
import bisect
import ctypes
import inspect
import math
import re
import struct

import pytest
import torch

from serving_helpers import gen, randn, rotary, serving_oracle

from rgd_triton_amd import _hip

T4 = _hip.desc4(0x1000, 4096, 64, 64)
D4 = (0x1000, 4096, 64, 64)
BUF = ctypes.c_void_p(0x1000)


# ------------------------------------------------------------------ oracle and buckets


@pytest.mark.parametrize("both", [False, True])
@pytest.mark.parametrize("nb,md", [(4, 9), (8, 5), (8, 20), (32, 128), (32, 127), (64, 700), (256, 900), (5, 40), (2, 3)])
def test_buckets_against_their_logarithm(nb, md, both):
    """away from the borders floor(log) decides, at the borders (a power hits them exactly) the next bucket begins; the ranges of
    the package say the same"""
    from rgd_triton_amd.functional import relative_ranges

    if both and nb % 2:
        pytest.skip("bidirectional buckets are even")
    if both and nb < 4:
        pytest.skip("bidirectional buckets need two a side")
    r = relative_ranges(nb, md, both)
    assert list(r.starts) == sorted(set(r.starts)) and len(set(r.buckets)) == r.n
    side = nb // 2 if both else nb
    e = side // 2
    for d in range(-md - 50, md + 51):
        b = serving_oracle.bucket_of(d, nb, md, both)
        assert b == r.buckets[bisect.bisect_right(r.starts, d) - 1]
        n = abs(d) if both else max(-d, 0)
        if n >= e:
            x = e + math.log(n / e) / math.log(md / e) * (side - e)
            if abs(x - round(x)) > 1e-9:
                assert b % side == min(side - 1, int(x)), (d, b, x)
            else:
                assert b % side == min(side - 1, round(x))
        else:
            assert b % side == n
        assert b // side == int(both and d > 0)


def test_oracle_rotation_is_complex_multiplication():
    g = gen(1)
    x, pe = randn(g, 10).double(), rotary(30, 6, torch.float64)
    y = serving_oracle.rotate_row(x, pe[0, 17], pe[1, 17])
    z = torch.view_as_complex(x[:6].reshape(3, 2).contiguous()) * torch.polar(torch.ones(3, dtype=torch.float64), 17 * 10000.0 ** (-torch.arange(0, 6, 2).double() / 6))
    assert torch.allclose(y[:6], torch.view_as_real(z).reshape(-1), atol=1e-12) and torch.equal(y[6:], x[6:])


def test_oracle_decode_is_softmax_attention():
    g = gen(2)
    q, k, v = randn(g, 1, 1, 4, 8), randn(g, 4, 3, 2, 8), randn(g, 4, 3, 2, 8)
    table = torch.tensor([[2, 0, 3]], dtype=torch.int32)
    o, lse, _, _ = serving_oracle.decode(q, k, v, table, torch.tensor([7]), 0.5)
    kk, vv = (c[[2, 0, 3]].reshape(9, 2, 8)[:7].double() for c in (k, v))
    for h in range(4):
        s = 0.5 * kk[:, h // 2] @ q[0, 0, h].double()
        assert torch.allclose(o[0, 0, h], torch.softmax(s, 0) @ vv[:, h // 2]) and torch.allclose(lse[0, h], torch.logsumexp(s, 0))


def test_oracle_bias_gradient_against_differences():
    g = gen(3)
    w, dy = randn(g, 8, 2).double(), randn(g, 1, 2, 9, 13).double()
    grad, mag = serving_oracle.relative_bias_grad(dy, 8, 6, True, 2)
    f = lambda t: (serving_oracle.relative_bias(t, 9, 13, 6, True, 2) * dy).sum()  # noqa: E731
    for b in range(8):
        e = torch.zeros_like(w)
        e[b, 1] = 1.0
        assert abs(f(w + e) - f(w) - grad[b, 1]) < 1e-10
    assert (mag >= grad.abs()).all()


# ------------------------------------------------------------------ refusals


def _packed(pack, a):
    """an argument structure from its members in order: descriptors as tuples, None for a null pointer or descriptor"""
    flat = []
    for name, x in a.items():
        if x is None:
            x = (0, 0, 0, 0) if name in ("q", "k", "v", "qo", "kc", "vc", "o") else 0
        flat += x if isinstance(x, tuple) else (x,)
    return pack(*flat)


def _append(**kw):
    a = dict(B=1, T=2, Hq=4, Hkv=2, D=64, q=D4, k=D4, v=D4, qo=D4, kc=D4, vc=D4, pages=8, size=16, table=0x1000, per=4, stride=4,
             lens=0x1000, new=None, pe=0x1000, P=64, R=64, ss=4096, sn=64, cq=99, ck=99, pdt=0, ln=0, dt=2, eps=0.0)
    a.update(kw)
    return _hip.lib().rgd_rope_cache_append(_packed(_hip.append_args, a), None)


def _decode(**kw):
    a = dict(B=1, Hq=4, Hkv=2, D=64, q=D4, kc=D4, vc=D4, o=D4, pages=8, size=16, table=0x1000, per=4, stride=4, lens=0x1000, w=None, ws=0,
             nb=0, n=0, starts=None, buckets=None, lse=None, work=0x1000, bytes=1 << 30, wdt=0, dt=2, scale=0.125)
    a.update(kw)
    return _hip.lib().rgd_paged_decode(_packed(_hip.decode_args, a), None)


@pytest.mark.parametrize("name,pack", [("rgd_cache_append_args", _hip.append_args), ("rgd_paged_decode_args", _hip.decode_args)])
def test_argument_structures_are_the_headers(name, pack):
    """the packed bytes have the members of the header's structure, in its order"""
    text = re.sub(r"/\*.*?\*/", "", open(_hip.HEADER_PATH).read(), flags=re.S)
    body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (name, name), text, flags=re.S).group(1)
    kinds = {"int64_t": "q", "int32_t": "i", "float": "f", "size_t": "N", "rgd_tensor4": "Pqqq"}
    want = ""
    for line in filter(None, (x.strip() for x in body.split(";"))):
        kind, names = re.match(r"((?:const )?\w+ ?\*?) ?(.*)", line, flags=re.S).groups()
        want += ("P" if "*" in line else kinds[kind.strip()]) * len(names.split(","))
    fmt = re.sub(r"(\d+)([a-zA-Z])", lambda m: m.group(2) * int(m.group(1)), pack.__self__.format.lstrip("@"))
    assert fmt.rstrip("x") == want
    assert len(fmt) - len(want) == -struct.calcsize("@" + want) % 8  # padded to the structure's alignment


def test_append_refusals():
    err = lambda: _hip.lib().rgd_last_error()  # noqa: E731
    assert _append(dt=0) == -1 and b"Only support fp16 and bf16" in err()
    assert _append(dt=9) == -1
    assert _append(D=129) == -1 and b"head dimensions up to 128" in err()
    assert _append(B=-1) == -1 and _append(pages=-1) == -1
    assert _append(size=0) == -1 and b"page size" in err()
    assert _append(R=66) == -1 and b"rotary dim" in err()
    assert _append(R=63) == -1 and b"even" in err()
    assert _append(P=63) == -1 and b"every position" in err()
    assert _append(pe=None) == -1 and b"pos_emb" in err()
    assert _append(pdt=1) == -2 and b"pos_emb must have" in err()
    assert _append(lens=None) == -1 and _append(table=None) == -1
    assert _append(q=None) == -1 and _append(vc=None) == -1 and b"null tensor" in err()
    assert _append(size=1 << 20, per=1 << 12) == -2 and b"2^31" in err()
    assert _append(B=1 << 20, T=1 << 12) == -2
    assert _append(B=1 << 14, T=1 << 14, Hq=2, Hkv=1) == -2 and b"one launch" in err()
    assert _hip.lib().rgd_rope_cache_append(None, None) == -1 and b"null arguments" in err()
    # nothing to do is no error
    assert _append(T=0) == 0 and _append(B=0) == 0 and _append(Hq=0, Hkv=0) == 0


def test_decode_refusals():
    err = lambda: _hip.lib().rgd_last_error()  # noqa: E731
    assert _decode(dt=0) == -1 and b"Only support fp16 and bf16" in err()
    assert _decode(D=129) == -1 and b"head dimensions up to 128" in err()
    assert _decode(D=0) == -1 and _decode(Hq=-1) == -1
    assert _decode(Hq=5) == -1 and b"multiple of the key heads" in err()
    assert _decode(Hkv=0) == -1
    assert _decode(size=0) == -1
    assert _decode(lens=None) == -1 and _decode(table=None) == -1 and _decode(kc=None) == -1
    assert _decode(q=None) == -1 and _decode(o=None) == -1
    assert _decode(size=1 << 20, per=1 << 12) == -2
    assert _decode(B=1 << 22, Hq=4) == -2 and b"query rows" in err()
    up, down, ids = (ctypes.c_int32 * 3)(-5, 0, 3), (ctypes.c_int32 * 3)(-5, 3, 0), (ctypes.c_int32 * 3)(0, 1, 2)
    starts, buckets = ctypes.addressof(up), ctypes.addressof(ids)
    rel = dict(w=0x1000, ws=4, nb=3, n=3, starts=starts, buckets=buckets)
    assert _decode(**{**rel, "wdt": 7}) == -1 and b"bias weights" in err()
    assert _decode(**{**rel, "nb": 2}) == -1 and b"bucket outside" in err()
    assert _decode(**{**rel, "n": 0}) == -1 and _decode(**{**rel, "n": 257}) == -1 and _decode(**{**rel, "starts": None}) == -1
    assert _decode(**{**rel, "starts": ctypes.addressof(down)}) == -1 and b"ascend" in err()
    need = _hip.lib().rgd_paged_decode_workspace(1, 4, 2, 64)
    assert need > 0 and _decode(bytes=need - 1) == -4 and b"workspace" in err() and _decode(work=None) == -4
    assert _hip.lib().rgd_paged_decode(None, None) == -1 and b"null arguments" in err()
    assert _decode(B=0) == 0 and _decode(Hq=0, Hkv=1) == 0


def test_rel_bias_refusals():
    lib = _hip.lib()
    err = lib.rgd_last_error
    up, down = (ctypes.c_int32 * 3)(-5, 0, 3), (ctypes.c_int32 * 3)(-5, 3, 0)
    ids, twice = (ctypes.c_int32 * 3)(2, 1, 0), (ctypes.c_int32 * 3)(0, 1, 1)

    def fwd(**kw):
        a = dict(H=2, Tq=4, Tk=4, w=BUF, ws=2, nb=3, wdt=0, n=3, starts=up, buckets=ids, off=0, bias=T4, bdt=0, work=None, bytes=0)
        a.update(kw)
        return lib.rgd_rel_bias_fwd(*a.values(), None)

    def bwd(**kw):
        a = dict(H=2, Tq=4, Tk=4, d=T4, ddt=0, n=3, starts=up, buckets=ids, off=0, dw=BUF, ws=2, nb=3, wdt=0, work=BUF, bytes=1 << 20)
        a.update(kw)
        return lib.rgd_rel_bias_bwd(*a.values(), None)

    for f in (fwd, bwd):
        assert f(wdt=3) == -1 and b"Only support" in err()
        assert f(Tq=-1) == -1 and f(H=70000) == -2 and f(Tk=1 << 30) == -2 and f(off=1 << 30) == -2 and f(off=-(1 << 30)) == -2
        assert f(Tq=1 << 29, Tk=1 << 29, off=(1 << 30) - 1) == -2 and b"distances" in err()
        assert f(n=0) == -1 and f(n=257) == -1 and f(nb=257) == -1 and f(starts=None) == -1
        assert f(starts=down) == -1 and b"ascend" in err()
        assert f(buckets=twice) == -1 and b"two ranges" in err()
        assert f(nb=2) == -1 and b"outside the weight" in err()
        assert f(H=0) == 0
    assert fwd(w=None) == -1 and fwd(bias=None) == -1 and bwd(d=None) == -1 and bwd(dw=None) == -1
    assert bwd(bytes=16) == -4 and b"workspace" in err()
    assert lib.rgd_rel_bias_bwd_workspace(0, 5, 5, 8) == 0 and lib.rgd_rel_bias_bwd_workspace(3, 5, 5, 8) > 0
    assert fwd(Tq=0) == 0
    # scratch only where the matrix is written in address order: beyond 64 MB
    assert lib.rgd_rel_bias_fwd_workspace(8, 2048, 2048, 2) == 0 and lib.rgd_rel_bias_fwd_workspace(8, 2048, 2049, 2) > 0
    assert lib.rgd_rel_bias_fwd_workspace(8, 2048, 2048, 0) > 0 and lib.rgd_rel_bias_fwd_workspace(1, 1 << 30, 8, 0) == 0


def test_ranges_refusals():
    from rgd_triton_amd import RelativePositionBias
    from rgd_triton_amd.functional import relative_ranges

    for args in ((1, 128, False), (257, 1000, False), (33, 128, True), (2, 128, True), (32, 16, False), (32, 8, True), (32, 2**30, True), (32.0, 128, True)):
        with pytest.raises(AssertionError):
            relative_ranges(*args)
    with pytest.raises(AssertionError):
        RelativePositionBias(31, 4)


def test_python_refusals_on_cpu_tensors_and_arguments():
    import rgd_triton_amd as rgd

    bf = torch.bfloat16
    q, kv = torch.zeros(2, 4, 1, 64, dtype=bf), torch.zeros(2, 2, 1, 64, dtype=bf)
    cache = torch.zeros(6, 16, 2, 64, dtype=bf)
    table, lens, pe = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), rotary(48, 32)

    def app(msg, q=q, k=kv, v=kv, pe=pe, kc=cache, vc=cache, table=table, lens=lens, **kw):
        with pytest.raises(AssertionError, match=msg):
            rgd.rope_cache_append_fn(q, k, v, pe, kc, vc, table, lens, **kw)

    app("GPU only")
    app("same type", k=kv.float())
    app("same type", kc=cache.half(), vc=cache.half())
    app("fp16 and bf16", q=q.float(), k=kv.float(), v=kv.float(), kc=cache.float(), vc=cache.float())
    app("shape", v=torch.zeros(2, 2, 2, 64, dtype=bf))
    app("shape", vc=cache[:5])
    app("shape", kc=cache[:, :, :1], vc=cache[:, :, :1])
    app("128", q=torch.zeros(2, 4, 1, 130, dtype=bf), k=torch.zeros(2, 2, 1, 130, dtype=bf), v=torch.zeros(2, 2, 1, 130, dtype=bf),
        kc=torch.zeros(6, 16, 2, 130, dtype=bf), vc=torch.zeros(6, 16, 2, 130, dtype=bf))
    app("unit-stride", kc=torch.zeros(6, 16, 64, 2, dtype=bf).transpose(2, 3))
    app("int32", table=table.long())
    app("int32", table=table[:1])
    app("int32", lens=lens.long())
    app("int32", new_lens=lens[:1])
    app("every position", pe=pe[:, :47])
    app("rotary dim", pe=rotary(48, 66))
    app("rotary dim", pe=rotary(48, 64)[..., :31])
    app("serving", q=q.clone().requires_grad_(True))
    qd = torch.zeros(2, 1, 4, 64, dtype=bf)

    def dec(msg, q=qd, kc=cache, vc=cache, table=table, lens=lens, **kw):
        with pytest.raises(AssertionError, match=msg):
            rgd.paged_decode_attn_func(q, kc, vc, table, lens, **kw)

    dec("GPU only")
    dec("one new token", q=torch.zeros(2, 2, 4, 64, dtype=bf))
    dec("groups", q=torch.zeros(2, 1, 3, 64, dtype=bf))
    dec("same type", q=qd.half())
    dec("same", q=torch.zeros(2, 1, 4, 32, dtype=bf))
    dec("int32", lens=lens.long())
    dec("rel_weight", rel_weight=torch.zeros(32, 5))
    dec("serving", rel_weight=torch.zeros(32, 4, requires_grad=True))
    dec("GPU only", rel_weight=torch.zeros(32, 4))
    with pytest.raises(AssertionError, match="GPU only"):
        rgd.RelativePositionBias(32, 4)(8, 8)
    with pytest.raises(AssertionError):
        rgd.relative_position_bias_fn(torch.zeros(32, 4, dtype=torch.float64), 8, 8)


def test_module_surface():
    import rgd_triton_amd as rgd

    names = lambda f: [n for n in inspect.signature(f).parameters if n != "self"]  # noqa: E731
    common = ["query", "key", "value", "pos_emb", "k_cache", "v_cache", "page_table", "cache_lens", "new_lens", "seq_cutoff", "heads_second"]
    assert names(rgd.RoPECacheAppend.forward) == common and names(rgd.FusedLNRoPECacheAppend.forward) == common + ["eps"]
    assert names(rgd.PagedDecodeAttention.forward) == ["q", "k_cache", "v_cache", "page_table", "seq_lens", "rel_bias", "softmax_scale"]
    assert names(rgd.RelativePositionBias.forward) == ["seqlen_q", "seqlen_k", "q_offset", "dtype"]
    m = rgd.RelativePositionBias(32, 6, max_distance=200, bidirectional=False, dtype=torch.bfloat16)
    assert m.weight.shape == (32, 6) and m.weight.dtype == torch.bfloat16 and list(m.state_dict()) == ["weight"]
    for cls in (rgd.RoPECacheAppend, rgd.FusedLNRoPECacheAppend, rgd.PagedDecodeAttention):
        c = cls()
        assert c.cache.fwd is None and not list(c.parameters())
        c.enable_cache(False)
        assert c.cache is None
