"""RelativePositionBias against the definition in 64 bits: values bit for bit, the gradient of the weight within the rounding of a
32-bit sum, and the pair with FlashAttention's own bias gradient."""
import pytest
import torch

from serving_helpers import dev, gen, half_step, randn, serving_oracle, spread

pytestmark = pytest.mark.gpu

SHAPES = [  # (Tq, Tk, q_offset)
    (1, 1, 0), (1, 700, 699), (700, 1, 0), (7, 5, 0), (64, 64, 0), (129, 257, 128), (255, 1031, -40), (530, 520, 0), (1025, 300, 5000),
    (520, 1100, 3), (2, 4099, 2048),
]
BUCKETS = [(32, 128, True), (32, 128, False), (8, 20, True), (64, 700, True), (2, 5, False), (5, 9, False), (256, 900, True)]


@pytest.mark.parametrize("Tq,Tk,off", SHAPES)
@pytest.mark.parametrize("wdtype,dtype", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.bfloat16), (torch.float32, torch.float32),
                                          (torch.float16, torch.float16), (torch.bfloat16, torch.float32)])
def test_rel_bias_values_and_gradient(Tq, Tk, off, wdtype, dtype):
    from rgd_triton_amd import relative_position_bias_fn

    i = SHAPES.index((Tq, Tk, off))
    nb, md, both = BUCKETS[(i + int(dtype == torch.float32)) % len(BUCKETS)]
    H = 1 + i % 4
    g = gen(100 + i)
    w, dy = randn(g, nb, H, dtype=wdtype), randn(g, 1, H, Tq, Tk, dtype=dtype, shift=0.3)
    wg = w.cuda().requires_grad_(True)
    bias = relative_position_bias_fn(wg, Tq, Tk, max_distance=md, bidirectional=both, q_offset=off, dtype=dtype)
    assert bias.shape == (1, H, Tq, Tk) and bias.dtype == dtype
    # one rounding of the weight, no arithmetic
    assert torch.equal(bias.detach().cpu(), serving_oracle.relative_bias(w, Tq, Tk, md, both, off).to(dtype))
    (dw,) = torch.autograd.grad(bias, wg, dy.cuda())
    _check_grad(dw, dy, nb, md, both, off)


def _check_grad(dw, dy, nb, md, both, off):
    ref, mag = serving_oracle.relative_bias_grad(dy, nb, md, both, off)
    Tq, Tk = dy.shape[2:]
    # longest chain of additions: at most 8 times 512 in a lane, then the partial sums of a bucket over 256 lanes
    depth = 4096 + (Tq // 512 + 1) * ((Tk + 511) // 256 + 1) + 16
    tol = depth * 2.0**-24 * mag
    # a sum beyond the type's largest number rounds to infinity (the sum of 307500 gradients of mean 0.3 is 92000, fp16 ends at 65504)
    over = ref.abs() - tol > torch.finfo(dw.dtype).max * (1 + half_step(dw.dtype))
    got = dw.cpu().double()
    assert torch.equal(got[over], ref[over].sign() * float("inf"))
    err = torch.where(over, 0.0, (got - ref).abs())
    assert (err <= tol + half_step(dw.dtype) * (ref.abs() + tol)).all(), f"gradient off: {(err - tol).max()}"


@pytest.mark.parametrize("nb,md,both", BUCKETS)
def test_rel_bias_bucket_borders(nb, md, both):
    """every distance from -md - 3 to md + 3, one at a time: which row of the weight is read, and that the gradient of one pair
    goes to that row alone"""
    from rgd_triton_amd import relative_position_bias_fn

    w = torch.arange(nb, dtype=torch.float32)[:, None]
    far = md + 3
    wg = w.cuda().requires_grad_(True)
    bias = relative_position_bias_fn(wg, 1, 2 * far + 1, max_distance=md, bidirectional=both, q_offset=far)
    want = [serving_oracle.bucket_of(d, nb, md, both) for d in range(-far, far + 1)]
    assert bias.flatten().tolist() == [float(b) for b in want]
    dy = torch.arange(1, 2 * far + 2, dtype=torch.float32, device="cuda").reshape(1, 1, 1, -1)
    (dw,) = torch.autograd.grad(bias, wg, dy)
    ref = torch.zeros(nb, dtype=torch.float64)
    for c, b in enumerate(want):
        ref[b] += c + 1
    assert torch.equal(dw.cpu().double()[:, 0], ref)  # whole numbers below 2^24


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rel_bias_gradient_layouts(dtype):
    """rows with gaps, an unaligned start, heads in another order, and an expanded gradient (stride 0)"""
    from rgd_triton_amd import RelativePositionBias

    H, Tq, Tk, g = 3, 77, 203, gen(7)
    m = RelativePositionBias(32, H, device="cuda")
    with torch.no_grad():
        m.weight.copy_(randn(g, 32, H).cuda())
    base = randn(g, 1, H, Tq, Tk, dtype=dtype)
    layouts = {
        "rows": dev(spread(base, (2, 3))),
        "shifted": dev(torch.cat([base[..., :1], base], -1))[..., 1:],
        "heads": dev(base.transpose(1, 2).contiguous()).transpose(1, 2),
        "columns": dev(base.transpose(2, 3).contiguous()).transpose(2, 3),
        "one row": dev(base[:, :, :1]).expand(1, H, Tq, Tk),
        "one number": torch.ones(1, 1, 1, 1, device="cuda", dtype=dtype).expand(1, H, Tq, Tk),
    }
    for name, dy in layouts.items():
        bias = m(Tq, Tk, dtype=dtype)
        (dw,) = torch.autograd.grad(bias, m.weight, dy)
        _check_grad(dw, dy.cpu(), 32, 128, True, 0)


def test_rel_bias_gradient_against_differences():
    """the bias is linear in the weight: with whole numbers in 32 bits, <dy, bias(W + e) - bias(W)> is the gradient exactly"""
    from rgd_triton_amd import relative_position_bias_fn

    g, nb, H, Tq, Tk = gen(8), 8, 2, 130, 190
    w = torch.randint(-8, 9, (nb, H), generator=g).float().cuda().requires_grad_(True)
    dy = torch.randint(-8, 9, (1, H, Tq, Tk), generator=g).float().cuda()
    f = lambda t: relative_position_bias_fn(t, Tq, Tk, max_distance=40, bidirectional=True, q_offset=9)  # noqa: E731
    (dw,) = torch.autograd.grad(f(w), w, dy)
    for b in range(nb):
        for h in range(H):
            e = torch.zeros_like(w)
            e[b, h] = 1.0
            assert ((f(w.detach() + e) - f(w.detach())) * dy).double().sum().item() == dw[b, h].item()


@pytest.mark.parametrize("Tq,Tk", [(0, 5), (5, 0), (0, 0)])
def test_rel_bias_empty(Tq, Tk):
    from rgd_triton_amd import RelativePositionBias

    m = RelativePositionBias(32, 4, device="cuda")
    bias = m(Tq, Tk)
    assert bias.shape == (1, 4, Tq, Tk)
    (dw,) = torch.autograd.grad(bias, m.weight, torch.empty_like(bias))
    assert torch.equal(dw, torch.zeros_like(dw))


def test_rel_bias_special_values():
    """a bucket of -inf or of the type's lowest value stays what it is; NaN in the gradient reaches its own bucket only"""
    from rgd_triton_amd import relative_position_bias_fn

    w = torch.zeros(8, 2)
    w[3], w[5] = -float("inf"), torch.finfo(torch.float32).min
    bias = relative_position_bias_fn(w.cuda().requires_grad_(True), 40, 40, max_distance=20, bidirectional=True, dtype=torch.float32)
    assert torch.equal(bias.detach().cpu().double(), serving_oracle.relative_bias(w, 40, 40, 20, True))
    wg = w.cuda().requires_grad_(True)
    dy = torch.ones(1, 2, 40, 40)
    dy[0, 0, 10, 10] = float("nan")
    (dw,) = torch.autograd.grad(relative_position_bias_fn(wg, 40, 40, max_distance=20, bidirectional=True), wg, dy.cuda())
    nan = torch.isnan(dw.cpu())
    assert nan[0, 0] and nan.sum() == 1


def test_rel_bias_is_reproducible_and_two_streams_agree():
    from rgd_triton_amd import relative_position_bias_fn

    g = gen(9)
    w = randn(g, 32, 8).cuda().requires_grad_(True)
    dy = randn(g, 1, 8, 700, 900, dtype=torch.bfloat16).cuda()

    def once():
        bias = relative_position_bias_fn(w, 700, 900, dtype=torch.bfloat16)
        return bias.detach(), torch.autograd.grad(bias, w, dy)[0]

    first = once()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for _ in range(10):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(once())
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, first))


@pytest.mark.parametrize("H,Tq,Tk,D", [(4, 200, 200, 64), (3, 130, 275, 128)])
def test_rel_bias_with_flash_attention(H, Tq, Tk, D):
    """The gradient of the weight through FlashAttention is the sum, over the buckets, of the bias gradient FlashAttention gives
    for the same bias as a leaf."""
    from rgd_triton_amd import FlashAttention, RelativePositionBias

    g, dt = gen(10), torch.bfloat16
    q, do = (randn(g, 2, Tq, H, D, dtype=dt).cuda() for _ in range(2))
    k, v = (randn(g, 2, Tk, H, D, dtype=dt).cuda() for _ in range(2))
    m = RelativePositionBias(32, H, device="cuda")
    with torch.no_grad():
        m.weight.copy_(randn(g, 32, H).cuda())
    attn = FlashAttention()
    bias = m(Tq, Tk, q_offset=Tk - Tq, dtype=dt)
    o = attn(q, k, v, bias=bias)
    (dw,) = torch.autograd.grad(o, m.weight, do)
    leaf = bias.detach().requires_grad_(True)
    o2 = attn(q, k, v, bias=leaf)
    assert torch.equal(o, o2)
    (dbias,) = torch.autograd.grad(o2, leaf, do)
    _check_grad(dw, dbias.cpu(), 32, 128, True, Tk - Tq)


def test_rel_bias_forward_in_a_graph_and_backward_refused():
    from rgd_triton_amd import RelativePositionBias

    m = RelativePositionBias(32, 3, device="cuda", dtype=torch.bfloat16)
    with torch.no_grad():
        m.weight.copy_(randn(gen(11), 32, 3).cuda())
        m(50, 70)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = m(50, 70)
        for _ in range(3):
            m.weight.mul_(-1.5)
            eager = m(50, 70)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, eager)


@pytest.mark.parametrize("H,Tq,Tk,off,dtype", [(5, 2601, 2603, 0, torch.bfloat16), (4, 3001, 2808, -700, torch.float16), (3, 2560, 2400, 0, torch.float32),
                                               (2, 2049, 4101, 2052, torch.float32), (1, 3, 11200001, 0, torch.bfloat16), (16, 2200001, 1, 9, torch.bfloat16),
                                               (9, 1040, 4096, 3056, torch.bfloat16)])
def test_rel_bias_large(H, Tq, Tk, off, dtype):
    """matrices beyond 64 MB, which are written in address order: every value, the same bits without scratch (the walk of small
    matrices), nothing written outside of rows with gaps, and the gradient"""
    from rgd_triton_amd import _hip, relative_position_bias_fn
    from rgd_triton_amd.functional import relative_ranges

    nb, md = 32, 128
    g = gen(40)
    w = randn(g, nb, H).cuda().requires_grad_(True)
    bias = relative_position_bias_fn(w, Tq, Tk, max_distance=md, bidirectional=True, q_offset=off, dtype=dtype)
    # row i of a head is the window of its diagonals' values that begins at Tq - 1 - i
    d = torch.arange(-(Tq - 1), Tk, device="cuda") - off
    near = torch.tensor([serving_oracle.bucket_of(x, nb, md, True) for x in range(-md, md + 1)], device="cuda")
    bucket = near[d.clamp(-md, md) + md]
    values = w.detach().t()[:, bucket].to(dtype)
    assert torch.equal(bias.detach()[0], values.unfold(1, Tk, 1).flip(1))
    lib, r = _hip.lib(), relative_ranges(nb, md, True)
    assert lib.rgd_rel_bias_fwd_workspace(H, Tq, Tk, _hip.dtype_code(dtype)) > 0
    walk = torch.empty_like(bias)
    rc = lib.rgd_rel_bias_fwd(H, Tq, Tk, w.data_ptr(), H, nb, 0, r.n, r.c_starts, r.c_buckets, off, _hip.desc4(walk.data_ptr(), 0, Tq * Tk, Tk),
                              _hip.dtype_code(dtype), None, 0, _hip.stream_ptr(w.device))
    assert rc == 0 and torch.equal(walk, bias)
    if Tk < 10**6:
        gaps = torch.full((H, Tq + 1, Tk + 5), 7.0, dtype=dtype, device="cuda")
        n = lib.rgd_rel_bias_fwd_workspace(H, Tq, Tk, _hip.dtype_code(dtype))
        ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        rc = lib.rgd_rel_bias_fwd(H, Tq, Tk, w.data_ptr(), H, nb, 0, r.n, r.c_starts, r.c_buckets, off,
                                  _hip.desc4(gaps.data_ptr() + 2 * gaps.element_size(), 0, gaps.stride(0), gaps.stride(1)), _hip.dtype_code(dtype),
                                  ws.data_ptr(), n, _hip.stream_ptr(w.device))
        assert rc == 0 and torch.equal(gaps[:, :Tq, 2:Tk + 2], bias[0])
        assert (gaps[:, Tq] == 7).all() and (gaps[:, :, :2] == 7).all() and (gaps[:, :, Tk + 2:] == 7).all()
    # whole numbers: every partial sum below 2^24 is exact whatever the order; 3 x 11200001 of them add up to 16.8 million, about
    # 2^24 = 16777216, so only the last addition (of two sums of half of them) can round, to the nearest number of 32 bits
    dy = torch.randint(0, 2, (1, 1, Tq, Tk), device="cuda", dtype=torch.int8).to(dtype)
    (dw,) = torch.autograd.grad(bias, w, dy.expand(1, H, Tq, Tk))
    ref = torch.zeros(nb, dtype=torch.int64, device="cuda")
    for i0 in range(0, Tq, max(1, 10**7 // Tk)):
        i1 = min(Tq, i0 + max(1, 10**7 // Tk))
        rel = torch.arange(Tk, device="cuda")[None] - torch.arange(i0, i1, device="cuda")[:, None] - off
        ref.index_add_(0, near[rel.clamp(-md, md) + md].flatten(), dy[0, 0, i0:i1].flatten().long())
    assert torch.equal(dw, ref.float()[:, None].expand(nb, H)), (dw[:, 0].long() - ref)
