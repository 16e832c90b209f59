"""The operators as they are used together: a prompt is appended to the cache, then every new token is appended and attends over
it, eagerly and from a replayed graph; and the same sequence through RoPE and FlashAttention as a whole."""
import math

import pytest
import torch

from serving_helpers import check_decode, gen, half_step, randn, rotary, serving_oracle

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


class Layer:
    """One attention layer's operators and a cache of `cap` positions for each of B sequences"""

    def __init__(self, B, H, D, size, cap, dtype, ln, buckets, seed):
        import rgd_triton_amd as rgd

        g = gen(seed)
        self.append = rgd.FusedLNRoPECacheAppend() if ln else rgd.RoPECacheAppend()
        self.decode, self.attn = rgd.PagedDecodeAttention(), rgd.FlashAttention()
        self.rotate = rgd.FusedLNRoPE() if ln else rgd.RoPE()
        each = -(-cap // size)
        self.pages = torch.randperm(B * each + 2, generator=g)[: B * each].to(torch.int32).reshape(B, each).cuda()
        self.k, self.v = (torch.full((B * each + 2, size, H, D), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
        self.table = rotary(each * size + 1, D // 2).cuda()
        self.rel = None
        if buckets:
            self.rel = rgd.RelativePositionBias(buckets, H, max_distance=40, bidirectional=False, device="cuda")
            with torch.no_grad():
                self.rel.weight.copy_(randn(g, buckets, H))

    def step(self, q, k, v, lens):
        """one new token of every sequence (B, H, 1, D); `lens` counts the tokens before it and is advanced on the GPU"""
        q = self.append(q, k, v, self.table, self.k, self.v, self.pages, lens)
        lens.add_(1)
        return self.decode(q.transpose(1, 2), self.k, self.v, self.pages, lens, rel_bias=self.rel)


@pytest.mark.parametrize("ln,buckets,dtype,D", [(False, 0, BF, 64), (True, 16, HF, 64), (False, 16, BF, 128), (True, 0, BF, 96)])
def test_prompt_then_tokens_is_the_whole_sequence(ln, buckets, dtype, D):
    from rgd_triton_amd import paged_decode_attn_func

    B, H, T, P = 2, 3, 75, 60  # 60 tokens of prompt, 15 one at a time
    layer = Layer(B, H, D, 16, 80, dtype, ln, buckets, 500)
    g = gen(501)
    q, k, v = (randn(g, B, H, T, D, dtype=dtype).cuda() for _ in range(3))
    with torch.no_grad():
        qr, kr = layer.rotate(q, k, layer.table)
        lens = torch.zeros(B, dtype=torch.int32, device="cuda")
        qp = layer.append(q[:, :, :P], k[:, :, :P], v[:, :, :P], layer.table, layer.k, layer.v, layer.pages, lens)
        # the same mathematics by two kernels: each within half a step of the exact row
        near = lambda a, b: (a.double() - b.double()).abs().max() <= 2 * half_step(dtype) * b.double().abs().max()  # noqa: E731
        assert near(qp, qr[:, :, :P])
        lens += P
        outs = [layer.step(q[:, :, t:t + 1], k[:, :, t:t + 1], v[:, :, t:t + 1], lens) for t in range(P, T)]
        bias = None if layer.rel is None else layer.rel(T, T, dtype=dtype)
        whole = layer.attn(*(x.transpose(1, 2) for x in (qr, kr, v)), bias=bias, causal=True)
    assert lens.tolist() == [T] * B
    kc, vc = layer.k.cpu(), layer.v.cpu()
    for b in range(B):
        at = [(int(layer.pages[b, j // 16]), j % 16) for j in range(T)]
        cached = torch.stack([kc[p, s] for p, s in at])
        assert near(cached, kr[b].transpose(0, 1).cpu())
        assert torch.equal(torch.stack([vc[p, s] for p, s in at]), v[b].transpose(0, 1).cpu())
    # against 64 bits on the cache as it stands, and against the whole sequence's rows
    w = None if layer.rel is None else layer.rel.weight.detach().cpu()
    for i, o in enumerate(outs):
        t = P + i
        row = whole[:, t:t + 1].double().cpu()
        # FlashAttention rounds its bias and its probabilities to 16 bits: logits off by half a step of the bias, outputs by one
        # of the probabilities and one of the values
        drift = (half_step(dtype) * (w.abs().max().item() if w is not None else 0.0) + 16 * half_step(dtype)) * v.double().abs().max().item()
        assert (o.double().cpu() - row).abs().max() <= drift
    qlast = qr[:, :, T - 1:T].transpose(1, 2)
    o, lse = paged_decode_attn_func(
        qlast, layer.k, layer.v, layer.pages, lens, rel_weight=None if w is None else layer.rel.weight.detach(), max_distance=40,
        bidirectional=False, return_lse=True)
    ref = serving_oracle.decode(qlast.cpu(), kc, vc, layer.pages.cpu(), lens.cpu(), D**-0.5, w, 40, False)
    check_decode(o, lse, ref, T, D)


@pytest.mark.parametrize("buckets", [0, 16])
def test_decode_step_replays_from_a_graph(buckets):
    """append and attention captured once, replayed for token after token with the lengths advancing on the GPU, two captured
    graphs of the same layer sizes in turn; every replay is compared bit for bit with an eager layer"""
    B, H, D = 5, 4, 64
    eager = Layer(B, H, D, 16, 200, BF, True, buckets, 510)
    layers = [Layer(B, H, D, 16, 200, BF, True, buckets, 510) for _ in range(2)]
    g = gen(511)
    ins = [randn(g, B, H, 1, D, dtype=BF).cuda() for _ in range(3)]
    start = torch.tensor([0, 15, 16, 100, 126], dtype=torch.int32)
    with torch.no_grad():
        prompt = [randn(g, B, H, 130, D, dtype=BF).cuda() for _ in range(3)]
        for l in [eager] + layers:
            l.append(*prompt, l.table, l.k, l.v, l.pages, torch.zeros(B, dtype=torch.int32, device="cuda"), new_lens=start.cuda())
            l.lens = start.cuda()
        warm = start.cuda()
        eager.step(*ins, warm)  # a first call outside of the captures (its token is written again below)
        torch.cuda.synchronize()
        graphs, outs = [], []
        for l in layers:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(l.step(*ins, l.lens))
            graphs.append(graph)
        for l in layers:
            l.lens.copy_(start)
        for rep in range(6):
            for x in ins:
                x.mul_(-0.9).add_(0.01 * rep)
            want = eager.step(*ins, eager.lens)
            torch.cuda.synchronize()
            for graph in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for l, out in zip(layers, outs):
                assert torch.equal(out, want), f"replay {rep}"
                assert torch.equal(l.lens, eager.lens)
                assert torch.equal(l.k.view(torch.int16), eager.k.view(torch.int16))


def test_training_step_gradient_against_differences():
    """bias, attention and both gradients in one step: the weight's gradient equals differences of the loss in the weight as
    32-bit attention has it on the CPU"""
    import rgd_triton_amd as rgd

    B, T, H, D, nb = 1, 48, 2, 32, 8
    g = gen(520)
    q, k, v, do = (randn(g, B, T, H, D, dtype=HF) for _ in range(4))
    m = rgd.RelativePositionBias(nb, H, max_distance=20, bidirectional=True, device="cuda")
    with torch.no_grad():
        m.weight.copy_(randn(g, nb, H))
    o = rgd.FlashAttention()(q.cuda(), k.cuda(), v.cuda(), bias=m(T, T))
    o.backward(do.cuda())

    qd, kd, vd, dod = (t.double().permute(0, 2, 1, 3)[0] for t in (q, k, v, do))  # (H, T, D)

    def forward(w):
        p = torch.softmax(qd @ kd.transpose(1, 2) * D**-0.5 + serving_oracle.relative_bias(w, T, T, 20, True)[0], -1)
        return p, p @ vd

    w = m.weight.detach().cpu().double()
    # dS = P (dP - delta): P, o and the products' operands are 16-bit, each off by at most half a step, so a pair is off by a few
    # half steps of P (sum |do v| + sum |do o|); a bucket by the sum over its pairs
    p, out = forward(w)
    pair = p * (dod.abs() @ vd.abs().transpose(1, 2) + (dod * out).abs().sum(-1, keepdim=True))
    allowed = serving_oracle.relative_bias_grad(4 * half_step(HF) * pair[None], nb, 20, True)[0] + 1e-5
    for b in range(nb):
        for h in range(H):
            e = torch.zeros_like(w)
            e[b, h] = 1e-4
            slope = ((forward(w + e)[1] - forward(w - e)[1]) * dod).sum().item() / 2e-4
            assert abs(m.weight.grad[b, h].item() - slope) <= allowed[b, h], (b, h, m.weight.grad[b, h].item(), slope)


def test_append_results_feed_decode_across_streams():
    """append on one stream, decode on another that waits for it"""
    layer = Layer(3, 4, 64, 16, 100, BF, False, 0, 530)
    g = gen(531)
    q, k, v = (randn(g, 3, 4, 90, 64, dtype=BF).cuda() for _ in range(3))
    qn = randn(g, 3, 1, 4, 64, dtype=BF).cuda()
    lens = torch.tensor([90, 50, 1], dtype=torch.int32, device="cuda")
    s = torch.cuda.Stream()
    with torch.no_grad():
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            layer.append(q, k, v, layer.table, layer.k, layer.v, layer.pages, torch.zeros_like(lens), new_lens=lens)
        torch.cuda.current_stream().wait_stream(s)
        o = layer.decode(qn, layer.k, layer.v, layer.pages, lens)
    ref = serving_oracle.decode(qn.cpu(), layer.k.cpu(), layer.v.cpu(), layer.pages.cpu(), lens.cpu(), 64**-0.5)
    check_decode(o, None, ref, 90, 64)


def test_calls_in_inference_mode_and_from_threads():
    """caches made in inference mode (they have no version counter), weights that require a gradient under no_grad, and two host
    threads at once on streams of their own"""
    import threading

    import rgd_triton_amd as rgd

    def work(seed, out):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream), torch.inference_mode():
            layer = Layer(3, 4, 64, 16, 100, BF, True, 16, seed)
            g = gen(seed + 1)
            q, k, v = (randn(g, 3, 4, 60, 64, dtype=BF).cuda() for _ in range(3))
            lens = torch.zeros(3, dtype=torch.int32, device="cuda")
            got = [layer.append(q, k, v, layer.table, layer.k, layer.v, layer.pages, lens)]
            lens += 60
            for t in range(8):
                got.append(layer.step(q[:, :, t:t + 1], k[:, :, t:t + 1], v[:, :, t:t + 1], lens))
            got.append(layer.rel(40, 50, dtype=BF))
        stream.synchronize()
        out.append(got)

    alone, together = [], []
    for seed in (540, 550):
        work(seed, alone)
    errors = []

    def guarded(seed, out):
        try:
            for _ in range(4):
                work(seed, out)
        except Exception as e:  # surfaced below
            errors.append(repr(e))

    lists = [[], []]
    threads = [threading.Thread(target=guarded, args=(s, o)) for s, o in zip((540, 550), lists)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for want, outs in zip(alone, lists):
        assert len(outs) == 4
        for got in outs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    w = torch.zeros(32, 4, device="cuda", requires_grad=True)
    kc = torch.zeros(4, 16, 4, 64, device="cuda", dtype=BF)
    args = (torch.zeros(1, 1, 4, 64, device="cuda", dtype=BF), kc, kc, torch.zeros(1, 4, device="cuda", dtype=torch.int32),
            torch.ones(1, device="cuda", dtype=torch.int32))
    with pytest.raises(AssertionError, match="no_grad"):
        rgd.paged_decode_attn_func(*args, rel_weight=w)
    with torch.no_grad():
        assert (rgd.paged_decode_attn_func(*args, rel_weight=w) == 0).all()


def test_bias_gradient_is_not_differentiated_twice():
    from rgd_triton_amd import relative_position_bias_fn

    w = torch.zeros(32, 2, device="cuda", requires_grad=True)
    dy = torch.ones(1, 2, 30, 30, device="cuda", requires_grad=True)
    (dw,) = torch.autograd.grad(relative_position_bias_fn(w, 30, 30), w, dy, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(dw.sum(), dy)


@pytest.mark.parametrize("Hq,Hkv,D,size,B,most", [(8, 1, 64, 16, 300, 90), (2, 2, 128, 8, 700, 40), (32, 2, 32, 1, 65, 70), (5, 5, 96, 48, 130, 33)])
def test_many_short_sequences(Hq, Hkv, D, size, B, most):
    """more sequences than one look at the lengths takes in (64), several units for each wavefront, empty ones among them; checked
    against torch in 64 bits on the GPU"""
    from rgd_triton_amd import paged_decode_attn_func

    g = gen(560)
    each = -(-most // size)
    total = B * each + 1
    pages = torch.randperm(total, generator=g)[: B * each].to(torch.int32).reshape(B, each)
    lens = torch.randint(0, most + 1, (B,), generator=g, dtype=torch.int32)
    lens[::7] = 0
    q = randn(g, B, 1, Hq, D, dtype=BF).cuda()
    k, v = (randn(g, total, size, Hkv, D, dtype=BF).cuda() for _ in range(2))
    pages, lens = pages.cuda(), lens.cuda()
    o, lse = paged_decode_attn_func(q, k, v, pages, lens, return_lse=True)
    kk, vv = (c[pages.long()].reshape(B, each * size, Hkv, D).double().repeat_interleave(Hq // Hkv, 2).permute(0, 2, 1, 3).contiguous() for c in (k, v))
    q64 = q.double().permute(0, 2, 1, 3)
    s = (kk * q64).sum(-1) * D**-0.5
    reach = (kk * q64).abs().sum(-1).amax(-1) * D**-0.5
    seen = torch.arange(each * size, device="cuda") < lens[:, None]
    s = s.masked_fill(~seen[:, None], float("-inf"))
    p = torch.softmax(s, -1).nan_to_num(0.0)
    ref = ((p[..., None] * vv).sum(2)[:, None], torch.logsumexp(s, -1), (p[..., None] * vv.abs()).sum(2)[:, None], reach)
    check_decode(o, lse, tuple(t.cpu() for t in ref), most, D)


def test_decode_softmax_scale_of_zero_is_the_mean():
    """scale 0 is a scale, not the default: every key weighs the same"""
    from rgd_triton_amd import paged_decode_attn_func

    g = gen(570)
    q, k, v = randn(g, 1, 1, 4, 64, dtype=BF).cuda(), randn(g, 5, 16, 2, 64, dtype=BF).cuda(), randn(g, 5, 16, 2, 64, dtype=BF).cuda()
    pages = torch.tensor([[3, 0, 4, 1]], dtype=torch.int32, device="cuda")
    o, lse = paged_decode_attn_func(q, k, v, pages, torch.tensor([55], dtype=torch.int32, device="cuda"), softmax_scale=0.0, return_lse=True)
    vv = v[pages[0].long()].reshape(64, 2, 64)[:55].double()
    ref, mag = (t.mean(0).repeat_interleave(2, 0) for t in (vv, vv.abs()))
    # one rounding to bf16 (2^-8), the probabilities' parts 2^-14, fp32 sums
    assert ((o[0, 0].double() - ref).abs() <= 2**-8 * ref.abs() + 2**-13 * mag).all()
    assert (lse.double() - math.log(55)).abs().max() <= 2**-20


def test_padded_prompt_rotated_beforehand_then_a_token():
    """a prompt through RoPE and FlashAttention, stored as it is rotated (no table), then a token: the cache holds RoPE's keys bit
    for bit, padding and foreign slots stay as they were, and the token sees its sequence"""
    import rgd_triton_amd as rgd

    B, H, T, D, size = 3, 4, 37, 64, 8
    layer = Layer(B, H, D, size, 48, BF, False, 0, 580)
    g = gen(581)
    q, k, v = (randn(g, B, H, T, D, dtype=BF).cuda() for _ in range(3))
    q1, k1, v1 = (randn(g, B, H, 1, D, dtype=BF).cuda() for _ in range(3))
    plens = torch.tensor([37, 0, 16], dtype=torch.int32, device="cuda")
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    with torch.no_grad():
        q, k = rgd.RoPE()(q, k, layer.table)
        out = layer.append(q, k, v, None, layer.k, layer.v, layer.pages, lens, new_lens=plens)
        lens += plens
        kc = layer.k.clone()
        o = layer.step(q1, k1, v1, lens)
    written = torch.zeros(kc.shape[:2], dtype=torch.bool, device="cuda")
    for b in range(B):
        n = int(plens[b])
        assert torch.equal(out[b, :, :n], q[b, :, :n]) and (out[b, :, n:] == 0).all()
        for j in range(n):
            page, slot = int(layer.pages[b, j // size]), j % size
            written[page, slot] = True
            assert torch.equal(kc[page, slot], k[b, :, j])
    assert kc[~written].isnan().all()
    assert lens.tolist() == [38, 1, 17]
    assert torch.equal(o[1, 0], v1[1, :, 0])  # its own key is all it sees
    ref = serving_oracle.decode(rgd.RoPE()(q1, k1, layer.table[:, 37:39].contiguous())[0][:1].transpose(1, 2).cpu(), layer.k.cpu(), layer.v.cpu(),
                                layer.pages[:1].cpu(), lens[:1].cpu(), D**-0.5, None, 0, False)[0]
    # the query's rotation is rounded by two kernels (half a step each way) in front of the logits
    assert (o[:1].double().cpu() - ref).abs().max() <= 16 * half_step(BF) * v.double().abs().max().item()
