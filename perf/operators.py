"""What the cache, decode and relative-bias operators are measured on: cases, inputs, their plain forms and their values in 64 bits.

Three operators: appending rotated keys and values to a paged cache (with and without the head LayerNorm), the attention of
one new token over that cache (grouped heads, optionally with a learned relative bias), and that learned bias as a matrix for
training, with the gradient of its weight."""
import math

import torch

own = False

DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # one user's next token: every microsecond of the call is seen
        dict(name="append_one", op="append", dtype="bf16", B=1, T=1, Hq=16, Hkv=16, D=64, R=32, page=16, cap=512,
             ln=False, ragged=False, heads_second=False, table="fp32"),
        # one step of a served batch, grouped heads
        dict(name="append_step", op="append", dtype="bf16", B=256, T=1, Hq=32, Hkv=8, D=128, R=128, page=16, cap=1024,
             ln=False, ragged=False, heads_second=False, table="bf16"),
        # prompts of unequal lengths, padded, head LayerNorm and a partial rotation, heads in front of tokens
        dict(name="append_prompts_ln", op="append", dtype="fp16", B=5, T=1023, Hq=24, Hkv=24, D=64, R=32, page=48, cap=1536,
             ln=True, ragged=True, heads_second=True, table="fp16"),
        # long prompts
        dict(name="append_long", op="append", dtype="bf16", B=8, T=4096, Hq=32, Hkv=8, D=128, R=128, page=64, cap=4352,
             ln=False, ragged=False, heads_second=False, table="fp32"),
        # one user, a short context
        dict(name="decode_one", op="decode", dtype="bf16", B=1, Hq=16, Hkv=16, D=64, page=16, least=200, most=200, cap=512,
             buckets=0, max_distance=0, bidirectional=False),
        # a served batch, every sequence at a place of its own
        dict(name="decode_batch", op="decode", dtype="bf16", B=64, Hq=32, Hkv=8, D=128, page=16, least=300, most=4100, cap=4352,
             buckets=0, max_distance=0, bidirectional=False),
        # one very long context: nothing but the split over its length fills the chip
        dict(name="decode_long", op="decode", dtype="fp16", B=1, Hq=32, Hkv=8, D=128, page=64, least=131000, most=131000,
             cap=131072, buckets=0, max_distance=0, bidirectional=False),
        # a model trained with the learned bias: a head per key head, an odd head dim, pages that end inside a tile, empty rows
        dict(name="decode_bias_odd", op="decode", dtype="fp16", B=19, Hq=24, Hkv=24, D=80, page=5, least=0, most=2000, cap=2005,
             buckets=32, max_distance=128, bidirectional=False),
        # the bias of a short training sequence, causal buckets
        dict(name="bias_short", op="bias", dtype="bf16", weight="bf16", H=8, Tq=128, Tk=128, offset=0, buckets=32,
             max_distance=128, bidirectional=False),
        # an ordinary training step
        dict(name="bias_train", op="bias", dtype="bf16", weight="fp32", H=16, Tq=2048, Tk=2048, offset=0, buckets=32,
             max_distance=128, bidirectional=True),
        # a chunk of queries behind earlier keys, nothing aligned
        dict(name="bias_odd", op="bias", dtype="fp32", weight="fp32", H=7, Tq=1001, Tk=1777, offset=776, buckets=64,
             max_distance=800, bidirectional=True),
        # the longest sequences that this repository times attention with
        dict(name="bias_large", op="bias", dtype="bf16", weight="fp32", H=24, Tq=4352, Tk=4352, offset=0, buckets=32,
             max_distance=128, bidirectional=True),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "bias"])
    if op == "bias":
        both = rng.random() < 0.5
        H, Tq, Tk = rng.randint(1, 24), _log(rng, 1, 4352), _log(rng, 1, 4352)
        buckets = rng.choice([8, 16, 32, 64])
        return dict(op=op, dtype=rng.choice(["bf16", "fp16", "fp32"]) if H * Tq * Tk < 2e8 else "bf16",
                    weight=rng.choice(["bf16", "fp32"]), H=H, Tq=Tq, Tk=Tk, offset=rng.choice([0, 0, _log(rng, 1, 4352)]),
                    buckets=buckets, max_distance=buckets + _log(rng, 1, 1000), bidirectional=both)
    page = rng.choice([1, 5, 8, 16, 16, 32, 48, 64, 128])
    group = rng.choice([1, 1, 2, 4, 8])
    Hkv = rng.randint(1, 16)
    if op == "append":
        D = 2 * rng.randint(8, 64) if rng.random() < 0.4 else rng.choice([32, 64, 128])
        B = _log(rng, 1, 256)
        # a third are single tokens; a prompt is bounded so that a pass moves no more than the largest listed one
        T = 1 if rng.random() < 0.34 else max(1, min(_log(rng, 2, 4096), int(3.0e8 / (B * Hkv * (group + 2) * D))))
        used = _log(rng, 1, 1000)
        return dict(op=op, dtype=rng.choice(["bf16", "fp16"]), B=B, T=T, Hq=Hkv * group, Hkv=Hkv, D=D,
                    R=rng.choice([D, D // 4 * 2]), page=page, cap=T + used, ln=rng.random() < 0.5, ragged=T > 1 and rng.random() < 0.5,
                    heads_second=rng.random() < 0.5, table=rng.choice(["same", "fp32"]))
    D = rng.randint(16, 128) if rng.random() < 0.3 else rng.choice([32, 64, 64, 96, 128, 128])
    B = _log(rng, 1, 256)
    most = max(1, min(_log(rng, 1, 131072), int(1.4e8 / (B * Hkv * D))))
    bias = rng.random() < 0.35
    return dict(op=op, dtype=rng.choice(["bf16", "fp16"]), B=B, Hq=Hkv * group, Hkv=Hkv, D=D, page=page, least=min(most, rng.choice([0 if B > 8 else 1, most // 3 + 1, most])),
                most=most, cap=most + rng.randint(0, most), buckets=32 if bias else 0, max_distance=_log(rng, 33, 600) if bias else 0,
                bidirectional=bias and rng.random() < 0.5)


def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * scale).to(dtype)


def _table(positions, R, dtype):
    """sin and cos (2, positions, R) of every position; the angles are taken in 64 bits."""
    rate = 10000.0 ** (-torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / max(R, 1))
    angle = torch.arange(positions, device=DEV, dtype=torch.float64)[:, None] * rate
    return torch.stack([angle.sin(), angle.cos()]).repeat_interleave(2, dim=-1).to(dtype)


def _paged(g, c, dtype):
    """Two caches with twenty spare pages, and for each sequence its pages, in no order."""
    pages_each = -(-c["cap"] // c["page"])
    total = c["B"] * pages_each + 20
    shape = (total, c["page"], c["Hkv"], c["D"])
    order = torch.randperm(total, generator=g, device=DEV)[: c["B"] * pages_each]
    return _normal(g, shape, dtype), _normal(g, shape, dtype), order.to(torch.int32).reshape(c["B"], pages_each)


def prepare(case, seed):
    c, g = case, _generator(seed)
    dtype = TYPES[c["dtype"]]
    if c["op"] == "bias":
        weight = _normal(g, (c["buckets"], c["H"]), TYPES[c["weight"]]).requires_grad_(True)
        return dict(case=c, weight=weight, grad=_normal(g, (1, c["H"], c["Tq"], c["Tk"]), dtype, 0.1))
    k_cache, v_cache, pages = _paged(g, c, dtype)
    s = dict(case=c, k_cache=k_cache, v_cache=v_cache, pages=pages)
    if c["op"] == "decode":
        s["q"] = _normal(g, (c["B"], 1, c["Hq"], c["D"]), dtype)
        s["lens"] = torch.randint(c["least"], c["most"] + 1, (c["B"],), generator=g, device=DEV, dtype=torch.int32)
        s["weight"] = _normal(g, (c["buckets"], c["Hq"]), torch.float32) if c["buckets"] else None
        return s
    for name, heads in (("q", c["Hq"]), ("k", c["Hkv"]), ("v", c["Hkv"])):
        s[name] = _normal(g, (c["B"], heads, c["T"], c["D"]) if c["heads_second"] else (c["B"], c["T"], heads, c["D"]), dtype)
    s["lens"] = torch.randint(0, c["cap"] - c["T"] + 1, (c["B"],), generator=g, device=DEV, dtype=torch.int32)
    s["new"] = torch.randint(0, c["T"] + 1, (c["B"],), generator=g, device=DEV, dtype=torch.int32) if c["ragged"] else None
    s["table"] = _table(pages.shape[1] * c["page"], c["R"], dtype if c["table"] == "same" else TYPES[c["table"]])
    return s


# ------------------------------------------------------------------------------------------------------------------
# the plain forms, in 32 bits
# ------------------------------------------------------------------------------------------------------------------


def _buckets(relative, buckets, max_distance, bidirectional):
    """The bucket of key position minus query position; distances next to a border need 64 bits."""
    first = torch.zeros_like(relative)
    if bidirectional:
        buckets //= 2
        first = (relative > 0) * buckets
        n = relative.abs()
    else:
        n = (-relative).clamp(min=0)
    exact = buckets // 2
    far = torch.log(n.clamp(min=1).double() / exact) / math.log(max_distance / exact) * (buckets - exact)
    far = (exact + torch.floor(far + 1e-9).long()).clamp(max=buckets - 1)
    return first + torch.where(n < exact, n, far)


def _plain_bias(s):
    c, W = s["case"], s["weight"].detach()
    Tq, Tk, H = c["Tq"], c["Tk"], c["H"]
    i, j = torch.arange(Tq, device=DEV), torch.arange(Tk, device=DEV)
    # one value for each diagonal, then every element from its diagonal
    diagonal = torch.arange(-(Tq - 1), Tk, device=DEV) - c["offset"]
    bucket = _buckets(diagonal, c["buckets"], c["max_distance"], c["bidirectional"])
    values = W.float()[bucket]
    bias = values.t()[:, j[None, :] - i[:, None] + Tq - 1].to(TYPES[c["dtype"]])[None]
    # rows padded by Tq and read with one element less shift by one each: columns become diagonals
    g = torch.nn.functional.pad(s["grad"][0].float().flip(1), (0, Tq)).reshape(H, -1)[:, : Tq * (Tq + Tk - 1)]
    along = g.reshape(H, Tq, Tq + Tk - 1).sum(1)
    chosen = (bucket[None, :] == torch.arange(c["buckets"], device=DEV)[:, None]).float()
    return bias, (chosen @ along.t()).to(W.dtype)


def _plain_rotate(x, sin, cos, R, ln):
    """x (..., D) in 32 bits, sin and cos (..., R)"""
    if ln:
        x = x - x.mean(-1, keepdim=True)
        x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6)
    r = x[..., :R]
    turned = torch.stack([-r[..., 1::2], r[..., 0::2]], dim=-1).reshape(r.shape)
    return torch.cat([r * cos + turned * sin, x[..., R:]], dim=-1)


def _plain_append(s):
    c, dtype = s["case"], TYPES[s["case"]["dtype"]]
    q, k, v = (s[n].transpose(1, 2) if c["heads_second"] else s[n] for n in "qkv")
    t = torch.arange(c["T"], device=DEV)
    at = s["lens"].long()[:, None] + t
    live = torch.ones_like(at, dtype=torch.bool) if s["new"] is None else t < s["new"].long()[:, None]
    sin, cos = (part[at][:, :, None, :] for part in s["table"].float())
    q = torch.where(live[:, :, None, None], _plain_rotate(q.float(), sin, cos, c["R"], c["ln"]), 0.0).to(dtype)
    k = _plain_rotate(k.float(), sin, cos, c["R"], c["ln"]).to(dtype)
    page = s["pages"].long().gather(1, at // c["page"])
    s["k_cache"][page[live], (at % c["page"])[live]] = k[live]
    s["v_cache"][page[live], (at % c["page"])[live]] = v[live]
    return (q.transpose(1, 2) if c["heads_second"] else q), s["k_cache"], s["v_cache"]


def _plain_decode(s):
    c = s["case"]
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    k, v = (s[n][s["pages"].long()].reshape(B, -1, Hkv, D).permute(0, 2, 1, 3).float() for n in ("k_cache", "v_cache"))
    at, last = torch.arange(k.shape[2], device=DEV), s["lens"].long()[:, None] - 1
    q = s["q"].float().reshape(B, Hkv, Hq // Hkv, D)
    logits = (q @ k.transpose(2, 3)).reshape(B, Hq, -1) / math.sqrt(D)
    if s["weight"] is not None:
        bucket = _buckets((at - last).clamp(max=0), c["buckets"], c["max_distance"], c["bidirectional"])
        logits = logits + s["weight"].float()[bucket].transpose(1, 2)
    logits = torch.where((at <= last)[:, None, :], logits, -math.inf)
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = (p.reshape(B, Hkv, Hq // Hkv, -1) @ v).reshape(B, Hq, D) / torch.where(total == 0, 1.0, total)
    return o.to(TYPES[c["dtype"]])[:, None], (top + torch.log(total))[..., 0]


def _own_bias(s):
    from rgd_triton_amd import relative_position_bias_fn

    c = s["case"]
    bias = relative_position_bias_fn(s["weight"], c["Tq"], c["Tk"], max_distance=c["max_distance"], bidirectional=c["bidirectional"],
                                     q_offset=c["offset"], dtype=TYPES[c["dtype"]])
    return bias.detach(), torch.autograd.grad(bias, s["weight"], s["grad"])[0]


def _own_append(s):
    from rgd_triton_amd import rope_cache_append_fn

    c = s["case"]
    q = rope_cache_append_fn(s["q"], s["k"], s["v"], s["table"], s["k_cache"], s["v_cache"], s["pages"], s["lens"], new_lens=s["new"],
                             heads_second=c["heads_second"], norm_eps=1e-6 if c["ln"] else None)
    return q, s["k_cache"], s["v_cache"]


def _own_decode(s):
    from rgd_triton_amd import paged_decode_attn_func

    c = s["case"]
    return paged_decode_attn_func(s["q"], s["k_cache"], s["v_cache"], s["pages"], s["lens"], rel_weight=s["weight"],
                                  max_distance=c["max_distance"], bidirectional=c["bidirectional"], return_lse=True)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"append": _own_append, "decode": _own_decode, "bias": _own_bias}[op](state)
    return {"append": _plain_append, "decode": _plain_decode, "bias": _plain_bias}[op](state)


def work(case):
    c, size = case, 4 if case["dtype"] == "fp32" else 2
    if c["op"] == "bias":
        # the matrix written once forward, its gradient read once and added up backward
        n = c["H"] * c["Tq"] * c["Tk"]
        return {"bytes": 2.0 * n * size, "flops": float(n)}
    if c["op"] == "append":
        n = c["B"] * c["T"] * (0.5 if c["ragged"] else 1.0)  # on the average
        heads = c["Hq"] + c["Hkv"]
        table = 2 * n * c["R"] * (4 if c["table"] == "fp32" else 2)
        # the padded rows of q are written too
        written = (n * 2 * c["Hkv"] + c["B"] * c["T"] * c["Hq"]) * c["D"] * size
        return {"bytes": n * (heads + c["Hkv"]) * c["D"] * size + written + table,
                "flops": n * heads * (3.0 * c["R"] + (8.0 * c["D"] if c["ln"] else 0))}
    keys = c["B"] * (c["least"] + c["most"]) / 2.0
    return {"bytes": 2.0 * keys * c["Hkv"] * c["D"] * size + 2.0 * c["B"] * c["Hq"] * c["D"] * size + 4.0 * keys / c["page"],
            "flops": 4.0 * keys * c["Hq"] * c["D"]}


# ------------------------------------------------------------------------------------------------------------------
# from the definitions, in 64 bits
# ------------------------------------------------------------------------------------------------------------------


def _bucket_of(d, buckets, max_distance, bidirectional):
    """The bucket of one distance d = key - query, with whole numbers: floor(m log(n/e) / log(x/e)) is the largest k with
    (n/e)^m >= (x/e)^k."""
    first, n = 0, max(-d, 0)
    if bidirectional:
        buckets //= 2
        first, n = (buckets if d > 0 else 0), abs(d)
    e = buckets // 2
    if n < e:
        return first + n
    m, k = buckets - e, 0
    while k < m - 1 and n**m >= max_distance ** (k + 1) * e ** (m - k - 1):
        k += 1
    return first + e + k


def _exact_bias(s):
    c, W, dy = s["case"], s["weight"].detach().double(), s["grad"][0]
    bias = torch.empty((c["H"], c["Tq"], c["Tk"]), dtype=torch.float64, device=DEV)
    dW = torch.zeros_like(W)
    far = c["max_distance"] + 1  # every distance from here on has the last bucket
    known = {d: _bucket_of(d, c["buckets"], c["max_distance"], c["bidirectional"]) for d in range(-far, far + 1)}
    for d in range(-(c["Tq"] - 1), c["Tk"]):
        b = known[max(-far, min(far, d - c["offset"]))]
        bias.diagonal(d, 1, 2).copy_(W[b][:, None].expand_as(bias.diagonal(d, 1, 2)))
        dW[b] += dy.diagonal(d, 1, 2).double().sum(-1)
    return bias[None], dW


def _exact_append(s):
    c = s["case"]
    R = c["R"]
    q, k, v = (s[n].double().transpose(1, 2) if c["heads_second"] else s[n].double() for n in "qkv")
    if c["ln"]:
        q, k = ((x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + 1e-6) for x in (q, k))
    out, k_cache, v_cache = torch.zeros_like(q), s["k_cache"].double(), s["v_cache"].double()
    lens = s["lens"].tolist()
    new = [c["T"]] * c["B"] if s["new"] is None else s["new"].tolist()
    table = s["table"].double()
    turn = torch.complex(table[1, :, 0::2], table[0, :, 0::2])
    for b in range(c["B"]):
        n, at = new[b], torch.arange(lens[b], lens[b] + new[b], device=DEV)
        rows = []
        for x in (q[b, :n], k[b, :n]):
            z = torch.view_as_complex(x[..., :R].reshape(n, x.shape[1], R // 2, 2).contiguous()) * turn[at][:, None, :]
            rows.append(torch.cat([torch.view_as_real(z).reshape(n, x.shape[1], R), x[..., R:]], dim=-1))
        out[b, :n] = rows[0]
        page = s["pages"][b].long()[at // c["page"]]
        k_cache[page, at % c["page"]] = rows[1]
        v_cache[page, at % c["page"]] = v[b, :n]
    return (out.transpose(1, 2) if c["heads_second"] else out), k_cache, v_cache


def _exact_decode(s):
    c = s["case"]
    group = c["Hq"] // c["Hkv"]
    o = torch.zeros((c["B"], 1, c["Hq"], c["D"]), dtype=torch.float64, device=DEV)
    lse = torch.full((c["B"], c["Hq"]), -math.inf, dtype=torch.float64, device=DEV)
    if c["buckets"]:
        far = c["max_distance"] + 1
        known = [_bucket_of(-n, c["buckets"], c["max_distance"], c["bidirectional"]) for n in range(far + 1)]
        known = torch.tensor(known, device=DEV)
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        at = torch.arange(n, device=DEV)
        page = s["pages"][b].long()[at // c["page"]]
        k, v = s["k_cache"][page, at % c["page"]], s["v_cache"][page, at % c["page"]]
        for h in range(c["Hkv"]):
            heads = slice(h * group, (h + 1) * group)
            x = s["q"][b, 0, heads].double() @ k[:, h].double().t() * c["D"] ** -0.5
            if c["buckets"]:
                x = x + s["weight"].double()[known[(n - 1 - at).clamp(max=far)], heads].t()
            lse[b, heads] = torch.logsumexp(x, -1)
            o[b, 0, heads] = torch.softmax(x, -1) @ v[:, h].double()
    return o, lse


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "bias": _exact_bias}[case["op"]](s)
