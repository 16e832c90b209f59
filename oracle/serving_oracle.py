"""The cache, decode and relative-bias operators from their definitions, in 64 bits on the CPU: one loop per sequence, token and
head, nothing shared with the package.  Test infrastructure only.

Pinned by tests/test_serving_cpu.py: buckets against the logarithm of their definition away from its borders, rotation against
complex multiplication, attention against torch.softmax, the bias gradient against differences.
"""
import functools
import math

import torch


@functools.lru_cache(maxsize=None)
def bucket_of(distance, num_buckets, max_distance, bidirectional):
    """Bucket of distance = key position - query position: the largest k with (n/e)^m >= (max_distance/e)^k, in integers."""
    first, n = 0, max(-distance, 0)
    if bidirectional:
        num_buckets //= 2
        first, n = (num_buckets if distance > 0 else 0), abs(distance)
    e = num_buckets // 2
    if n < e:
        return first + n
    m, k = num_buckets - e, 0
    while k < m - 1 and n**m >= max_distance ** (k + 1) * e ** (m - k - 1):
        k += 1
    return first + e + k


def relative_bias(weight, Tq, Tk, max_distance, bidirectional, q_offset=0):
    """(1, H, Tq, Tk) in 64 bits"""
    nb, H = weight.shape
    out = torch.empty(1, H, Tq, Tk, dtype=torch.float64)
    for i in range(Tq):
        rows = [bucket_of(j - i - q_offset, nb, max_distance, bidirectional) for j in range(Tk)]
        out[0, :, i] = weight.double()[rows].t()
    return out


def relative_bias_grad(dbias, num_buckets, max_distance, bidirectional, q_offset=0):
    """(gradient of the weight, sum of the magnitudes that went into it), both (num_buckets, H) in 64 bits"""
    _, H, Tq, Tk = dbias.shape
    grad, mag = (torch.zeros(num_buckets, H, dtype=torch.float64) for _ in range(2))
    for d in range(-(Tq - 1), Tk):
        b = bucket_of(d - q_offset, num_buckets, max_distance, bidirectional)
        line = dbias[0].double().diagonal(d, 1, 2)
        grad[b] += line.sum(-1)
        mag[b] += line.abs().sum(-1)
    return grad, mag


def rotate_row(x, sin, cos):
    """x (D), sin and cos (R): the first R channels in pairs, the table taken at the output channel"""
    y = x.clone()
    for c in range(0, sin.numel(), 2):
        y[c] = x[c] * cos[c] - x[c + 1] * sin[c]
        y[c + 1] = x[c + 1] * cos[c + 1] + x[c] * sin[c + 1]
    return y


def append(q, k, v, pos_emb, k_cache, v_cache, page_table, cache_lens, new_lens=None, cutoff=None, norm_eps=None):
    """q (B, Hq, T, D), k and v (B, Hkv, T, D), caches (pages, page_size, Hkv, D).  Returns (q out, k_cache, v_cache, written)
    in 64 bits, `written` (pages, page_size) true where a token was stored."""
    B, _, T, _ = q.shape
    pages, size = k_cache.shape[:2]
    qo, kc, vc = torch.zeros_like(q, dtype=torch.float64), k_cache.double(), v_cache.double()
    written = torch.zeros(pages, size, dtype=torch.bool)
    pe = None if pos_emb is None else pos_emb.double()
    cuts = cutoff if isinstance(cutoff, tuple) else (cutoff, cutoff)

    def row(x, pos, cut):
        x = x.double()
        if norm_eps is not None:
            x = x - x.mean()
            x = x / math.sqrt((x * x).mean().item() + norm_eps)
        if pe is not None and (cut is None or pos < cut):
            x = rotate_row(x, pe[0, pos], pe[1, pos])
        return x

    for b in range(B):
        for t in range(T):
            pos = int(cache_lens[b]) + t
            if (new_lens is not None and t >= int(new_lens[b])) or pos < 0 or pos >= page_table.shape[1] * size:
                continue
            for h in range(q.shape[1]):
                qo[b, h, t] = row(q[b, h, t], pos, cuts[0])
            page = int(page_table[b, pos // size])
            if 0 <= page < pages:
                for h in range(k.shape[1]):
                    kc[page, pos % size, h] = row(k[b, h, t], pos, cuts[1])
                    vc[page, pos % size, h] = v[b, h, t].double()
                written[page, pos % size] = True
    return qo, kc, vc, written


def decode(q, k_cache, v_cache, page_table, seq_lens, scale, rel_weight=None, max_distance=128, bidirectional=True):
    """q (B, 1, Hq, D).  Returns (o, lse, weighted, reach) in 64 bits: weighted = sum_j p_j |v_j| and
    reach = max_j scale sum_d |q_d k_jd|, which bound the rounding errors of a computation in 32 bits."""
    B, _, Hq, D = q.shape
    pages, size, Hkv, _ = k_cache.shape
    o, weighted = torch.zeros(B, 1, Hq, D, dtype=torch.float64), torch.zeros(B, 1, Hq, D, dtype=torch.float64)
    lse = torch.full((B, Hq), -math.inf, dtype=torch.float64)
    reach = torch.zeros(B, Hq, dtype=torch.float64)
    for b in range(B):
        n = min(max(int(seq_lens[b]), 0), page_table.shape[1] * size)
        at = [j for j in range(n) if 0 <= int(page_table[b, j // size]) < pages]
        if not at:
            continue
        page, slot = page_table[b, [j // size for j in at]].long(), torch.tensor([j % size for j in at])
        for h in range(Hq):
            kk, vv = (c[page, slot, h // (Hq // Hkv)].double() for c in (k_cache, v_cache))
            s = scale * (kk @ q[b, 0, h].double())
            reach[b, h] = abs(scale) * (kk.abs() @ q[b, 0, h].double().abs()).max()
            if rel_weight is not None:
                nb = rel_weight.shape[0]
                s = s + rel_weight.double()[[bucket_of(j - (n - 1), nb, max_distance, bidirectional) for j in at], h]
            top = s.max()
            if top == -math.inf:
                continue
            p = torch.exp(s - top)
            lse[b, h] = top + torch.log(p.sum())
            p = p / p.sum()
            o[b, 0, h] = p @ vv
            weighted[b, 0, h] = p @ vv.abs()
    return o, lse, weighted, reach
