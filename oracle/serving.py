"""64-bit CPU restatements of the operators around the decode -- TEST INFRASTRUCTURE ONLY.

rope_ref       rotary positions on one or several axes (one token at a time)
weights_ref    attention weight received by each cached token, and a bound on what fp32
               scores and exponents may be off
evict_ref      eviction by weight: indices, moved pools, moved weights
Token t of sequence b lives in slot t % P of page block_table[b, t // P] throughout.
"""
import math

import torch


def rope_ref(x, cos, sin, rows, interleaved=False):
    """x [T, H, 128]; rows [T, R/2]: the table row that turns each pair.  fp64 [T, H, 128]."""
    x = x.cpu().double().clone()
    R = 2 * cos.shape[1]
    cos, sin = cos.cpu().double(), sin.cpu().double()
    for t in range(x.shape[0]):
        for i in range(R // 2):
            j, k = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
            c, s = cos[rows[t, i], i], sin[rows[t, i], i]
            a, b = x[t, :, j].clone(), x[t, :, k].clone()
            x[t, :, j] = a * c - b * s
            x[t, :, k] = b * c + a * s
    return x


def weights_ref(q, k_cache, block_table, seq_lens, lse, weights, scale, causal=False, k_scale=None):
    """Returns (weights after the call, bound), both fp64 [num_pages, Hkv, P].

    bound: fp32 scores of 128 exact products (each sum within 128 * 2^-23 of the products'
    magnitudes, whatever the order and even if truncated), the log-sum-exp in log2 units
    (2^-23 relative), an exponential within 2^-21, fp32 sums over the rows and the pool."""
    q, lse, bt, lens = q.cpu().double(), lse.cpu().double(), block_table.cpu().long(), seq_lens.cpu()
    if q.dim() == 3:
        q = q.unsqueeze(1)
    B, Sq, Hq, _ = q.shape
    Hkv, P = k_cache.shape[2], k_cache.shape[1]
    g = Hq // Hkv
    k = k_cache.cpu().float().double()
    if k_scale is not None:
        k = k * k_scale.cpu().double().view(1, 1, Hkv, 1)
    w = weights.cpu().double().clone()
    bound = torch.zeros_like(w)
    for b in range(B):
        for t in range(int(lens[b])):
            pg, sl = int(bt[b, t // P]), t % P
            for h in range(Hkv):
                for i in range(Sq):
                    if causal and t > int(lens[b]) - Sq + i:
                        continue
                    for a in range(h * g, (h + 1) * g):
                        le = float(lse[b, a, i])
                        if le == -math.inf:
                            continue
                        prod = q[b, i, a] * k[pg, sl, h]
                        p = math.exp(float(prod.sum()) * scale - le)
                        off = float(prod.abs().sum()) * scale * 128 * 2.0 ** -23 + abs(le) * 2.0 ** -22 + 2.0 ** -21
                        w[pg, h, sl] += p
                        bound[pg, h, sl] += p * (off + g * Sq * 2.0 ** -24)
                bound[pg, h, sl] += w[pg, h, sl].abs() * 2.0 ** -23
    return w, bound


def evict_ref(k_cache, v_cache, weights, block_table, seq_lens, keep, sinks, recent, weights_out=None):
    """Returns (kept, new_lens, k, v, weights after the call in weights_out's place)."""
    k, v, w = k_cache.cpu().clone(), v_cache.cpu().clone(), weights.cpu()
    raw = [x.view(torch.uint8) for x in (k, v)]
    old = [x.clone() for x in raw]
    out = (weights if weights_out is None else weights_out).cpu().clone()
    bt = block_table.cpu().long()
    B, (_, Hkv, P) = bt.shape[0], w.shape
    kept = torch.full((B, Hkv, keep), -1, dtype=torch.int32)
    new = torch.zeros(B, dtype=torch.int32)
    for b in range(B):
        L = int(seq_lens[b])
        new[b] = min(L, keep)
        for h in range(Hkv):
            row = [float(w[bt[b, t // P], h, t % P]) for t in range(L)]
            stay = list(range(L))
            if L > keep:
                mid = list(range(sinks, L - recent))
                top = {t: math.inf if math.isnan(row[t]) else row[t] for t in mid}
                # NaN before +inf before the rest; equal weights by index
                mid.sort(key=lambda t: (not math.isnan(row[t]), -top[t], t))
                stay = list(range(sinks)) + sorted(mid[:keep - sinks - recent]) + list(range(L - recent, L))
            for j, t in enumerate(stay):
                kept[b, h, j] = t
                for dst, src in zip(raw, old):
                    dst[bt[b, j // P], j % P, h] = src[bt[b, t // P], t % P, h]
                out[bt[b, j // P], h, j % P] = w[bt[b, t // P], h, t % P]
    return kept, new, k, v, out
