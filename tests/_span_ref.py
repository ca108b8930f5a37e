"""Attention over spans of a cache and eviction in 64 bits, straight from their definitions, and what the kernels may be off by."""

import math

import torch


def attention(q, k, v, pos, *, window=0, sinks=0, prefix=None, scale=None):
    """q (B, H, n, D), caches (B, KV_H, S, D) that hold the tokens' rows, all float64 on the CPU; pos: a list.  Returns the output, the
    probabilities per (b, kv head) summed over rows [B][KV_H] -> (S,), sum_j p |v|, and max over rows of sum_d |q k|."""
    b, h, n, d = q.shape
    kv_h, s = k.shape[1], k.shape[2]
    g = h // kv_h
    scale = scale or 1.0 / math.sqrt(d)
    out, mag = torch.zeros(b, h, n, d, dtype=torch.float64), torch.zeros(b, h, n, d, dtype=torch.float64)
    w = torch.zeros(b, kv_h, s, dtype=torch.float64)
    big = 0.0
    for i in range(b):
        p = pos[i if len(pos) > 1 else 0]
        if p < 0 or p + n > s:
            continue
        for hq in range(h):
            kh = hq // g
            for t in range(n):
                rows = [j for j in range(p + t + 1) if window <= 0 or j > p + t - window or j < sinks]
                kk, vv = k[i, kh, rows], v[i, kh, rows]
                if prefix is not None:
                    kk, vv = torch.cat([prefix[0][kh], kk]), torch.cat([prefix[1][kh], vv])
                x = kk @ q[i, hq, t] * scale
                big = max(big, float((kk.abs() @ q[i, hq, t].abs()).max()) * scale)
                pr = torch.softmax(x, 0)
                out[i, hq, t], mag[i, hq, t] = pr @ vv, pr @ vv.abs()
                if prefix is None:
                    w[i, kh, rows] += pr
    return out, w, mag, big


def attention_wide(q, k, v, pos, *, window=0, sinks=0, prefix=None, weights=None):
    """The output and sum_j p |v| of ``attention`` by masks over whole score matrices, on the tensors' own device (for long calls).
    ``weights`` (B, KV_H, S) grows by the probabilities."""
    b, h, n, d = q.shape
    kv_h, s = k.shape[1], k.shape[2]
    g = h // kv_h
    out, mag = torch.zeros_like(q), torch.zeros_like(q)
    j = torch.arange(s, device=q.device)
    for i in range(b):
        p = pos[i if len(pos) > 1 else 0]
        if p < 0 or p + n > s:
            continue
        row = p + torch.arange(n, device=q.device)[:, None]
        seen = j <= row
        if window > 0:
            seen &= (j > row - window) | (j < sinks)
        any_row = seen.any(0)
        for hq in range(h):
            kk, vv, m = k[i, hq // g][any_row], v[i, hq // g][any_row], seen[:, any_row]
            if prefix is not None:
                kk, vv = torch.cat([prefix[0][hq // g], kk]), torch.cat([prefix[1][hq // g], vv])
                m = torch.cat([torch.ones(n, prefix[0].shape[1], dtype=torch.bool, device=q.device), m], 1)
            x = (q[i, hq] @ kk.T / math.sqrt(d)).masked_fill(~m, -math.inf)
            pr = torch.softmax(x, -1)
            out[i, hq], mag[i, hq] = pr @ vv, pr @ vv.abs()
            if weights is not None:
                weights[i, hq // g, any_row] += pr.sum(0)
    return out, mag


def out_bound(out, mag, dtype):
    """A probability enters P V rounded to fp16 (2^-11 of it); half as much again for the scores' and sums' 32 bits; the output is
    rounded once."""
    return 1.5 * 2.0 ** -11 * mag + torch.finfo(dtype).eps / 2 * out.abs() + 1e-7


def weight_bound(w, big, d):
    """A score is off by at most D roundings of sum |q k| (2^-24 each); a probability by that much twice (its score, the row's sum), the
    exponential's and the sums' last bits on top."""
    return w * (2 * d * 2.0 ** -24 * big + 2.0 ** -19) + 1e-9


def evict(w, length, keep, sinks, recent):
    """The rows that stay, ascending."""
    if length <= keep:
        return list(range(length))
    fixed = list(range(sinks)) + list(range(length - recent, length))
    rest = sorted(range(sinks, length - recent), key=lambda j: (math.isnan(w[j]), -w[j] if not math.isnan(w[j]) else 0.0, j))
    return sorted(fixed + rest[:keep - len(fixed)])
