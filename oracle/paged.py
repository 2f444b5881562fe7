"""A KV cache of pages, restated slot by slot in 64 bits (CPU, torch).
TEST INFRASTRUCTURE ONLY.

  gather      the keys or values a table row maps slots [lo, hi) to
  attention   softmax attention of one token per request over its visible
              slots, scores optionally capped by a tanh, with what an error
              bound needs: the weights' sum of |v| and the largest score terms
  rotate      rotation of element pairs by angles given as cos and sin
  append      rows into the pages one at a time, in row order
"""
import math

import torch


def gather(pool, table_row, lo, hi):
    """[hi - lo, Hkv, D] of pool [n_pages, Hkv, page_size, D], one slot at a time."""
    ps = pool.shape[2]
    rows = [pool[int(table_row[t // ps]), :, t % ps] for t in range(lo, hi)]
    return torch.stack(rows) if rows else pool.new_zeros((0, pool.shape[1], pool.shape[3]))


def attention(q, k_pages, v_pages, table, lens, sm_scale=None, softcap=0.0, window=0):
    """(out [B, Hq, D], lse [B, Hq], spread [B, Hq, D], terms [B, Hq]) in 64 bits:
    spread = sum of weight * |v|, terms = the largest sum of |q_d k_d| * scale."""
    B, Hq, D = q.shape
    G = Hq // k_pages.shape[1]
    scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    out = torch.zeros((B, Hq, D), dtype=torch.float64)
    lse = torch.full((B, Hq), float("-inf"), dtype=torch.float64)
    spread, terms = torch.zeros_like(out), torch.zeros((B, Hq), dtype=torch.float64)
    for b, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        if n <= lo:
            continue
        k, v = (gather(x, table[b], lo, n).double() for x in (k_pages, v_pages))
        for h in range(Hq):
            qh, kh, vh = q[b, h].double(), k[:, h // G], v[:, h // G]
            s = (kh * qh).sum(-1) * scale
            terms[b, h] = ((kh * qh).abs().sum(-1) * scale).max()
            if softcap:
                s = softcap * torch.tanh(s / softcap)
            l = torch.logsumexp(s, 0)
            p = torch.exp(s - l)
            out[b, h], spread[b, h], lse[b, h] = (p[:, None] * vh).sum(0), (p[:, None] * vh.abs()).sum(0), l
    return out, lse, spread, terms


def rotate(x, cos, sin, interleaved):
    """x [T, H, D], cos / sin [T, rot / 2] -> (turned, sum of the two products' sizes), 64 bits."""
    y, size = x.double().clone(), x.double().abs()
    half = cos.shape[1]
    for i in range(half):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        xa, xb = x[..., a].double(), x[..., b].double()
        c, s = cos[:, i, None].double(), sin[:, i, None].double()
        y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
        size[..., a], size[..., b] = (xa * c).abs() + (xb * s).abs(), (xb * c).abs() + (xa * s).abs()
    return y, size


def append(pool, rows, table, seq_len, cu_q, picks=None):
    """A copy of pool (64 bits) with request b's rows written behind its seq_len[b] slots: rows
    cu_q[b] .. cu_q[b + 1] - 1, or the packed rows picks[b]."""
    out = pool.double().clone()
    ps = pool.shape[2]
    for b, n0 in enumerate(seq_len):
        src = picks[b] if picks is not None else range(cu_q[b], cu_q[b + 1])
        for j, r in enumerate(src):
            t = n0 + j
            out[int(table[b][t // ps]), :, t % ps] = rows[r].double()
    return out
