"""64-bit restatement of the paged 4-bit cache and window attention operators
(test infrastructure only; CPU, torch float64, plain loops over batch and head).

Each attention result comes with the terms of its error bound: ``mass`` =
sum_j p_j |v_j| per output element and ``reach`` = max_j scale * sum_c |q_c k_jc|
per row, from which a test derives its tolerance.
"""
import math

import torch

GROUP, BLOCK, TINY = 64, 16, 2.0 ** -126


def quantise(x):
    """(codes [.., D], scale [.., D/64], minimum) with the FP32 arithmetic of the definition."""
    y = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = y.amin(-1), y.amax(-1)
    s, m = ((hi - lo) * torch.tensor(1.0 / 15.0)).to(torch.bfloat16).float(), lo.to(torch.bfloat16).float()
    s = torch.where(s < TINY, torch.zeros_like(s), s)
    inv = torch.where(s == 0, torch.zeros_like(s), 1.0 / s)
    u = ((y - m[..., None]) * inv[..., None]).round().clamp(0, 15).nan_to_num(nan=0.0)
    return u.flatten(-2), s, m


def dequantise(u, s, m):
    """scale * code + minimum in FP32 (product and sum rounded)."""
    return (u.float().unflatten(-1, (-1, GROUP)) * s[..., None] + m[..., None]).flatten(-2)


def rotate(x, cos, sin, interleaved):
    """FP32 rotation of the first 2*cos.shape[-1] channels; cos/sin broadcast to x's rows."""
    x = x.float().clone()
    R = 2 * cos.shape[-1]
    a, b = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    p, q = x[..., a].clone(), x[..., b].clone()
    x[..., a] = p * cos - q * sin
    x[..., b] = q * cos + p * sin
    return x


def decode(pool, table_row, head, n):
    """FP32 (K, V) [n, D] of the first n tokens of one sequence and head, byte by byte from the records."""
    blocks, D = pool.shape[2], pool.shape[3] // 18
    page = blocks * BLOCK
    out = torch.zeros((2, n, D))
    for j in range(n):
        rec = pool[int(table_row[j // page]), head, j % page // BLOCK]
        t = j % BLOCK
        for w in range(2):
            code = rec[w * 8 * D + t * D // 2: w * 8 * D + (t + 1) * D // 2].int()
            u = torch.stack((code & 15, code >> 4), -1).flatten()
            at = (16 + w) * D + t * D // GROUP * 4
            sm = rec[at: at + D // GROUP * 4].contiguous().view(torch.bfloat16).float().view(-1, 2)
            out[w, j] = dequantise(u, sm[:, 0], sm[:, 1])
    return out[0], out[1]


def visible(pos, n, causal, window, sinks):
    """Bool [len(pos), n]."""
    i, j = pos[:, None], torch.arange(n)[None, :]
    ok = torch.ones((len(pos), n), dtype=torch.bool)
    if causal:
        ok &= j <= i
    if window:
        ok &= (j > i - window) | (j < sinks)
    return ok


def attend(q, k, v, ok, scale):
    """One head: q [R,D], k/v [n,D], ok [R,n] -> (out, mass [R,D], reach [R]) in float64."""
    q, k, v = q.double(), k.double(), v.double()
    R, n = ok.shape
    if n == 0:
        return torch.zeros_like(q), torch.zeros_like(q), torch.zeros(R, dtype=torch.float64)
    s = (q @ k.T) * scale
    s = s.masked_fill(~ok, -math.inf)
    any_ = ok.any(-1, keepdim=True)
    p = torch.softmax(torch.where(any_, s, torch.zeros_like(s)), -1) * any_
    used = ok.any(0)                     # what no row sees may hold anything
    v = torch.where(used[:, None], v, torch.zeros_like(v))
    reach = ((q.abs() @ k.abs().T) * scale).masked_fill(~ok, 0.0).amax(-1)
    return p @ v, p @ v.abs(), reach


def paged_attention(q, pool, table, lengths, *, q_lengths=None, causal=True, window=0, sinks=0, scale=None):
    """HND q [B,Hq,Sq,D] over the cache -> (out, mass, reach [B,Hq,Sq])."""
    B, Hq, Sq, D = q.shape
    Hkv = pool.shape[1]
    scale = D ** -0.5 if scale is None else scale
    out, mass = torch.zeros((B, Hq, Sq, D), dtype=torch.float64), torch.zeros((B, Hq, Sq, D), dtype=torch.float64)
    reach = torch.zeros((B, Hq, Sq), dtype=torch.float64)
    for b in range(B):
        n = int(lengths[b])
        nq = Sq if q_lengths is None else min(int(q_lengths[b]), Sq)
        pos = n - nq + torch.arange(nq)
        ok = visible(pos, n, causal, window, sinks)
        for hk in range(Hkv):
            k, v = decode(pool, table[b], hk, n)
            for h in range(hk * (Hq // Hkv), (hk + 1) * (Hq // Hkv)):
                out[b, h, :nq], mass[b, h, :nq], reach[b, h, :nq] = attend(q[b, h, :nq], k, v, ok, scale)
    return out, mass, reach


def window_attention(q, k, v, *, kv_lengths=None, causal=True, window=0, sinks=0, scale=None):
    """HND q [B,Hq,Sq,D], k/v [B,Hkv,Sk,D] -> (out, mass, reach)."""
    B, Hq, Sq, D = q.shape
    Hkv, Sk = k.shape[1], k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    out, mass = torch.zeros((B, Hq, Sq, D), dtype=torch.float64), torch.zeros((B, Hq, Sq, D), dtype=torch.float64)
    reach = torch.zeros((B, Hq, Sq), dtype=torch.float64)
    for b in range(B):
        n = Sk if kv_lengths is None else max(0, min(int(kv_lengths[b]), Sk))
        ok = visible(Sk - Sq + torch.arange(Sq), n, causal, window, sinks)
        for h in range(Hq):
            hk = h // (Hq // Hkv)
            out[b, h], mass[b, h], reach[b, h] = attend(q[b, h], k[b, hk, :n], v[b, hk, :n], ok, scale)
    return out, mass, reach


UNIT = {torch.bfloat16: 2.0 ** -7, torch.float16: 2.0 ** -10}   # spacing at 1.0; half of it is a rounding


def attention_tolerance(out, mass, reach, dtype, D, *, operand_bits):
    """Elementwise bound of a kernel's error against the 64-bit result.

    The output is rounded once to ``dtype`` (half a unit).  With r = 2^-operand_bits
    the rounding of an operand of the matrix products (probabilities; keys and values
    too where the kernel rounds those): logits move by at most r * reach plus the FP32
    sum's D * 2^-23 * reach, which moves each probability by twice that relatively
    (itself and the sum), the probabilities' own rounding moves the result by r and the
    denominator's by r, the values' by r; the FP32 exponent and sums by 2^-18.
    """
    r = 2.0 ** -operand_bits
    logit = (r + D * 2.0 ** -23) * reach
    rel = 2 * logit + 3 * r + 2.0 ** -18
    floor = 2.0 ** -24 if dtype is torch.float16 else 0.0   # half the least subnormal, and a little
    return UNIT[dtype] / 2 * out.abs() * (1 + 2.0 ** -6) + rel[..., None] * 1.05 * mass + floor
