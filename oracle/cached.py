"""float64 CPU restatement of the operators that continue sequences from cached state.

* the paged KV cache and causal attention over it: per segment the eager path ``softmax(q @
  repeat_kv(k)^T * scale + causal) @ repeat_kv(v)`` ([tf]:582-617) over gathered cache rows;
* the recurrent gated delta rule from a given state ([tf]:314-353);
* the causal convolution + SiLU behind cached inputs ([tf]:451-474).
"""
from __future__ import annotations

import math

import torch

F64 = torch.float64


def power_of_two(e: torch.Tensor) -> torch.Tensor:
    return torch.ldexp(torch.ones(e.shape, dtype=F64), e)


def e4m3_round(y: torch.Tensor) -> torch.Tensor:
    """Nearest e4m3 value (ties to even), float64; |y| <= 448 expected.  Spacing 2^(floor(log2|y|) - 3),
    2^-9 below 2^-6."""
    m, e = torch.frexp(y.abs().clamp_min(2.0 ** -6))
    step = torch.ldexp(torch.ones_like(m), e - 4)
    return torch.round(y / step) * step


def quantise(x: torch.Tensor):
    """Row scale exponents and the values an e4m3 cache row stands for: the smallest e in [-127, 127]
    with max|x| <= 448 * 2^e."""
    x = x.to(F64)
    m, e = torch.frexp(x.abs().amax(-1))
    e = (e - 9 + (m > 0.875).to(e.dtype))
    e = torch.where(m == 0, torch.full_like(e, -127), e).clamp(-127, 127)
    s = power_of_two(e)[..., None]
    return e, e4m3_round(x / s) * s


def cache_rows(cache, scale, page_table_row, length: int):
    """Rows [0, length) of one sequence, [length, Hkv, D] float64, decoded from their bits."""
    page = cache.shape[2]
    pos = torch.arange(length)
    ids = page_table_row.long()[pos // page]
    if cache.dtype == torch.bfloat16:
        return cache[ids, :, pos % page].to(F64)
    b = cache.view(torch.uint8)[ids, :, pos % page].long()
    exp, man = (b >> 3) & 15, (b & 7).to(F64)
    mag = torch.where(exp > 0, torch.ldexp(1 + man / 8, exp - 7), man / 8 * 2.0 ** -6)
    val = torch.where(b >= 128, -mag, mag)
    return val * power_of_two(scale[ids, :, pos % page].long() - 127)[..., None]


def paged_attention(q, k_cache, v_cache, page_table, cu, kv_lens, k_scale=None, v_scale=None, scale=None):
    """Returns ``(out, mag, size)``: out [T, Hq, D]; per element, sum_p softmax(..)_p |v_p| -- what a
    relative rounding of the softmax weights is multiplied by; and per row [T, Hq, 1], the largest
    scale * sum_d |q_d k_pd| over its visible keys -- what a score's accumulation error is relative to."""
    T, hq, D = q.shape
    hkv = k_cache.shape[1]
    rep = hq // hkv
    sc = D ** -0.5 if scale is None else scale
    out, mag = torch.zeros(T, hq, D, dtype=F64), torch.zeros(T, hq, D, dtype=F64)
    size = torch.zeros(T, hq, 1, dtype=F64)
    for s in range(len(kv_lens)):
        t0, t1, length = int(cu[s]), int(cu[s + 1]), int(kv_lens[s])
        n = t1 - t0
        if n <= 0 or length <= 0:
            continue
        k = cache_rows(k_cache, k_scale, page_table[s], length)
        v = cache_rows(v_cache, v_scale, page_table[s], length)
        last = length - n + torch.arange(n)
        for h in range(hq):
            z = q[t0:t1, h].to(F64) @ k[:, h // rep].t() * sc
            hidden = torch.arange(length)[None] > last[:, None]
            za = (q[t0:t1, h].to(F64).abs() @ k[:, h // rep].t().abs() * abs(sc)).masked_fill(hidden, 0)
            size[t0:t1, h, 0] = za.amax(-1)
            z = z.masked_fill(hidden, -math.inf)
            p = torch.exp(z - z.amax(-1, keepdim=True).clamp_min(-1e300))
            p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
            out[t0:t1, h] = p @ v[:, h // rep]
            mag[t0:t1, h] = p @ v[:, h // rep].abs()
    return out, mag, size


def recurrent_delta(q, k, v, g, beta, state, cu, l2norm: bool = True):
    """``q, k [T, Hk, Dk]``, ``v [T, H, Dv]``, ``state [S, H, Dk, Dv]`` -> (o [T, H, Dv], states [S, ...])."""
    q, k, v, g, beta = (t.to(F64) for t in (q, k, v, g, beta))
    rep = v.shape[1] // q.shape[1]
    q, k = q.repeat_interleave(rep, 1), k.repeat_interleave(rep, 1)
    if l2norm:
        q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + 1e-6)
        k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    q = q / math.sqrt(q.shape[-1])
    out = torch.zeros(v.shape, dtype=F64)
    finals = []
    for s in range(len(cu) - 1):
        S = state[s].to(F64)
        for t in range(int(cu[s]), int(cu[s + 1])):
            S = S * g[t].exp()[:, None, None]
            u = beta[t][:, None] * (v[t] - (S * k[t][:, :, None]).sum(1))
            S = S + k[t][:, :, None] * u[:, None, :]
            out[t] = (S * q[t][:, :, None]).sum(1)
        finals.append(S)
    return out, torch.stack(finals)


def conv_silu(x, w, history, cu):
    """``x [T, C]``, ``w [C, K]``, ``history [S, K - 1, C]`` -> (y [T, C], pre-activation, new history)."""
    K = w.shape[1]
    y = torch.zeros(x.shape, dtype=F64)
    finals = []
    for s in range(len(cu) - 1):
        rows = torch.cat([history[s].to(F64), x[int(cu[s]):int(cu[s + 1])].to(F64)])
        n = rows.shape[0] - (K - 1)
        for t in range(n):
            y[int(cu[s]) + t] = (rows[t:t + K] * w.to(F64).t()).sum(0)
        finals.append(rows[n:])
    return y * torch.sigmoid(y), y, torch.stack(finals)
