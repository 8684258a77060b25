"""Definitions of the prompt operators in float64, token by token and sequence by sequence."""

import math

import torch

F64 = torch.float64
EPS = 1e-6


def gdn(mixed, a, b, a_log, dt_bias, states, lens, fresh):
    """The recurrence of each sequence from ``states`` [N,HV,V,K] (zeros where ``fresh``): out [T,HV,V], states."""
    hv = states.shape[1]
    h = (mixed.shape[1] - hv * 128) // 256
    x = mixed.to(F64)
    q = x[:, :h * 128].reshape(-1, h, 128)
    k = x[:, h * 128:2 * h * 128].reshape(-1, h, 128)
    v = x[:, 2 * h * 128:].reshape(-1, hv, 128)
    q = (q / ((q * q).sum(-1, keepdim=True) + EPS).sqrt() / math.sqrt(128)).repeat_interleave(hv // h, 1)
    k = (k / ((k * k).sum(-1, keepdim=True) + EPS).sqrt()).repeat_interleave(hv // h, 1)
    g = -a_log.to(F64).exp() * torch.nn.functional.softplus(a.to(F64) + dt_bias.to(F64), threshold=1e9)
    beta = b.to(F64).sigmoid()
    out = torch.zeros(len(x), hv, 128, dtype=F64, device=x.device)
    final, t = [], 0
    for n, m in enumerate(lens):
        s = states[n].to(F64) * (0.0 if fresh[n] else 1.0)
        for _ in range(m):
            s = s * g[t].exp()[:, None, None]
            d = beta[t][:, None] * (v[t] - (s @ k[t][..., None])[..., 0])
            s = s + d[..., None] * k[t][:, None, :]
            out[t] = (s @ q[t][..., None])[..., 0]
            t += 1
        final.append(s)
    return out, torch.stack(final) if final else states.to(F64)


def norm_rope(x, weight, offset, eps, rows, interleaved):
    """x [T,H,D]; rows [T,rot] of the table."""
    x = x.to(F64)
    if weight is not None:
        x = x / ((x * x).mean(-1, keepdim=True) + eps).sqrt() * (weight.to(F64) + offset)
    half = rows.shape[1] // 2
    y = x.clone()
    for m in range(half):
        i, j = (2 * m, 2 * m + 1) if interleaved else (m, m + half)
        c, s = rows[:, m].to(F64)[:, None], rows[:, half + m].to(F64)[:, None]
        y[..., i] = x[..., i] * c - x[..., j] * s
        y[..., j] = x[..., j] * c + x[..., i] * s
    return y


def attention(q, k_cache, v_cache, table, kv_lens, q_lens, scale):
    """out [T,Hq,D], lse [T,Hq]; rows without a place are 0 and -inf."""
    hq, d = q.shape[1:]
    page, hk = k_cache.shape[1:3]
    outs, lses, t = [], [], 0
    for n, m in enumerate(q_lens):
        kv = int(kv_lens[n])
        pages = table[n, :-(-kv // page)].long() if kv else table[n, :0].long()
        k = k_cache[pages].reshape(-1, hk, d)[:kv].to(F64).repeat_interleave(hq // hk, 1)
        v = v_cache[pages].reshape(-1, hk, d)[:kv].to(F64).repeat_interleave(hq // hk, 1)
        x = torch.einsum("thd,shd->hts", q[t:t + m].to(F64), k) * scale
        seen = torch.arange(kv, device=q.device)[None, :] <= torch.arange(kv - m, kv, device=q.device)[:, None]
        x = x.masked_fill(~seen, -math.inf)
        lse = torch.logsumexp(x, -1) if kv else torch.full((hq, m), -math.inf, dtype=F64, device=q.device)
        w = torch.where(seen, torch.exp(x - torch.where(torch.isfinite(lse), lse, 0.0)[..., None]), 0.0)
        outs.append(torch.einsum("hts,shd->thd", w, v))
        lses.append(lse.T)
        t += m
    if not outs:
        return torch.zeros(q.shape, dtype=F64, device=q.device), torch.zeros(q.shape[:2], dtype=F64, device=q.device)
    return torch.cat(outs), torch.cat(lses)


def rel(x, y):
    """Relative 2-norm of x - y."""
    x, y = x.to(F64), y.to(F64)
    return float((x - y).norm() / y.norm().clamp(min=1e-300))


def cu(lens, device="cuda"):
    return torch.tensor([0] + list(lens), device=device).cumsum(0).to(torch.int32)
