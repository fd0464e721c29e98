"""CPU oracle of latent attention: the expanded form with its gradient, the
absorbed form over a paged cache and the rotation.

TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).

Plain restatements of the formulas in float64.  ``expanded`` and ``decode``
loop over batch rows and heads; ``expanded_grads`` returns, beside each
gradient, the sum of the absolute values of its terms, from which a test takes
the error that rounding the operands of a product can cause.
"""
from __future__ import annotations

import math

import torch

F = torch.float64


def rotate(x, positions, cos, sin, interleaved):
    """x [..., N, (H,) dr] with positions [N]; each pair turned by its angle."""
    d = x.shape[-1]
    x = x.to(F)
    c, s = cos.to(F)[positions.long()], sin.to(F)[positions.long()]
    while c.dim() < x.dim():
        c, s = c.unsqueeze(-2), s.unsqueeze(-2)
    out = torch.empty_like(x)
    i = torch.arange(d // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + d // 2)
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def _lens(t, n, most):
    return [most] * n if t is None else [min(max(int(v), 0), most) for v in t]


def visible(T, S, ql, kl, causal):
    """bool [T, S]: query i (of ql) sees key j (of kl)."""
    i, j = torch.arange(T)[:, None], torch.arange(S)[None]
    v = (i < ql) & (j < kl)
    return v & (j <= i + kl - ql) if causal else v


def _head(q, kv, k_pe, b, h):
    dn = q.shape[-1] - k_pe.shape[-1]
    k = torch.cat((kv[b, :, h, :dn], k_pe[b]), -1).to(F)
    return q[b, :, h].to(F), k, kv[b, :, h, dn:].to(F)


def _probs(q, k, scale, see):
    """(p, lse) with masked places left out altogether (they may hold anything)."""
    s = torch.where(see, q @ k.t() * scale, torch.full((), -math.inf, dtype=F))
    lse = torch.logsumexp(s, 1)
    p = torch.where(see, torch.exp(s - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[:, None]),
                    torch.zeros((), dtype=F))
    return p, lse


def _clean(x, n):
    """Rows past n as zeros."""
    x = x.clone()
    x[n:] = 0
    return x


def expanded(q, kv, k_pe, scale, causal=True, q_lens=None, kv_lens=None):
    """(o [B, T, H, dv], lse [B, H, T], the sum of p |v| [B, T, H, dv])."""
    B, T, H, _ = q.shape
    S = kv.shape[1]
    dv = kv.shape[3] - (q.shape[3] - k_pe.shape[2])
    o, mag = torch.zeros(B, T, H, dv, dtype=F), torch.zeros(B, T, H, dv, dtype=F)
    lse = torch.full((B, H, T), -math.inf, dtype=F)
    for b, (ql, kl) in enumerate(zip(_lens(q_lens, B, T), _lens(kv_lens, B, S))):
        see = visible(T, S, ql, kl, causal)
        for h in range(H):
            qh, k, v = _head(q, kv, k_pe, b, h)
            k, v = _clean(k, kl), _clean(v, kl)
            p, lse[b, h] = _probs(_clean(qh, ql), k, scale, see)
            o[b, :, h], mag[b, :, h] = p @ v, p @ v.abs()
    return o, lse, mag


def expanded_grads(q, kv, k_pe, dout, scale, causal=True, q_lens=None, kv_lens=None):
    """((dq, dkv, dk_pe), (their magnitudes)).  A magnitude is the sum of the
    absolute values of the gradient's terms, with |ds| taken as
    p (|dp| + 2 sum p |v| |do|): what ds can be off by, relative to one rounding of
    o and one of itself."""
    B, T, H, _ = q.shape
    S, dr = k_pe.shape[1:]
    dn = q.shape[3] - dr
    g = [torch.zeros(t.shape, dtype=F) for t in (q, kv, k_pe)]
    m = [torch.zeros(t.shape, dtype=F) for t in (q, kv, k_pe)]
    for b, (ql, kl) in enumerate(zip(_lens(q_lens, B, T), _lens(kv_lens, B, S))):
        see = visible(T, S, ql, kl, causal)
        for h in range(H):
            qh, k, v = _head(q, kv, k_pe, b, h)
            qh, k, v, do = _clean(qh, ql), _clean(k, kl), _clean(v, kl), _clean(dout[b, :, h].to(F), ql)
            p, _ = _probs(qh, k, scale, see)
            dp = do @ v.t()
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
            size = p * (dp.abs() + 2 * ((p @ v.abs()) * do.abs()).sum(1, keepdim=True)) * abs(scale)
            for out, w, x in ((g, ds, lambda t: t), (m, size, torch.abs)):
                out[0][b, :, h] = w @ x(k)
                dk = w.t() @ x(qh)
                out[1][b, :, h, :dn] = dk[:, :dn]
                out[1][b, :, h, dn:] = p.t() @ x(do)
                out[2][b] += dk[:, dn:]
    return g, m


def decode(q, w_kv, cache, table, kv_lens, scale, cos=None, sin=None, interleaved=False):
    """o [B, n, H, dv] by the expanded formula: each cached latent is turned
    into the heads' keys and values first."""
    B, n, H, d = q.shape
    dc = w_kv.shape[2]
    dr = cache.shape[2] - dc
    dn, dv = d - dr, w_kv.shape[1] - (d - dr)
    page = cache.shape[1]
    o = torch.zeros(B, n, H, dv, dtype=F)
    for b in range(B):
        ln = min(max(int(kv_lens[b]), 0), table.shape[1] * page)
        rows = torch.stack([cache[int(table[b, j // page]), j % page] for j in range(ln)]).to(F) if ln else None
        for t in range(n):
            pos = ln - n + t
            if pos < 0:
                continue
            for h in range(H):
                up = rows[:pos + 1, :dc] @ w_kv[h].to(F).t()
                qp = q[b, t, h, dn:].to(F)
                if cos is not None:
                    qp = rotate(qp[None], torch.tensor([pos]), cos, sin, interleaved)[0]
                s = (up[:, :dn] @ q[b, t, h, :dn].to(F) + rows[:pos + 1, dc:] @ qp) * scale
                o[b, t, h] = torch.softmax(s, 0) @ up[:, dn:]
    return o
