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


def _tokens(cache, table, ln):
    page = cache.shape[1]
    rows = [cache[int(table[j // page]), j % page] for j in range(ln)]
    return torch.stack(rows).to(F) if rows else torch.zeros(0, cache.shape[2], dtype=F)


def decode_shared(q, w_kv, cache, prefix_table, prefix_lens, table, kv_lens, scale, cos=None, sin=None,
                  interleaved=False):
    """(o [B, n, H, dv], weights [B, tokens of the table]): the sequences' own tokens
    stand behind their prefix's; ``weights`` sum each own token's probabilities over the
    heads and query tokens.  ``prefix_table`` None: no prefixes."""
    B, n, H, d = q.shape
    dc = w_kv.shape[2]
    dn = d - (cache.shape[2] - dc)
    page = cache.shape[1]
    w = w_kv.to(F)
    o = torch.zeros(B, n, H, w.shape[1] - dn, dtype=F)
    weights = torch.zeros(B, table.shape[1] * page, dtype=F)
    for b in range(B):
        ln = min(max(int(kv_lens[b]), 0), table.shape[1] * page)
        rows = _tokens(cache, table[b], ln)
        P = 0
        if prefix_table is not None:
            g = b // (B // prefix_table.shape[0])
            P = min(max(int(prefix_lens[g]), 0), prefix_table.shape[1] * page)
            rows = torch.cat((_tokens(cache, prefix_table[g], P), rows))
        up = torch.einsum("hrc,jc->hjr", w, rows[:, :dc])                       # each head's keys and values
        for t in range(n):
            pos = P + ln - n + t
            if pos < 0:
                continue
            qp = q[b, t, :, dn:].to(F)
            if cos is not None:
                qp = rotate(qp, torch.full((H,), pos), cos, sin, interleaved)
            seen = slice(0, pos + 1)
            s = (torch.einsum("hjr,hr->hj", up[:, seen, :dn], q[b, t, :, :dn].to(F)) + qp @ rows[seen, dc:].t()) * scale
            p = torch.softmax(s, 1)
            o[b, t] = torch.einsum("hj,hjv->hv", p, up[:, seen, dn:])
            own = p[:, P:].sum(0)
            weights[b, :own.numel()] += own
    return o, weights


def gathered(before, add, kv_lens, n):
    """The weights [B, W] after a step of n query tokens whose sums are ``add`` [B, ...]."""
    after = before.to(F).clone()
    for b, ln in enumerate(kv_lens):
        for j in range(min(max(int(ln), 0), add.shape[1])):
            after[b, j] = (after[b, j] if j < int(ln) - n else 0) + add[b, j]
    return after


def evict(kv_lens, weights, order, keep, sinks, recent):
    """(kv_lens, weights, order, source) as lists of the sequences' rows; a list's
    length is the new length."""
    out = []
    for b, ln in enumerate(kv_lens):
        w, age = [float(x) for x in weights[b, :ln]], [int(x) for x in order[b, :ln]]
        fresh = [j for j in range(ln) if age[j] < 0]
        top = max(age, default=-1)
        for j in fresh:
            age[j] = max(top, -1) + 1 + j - fresh[0]
        new = max(age, default=-1)
        safe = lambda j: age[j] < sinks or age[j] > new - recent  # noqa: E731
        rank = lambda j: (not safe(j), math.isnan(w[j]), -w[j] if not math.isnan(w[j]) else 0, j)  # noqa: E731
        stay = set(sorted(range(ln), key=rank)[:keep])
        came = iter(sorted(j for j in stay if j >= keep))
        source = [j if j in stay else next(came) for j in range(min(ln, keep))]
        out.append((len(source), [w[j] for j in source], [age[j] for j in source], source))
    return tuple(list(x) for x in zip(*out))
