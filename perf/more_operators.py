"""Serving from the latent cache when it is shared and when it is full, as timed cases.

The absorbed form of latent attention for a batch whose sequences share a long
prefix, the attention weight that each cached token has gathered, and the
eviction of the tokens that have gathered least.

``listed()`` gives the named cases, ``draw(rng)`` further ones of the same
ranges, ``prepare`` / ``run`` one pass, ``work`` what the pass cannot do without
and ``exact`` the same results in 64 bits.  ``run`` computes the operators in
plain torch operations in 32 bits, or with ``own`` set through the library.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

_PKG = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "atomic_ai_hybrid-v0.1_amd")
_DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
_ES = {"bf16": 2, "fp32": 4}


def _latent():
    if _PKG not in sys.path:
        sys.path.insert(0, _PKG)
    from atomic_ops import latent
    return latent


# ------------------------------------------------------------------- cases
# attend: B sequences of n query tokens and H heads; G prefixes of P tokens (0: none), the sequences in G equal runs;
# L own tokens of the longest; scored: the tokens' weights are gathered; dn / dr: key width without position and
# rotated; dv: value width; dc: latent width; page: tokens a cache page.
# evict: L tokens of the longest, of which `keep` stay, the first `sinks` and the newest `recent` among them;
# settled: rows that an earlier eviction has left in another order.
_MODEL = dict(dn=128, dr=64, dv=128, dc=512)
_SMALL = dict(dn=64, dr=32, dv=64, dc=256)


def _attend(name, B, H, L, n=1, G=1, P=0, page=64, ragged=False, idle=False, scored=False, interleaved=False,
            dtype="bf16", dims=None):
    c = dict(op="attend", B=B, n=n, H=H, G=G, P=P, L=L, page=page, ragged=ragged, idle=idle, scored=scored,
             interleaved=interleaved, dtype=dtype, **(dims or _MODEL))
    return dict(c, name=name) if name else c


def _evict(name, B, L, keep, sinks, recent, settled, page=64, ragged=False, dr=64, dc=512, dtype="bf16"):
    c = dict(op="evict", B=B, L=L, keep=keep, sinks=sinks, recent=recent, settled=settled, page=page, ragged=ragged,
             dr=dr, dc=dc, dtype=dtype)
    return dict(c, name=name) if name else c


def listed():
    return [
        # four questions to one short instruction: latency
        _attend("shared_few", B=4, H=6, P=777, L=33, page=16),
        # a full batch of conversations behind one system prompt
        _attend("shared_batch", B=64, H=16, P=8192, L=1024, ragged=True),
        # many questions to one long document
        _attend("shared_long", B=64, H=16, P=32768, L=512),
        # eight samples of each of four prompts, drafts of four tokens checked at once, one slot idle
        _attend("shared_samples", B=32, n=4, H=16, G=4, P=4096, L=777, page=128, ragged=True, idle=True,
                interleaved=True),
        # the float32 form, as for checking a model before going to bf16
        _attend("shared_fp32", B=6, H=8, G=2, P=1501, L=130, page=32, ragged=True, dtype="fp32", dims=_SMALL),
        # one user whose tokens' weights are gathered: latency
        _attend("scored_one", B=1, H=6, L=1000, page=16, scored=True),
        # a full batch, each token's weight gathered in every step
        _attend("scored_batch", B=64, H=16, L=8192, ragged=True, scored=True),
        # the same behind a shared prefix, which is never evicted
        _attend("scored_shared", B=32, H=16, P=8192, L=2048, scored=True, interleaved=True),
        # every step of a full cache: one token over the budget
        _evict("evict_step", B=64, L=2049, keep=2048, sinks=4, recent=256, settled=2048),
        # after a batch of prompts: a quarter stays
        _evict("evict_prompt", B=32, L=8192, keep=2048, sinks=4, recent=512, settled=0, ragged=True),
        # two long documents: an eighth stays
        _evict("evict_long", B=2, L=131072, keep=16384, sinks=4, recent=1024, settled=0),
        # odd sizes in float32; half of the sequences fit as they are
        _evict("evict_odd", B=7, L=5001, keep=3001, sinks=1, recent=100, settled=1500, page=24, ragged=True, dr=32,
               dc=256, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    op = rng.choice(["attend", "attend", "scored", "evict"])
    while True:
        dn, dr, dv = rng.choice([(128, 64, 128), (128, 64, 128), (64, 32, 64), (96, 32, 64), (56, 24, 72), (128, 32, 96)])
        dims = dict(dn=dn, dr=dr, dv=dv, dc=rng.choice([128, 256, 512, 512, 448]))
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        page = rng.choice([1, 16, 24, 64, 128, 256])
        if op == "evict":
            L = _log_int(rng, 2, 131072)
            keep = max(1, int(L * rng.choice([1.1, 0.98, rng.uniform(0.05, 0.95), rng.uniform(0.05, 0.95)])))
            sinks = min(rng.choice([0, 1, 4]), keep)
            c = _evict(None, B=_log_int(rng, 1, 64), L=L, keep=keep, sinks=sinks,
                       recent=int((keep - sinks) * rng.choice([0, rng.random() ** 2, 1])),
                       settled=rng.choice([0, min(keep, L), min(keep, L) // 2]), page=page, ragged=rng.random() < 0.5,
                       dr=dims["dr"], dc=dims["dc"], dtype=dtype)
            if c["B"] * L * (c["dc"] + c["dr"]) * _ES[dtype] <= 302 << 20:
                return c
        else:
            scored = op == "scored"
            G = rng.choice([1, 1, 2, 5])
            P = 0 if scored and rng.random() < 0.5 else _log_int(rng, 1, 32768)
            c = _attend(None, B=G * _log_int(rng, 1, 128 // G), H=_log_int(rng, 1, 64), L=_log_int(rng, 1, 8192),
                        n=rng.choice([1, 1, 1, 2, 5, 8]), G=G, P=P, page=page, ragged=rng.random() < 0.5,
                        idle=rng.random() < 0.2, scored=scored, interleaved=rng.random() < 0.5, dtype=dtype, dims=dims)
            rows = c["B"] * c["n"] * c["H"]
            if rows * P <= (1 << 25 if dtype == "bf16" else 1 << 22) and rows * c["L"] <= 1 << 23 and \
                    c["B"] * c["L"] * (c["dc"] + c["dr"]) <= (1 << 27 if dtype == "bf16" else 1 << 23):
                return c


def _lengths(B, most, ragged, idle=False):
    """The sequences' lengths of a case: the first is whole, the others between half and whole where ragged."""
    n = [most - (b * 7919) % (most // 2 + 1) if ragged else most for b in range(B)]
    if idle:
        n[-1] = 0
    return n


def _prefixes(c):
    return _lengths(c["G"], c["P"], c["ragged"])


def _owns(c):
    return _lengths(c["B"], c["L"], c["ragged"], c.get("idle", False))


# ------------------------------------------------------------------ inputs
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _rand(gen, *shape):
    return torch.rand(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _tables(rows, dr):
    """cos / sin of the rotation, as a model keeps them."""
    f = 1e4 ** (-torch.arange(0, dr, 2, device="cuda", dtype=torch.float64) / dr)
    a = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * f
    return a.cos().float(), a.sin().float()


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[c["dtype"]]
    B, L, page = c["B"], c["L"], c["page"]
    per = -(-L // page)
    lens = _owns(c)
    s = {"case": c, "kv_lens": _ints(lens)}
    if c["op"] == "attend":
        G, P = c["G"], c["P"]
        front = -(-P // page)
        pages = B * per + G * front + 1
        ids = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        s.update(q=_randn(gen, B, c["n"], c["H"], c["dn"] + c["dr"]).to(dt),
                 w_kv=(_randn(gen, c["H"], c["dn"] + c["dv"], c["dc"]) / math.sqrt(c["dc"])).to(dt),
                 cache=_randn(gen, pages, page, c["dc"] + c["dr"]).to(dt), scale=(c["dn"] + c["dr"]) ** -0.5,
                 table=ids[:B * per].view(B, per), prefix_table=ids[B * per:B * per + G * front].view(G, front),
                 prefix_lens=_ints(_prefixes(c)))
        s["cos"], s["sin"] = _tables(P + L + 1, c["dr"])
        if c["scored"]:   # what sixteen earlier steps have gathered
            s["weights"] = _rand(gen, B, per * page).square_() * (3 * 16 * c["H"] * c["n"] / L)
    else:
        pages = B * per + 1
        s.update(cache=_randn(gen, pages, page, c["dc"] + c["dr"]).to(dt),
                 table=torch.randperm(pages, generator=gen, device="cuda")[:B * per].view(B, per).to(torch.int32))
        W = per * page
        # a few tokens gather most of the weight; some were not looked at at all
        w = _randn(gen, B, W).mul_(2).exp_().mul_(_rand(gen, B, W) > 1 / 16)
        order = torch.full((B, W), -1, dtype=torch.int32, device="cuda")
        n = c["settled"]
        if n:             # the rows as earlier evictions left them: the sinks first, the others in no order
            first = min(c["sinks"], n)
            order[:, :first] = torch.arange(first, device="cuda", dtype=torch.int32)
            rest = torch.rand(B, 2 * n, generator=gen, device="cuda").argsort(1)[:, :n - first]
            order[:, first:n] = (first + rest).to(torch.int32)
        gone = torch.arange(W, device="cuda") >= s["kv_lens"][:, None]
        s.update(weights=w.masked_fill_(gone, 0), order=order.masked_fill_(gone, -1))
    return s


# ------------------------------------------------------------- plain forms
def _rotated(x, cos, sin, interleaved):
    """x [..., dr] (32 bits) rotated by cos / sin [..., dr / 2]."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_attend(s):
    c = s["case"]
    B, n, H, G, dn, dc = c["B"], c["n"], c["H"], c["G"], c["dn"], c["dc"]
    lat = s["cache"][s["table"].long()].flatten(1, 2).float()              # [B, tokens, dc + dr]
    front = s["cache"][s["prefix_table"].long()].flatten(1, 2).float()     # [G, tokens, dc + dr]
    P = front.shape[1]
    dev = lat.device
    lens, pre = s["kv_lens"].long(), s["prefix_lens"].long().repeat_interleave(B // G)
    at = lens[:, None] - n + torch.arange(n, device=dev)                   # [B, n], from the first own token on
    pos = (pre[:, None] + at).clamp(min=0)
    w, q = s["w_kv"].float(), s["q"].float()
    q_pe = _rotated(q[..., dn:], s["cos"][pos][:, :, None], s["sin"][pos][:, :, None], c["interleaved"])
    q_lat = torch.matmul(q[..., :dn].unsqueeze(-2), w[:, :dn]).squeeze(-2)   # [B, n, H, dc]
    rows = torch.cat((q_lat, q_pe), -1)
    sc = torch.cat((torch.matmul(rows.reshape(G, B // G * n * H, -1), front.transpose(1, 2)).view(B, n * H, P),
                    torch.matmul(rows.flatten(1, 2), lat.transpose(1, 2))), -1).mul_(s["scale"])
    tok = torch.arange(P, device=dev)
    see = torch.cat(((tok < pre[:, None, None]) & (tok <= pre[:, None, None] + at[..., None]),
                     torch.arange(lat.shape[1], device=dev) <= at[..., None]), -1).repeat_interleave(H, 1)
    sc.masked_fill_(~see, -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = sc.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    p.div_(p.sum(-1, keepdim=True).clamp_(min=1e-30))
    o_lat = torch.matmul(p[..., :P].reshape(G, B // G * n * H, P), front[..., :dc]).view(B, n, H, dc) + \
        torch.matmul(p[..., P:], lat[..., :dc]).view(B, n, H, dc)
    out = {"o": torch.matmul(w[:, dn:], o_lat.unsqueeze(-1)).squeeze(-1).to(s["q"].dtype)}
    if c["scored"]:
        j, wt = torch.arange(lat.shape[1], device=dev), s["weights"]
        wt.masked_fill_((j >= lens[:, None] - n) & (j < lens[:, None]), 0)   # the newest tokens' begin here
        out["weights"] = wt.add_(p[..., P:].sum(1))
    return out


def _plain_evict(s):
    c = s["case"]
    keep, page = c["keep"], c["page"]
    dev = s["cache"].device
    B, W = s["weights"].shape
    j = torch.arange(W, device=dev)
    lens = s["kv_lens"].long()[:, None]
    here = j < lens
    order = s["order"].long()
    new = here & (order < 0)                  # rows that no eviction has seen: the newest, in their order
    last = torch.where(here, order, -1).amax(1, keepdim=True)
    first = torch.where(new, j, W).amin(1, keepdim=True)
    order = torch.where(new, last + 1 + j - first, order)
    newest = torch.where(here, order, -1).amax(1, keepdim=True)
    safe = (order < c["sinks"]) | (order > newest - c["recent"])
    rank = torch.where(safe, math.inf, s["weights"]).masked_fill(~here, -math.inf)
    best = rank.sort(dim=1, descending=True, stable=True).indices[:, :keep]
    stay = torch.zeros(B, W, dtype=torch.bool, device=dev).scatter_(1, best, True) & here
    mover, hole = stay & (j >= keep), here & ~stay & (j < keep)
    # the k-th kept row past the budget goes to the k-th hole below it
    by_rank = torch.zeros(B, W + 1, dtype=torch.long, device=dev)
    by_rank.scatter_(1, torch.where(mover, mover.cumsum(1) - 1, W), j.expand(B, W))
    source = torch.where(hole, by_rank.gather(1, hole.cumsum(1).sub_(1).clamp_(min=0)), j.expand(B, W))
    left = lens.clamp(max=keep)
    inside = j < left
    b, to = (inside & (source != j)).nonzero(as_tuple=True)
    rows = s["cache"].view(-1, s["cache"].shape[2])
    slot = lambda t: s["table"][b, t // page].long() * page + t % page  # noqa: E731
    rows[slot(to)] = rows[slot(source[b, to])]
    source = torch.where(inside, source, 0)
    src = torch.where(inside, source, -1)[:, :keep]
    if keep > W:
        src = torch.cat((src, src.new_full((B, keep - W), -1)), 1)
    return {"cache": s["cache"], "kv_lens": left[:, 0].to(torch.int32), "source": src.to(torch.int32),
            "weights": torch.where(inside, s["weights"].gather(1, source), 0.0),
            "order": torch.where(inside, order.gather(1, source), -1).to(torch.int32)}


# -------------------------------------------------------------------- pass
def run(state):
    s, c = state, state["case"]
    if not own:
        return _plain_attend(s) if c["op"] == "attend" else _plain_evict(s)
    L = _latent()
    if c["op"] == "evict":
        lens, weights, order, source = L.evict(s["cache"], s["table"], s["kv_lens"], s["weights"], s["order"],
                                               c["keep"], sinks=c["sinks"], recent=c["recent"])
        return {"cache": s["cache"], "kv_lens": lens, "source": source, "weights": weights, "order": order}
    kw = dict(cos=s["cos"], sin=s["sin"], interleaved=c["interleaved"], weights=s.get("weights"))
    if c["P"]:
        o = L.decode_shared(s["q"], s["w_kv"], s["cache"], s["prefix_table"], s["prefix_lens"], s["table"],
                            s["kv_lens"], s["scale"], **kw)
    else:
        o = L.decode(s["q"], s["w_kv"], s["cache"], s["table"], s["kv_lens"], s["scale"], **kw)
    return {"o": o, "weights": s["weights"]} if c["scored"] else {"o": o}


# -------------------------------------------------------------------- work
def work(case):
    c, es = case, _ES[case["dtype"]]
    lens, row = _owns(c), c["dc"] + c["dr"]
    if c["op"] == "evict":
        keep, fixed = c["keep"], c["sinks"] + c["recent"]
        moved = 0.0
        for ln in lens:
            if ln > keep:      # the newest tokens, and of the others past the budget the share that stays
                late = min(c["recent"], ln - keep)
                moved += late + (ln - keep - late) * (keep - fixed) / max(1, ln - fixed)
        return {"bytes": 2 * moved * es * row + 16 * sum(lens) + 4 * c["B"] * keep + 8 * c["B"], "flops": sum(lens)}
    B, n, H, S = c["B"], c["n"], c["H"], c["B"] // c["G"]
    front, wide = _prefixes(c), c["dn"] + c["dv"]
    pairs = sum(max(0, min(front[b // S], front[b // S] + ln - n + t + 1)) + max(0, ln - n + t + 1)
                for b, ln in enumerate(lens) for t in range(n))
    return {"bytes": es * ((sum(lens) + sum(front)) * row + H * wide * c["dc"]
                           + B * n * H * (c["dn"] + c["dr"] + c["dv"]))
            + 4 * sum(-(-ln // c["page"]) for ln in lens + front) + (8 * sum(lens) if c["scored"] else 0),
            "flops": 2 * H * (pairs * (2 * c["dc"] + c["dr"]) + B * n * c["dc"] * wide)}


# ------------------------------------------------------------------ 64 bits
def _turn(x, pos, dr, interleaved, tables):
    """The pairs of x as complex numbers, each times cos + i sin of its angle."""
    z = x.double().reshape(*x.shape[:-1], dr // 2, 2) if interleaved else \
        x.double().reshape(*x.shape[:-1], 2, dr // 2).transpose(-1, -2)
    turn = torch.complex(tables[0].double()[pos], tables[1].double()[pos])
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
    return z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)


def _exact_attend(c, s):
    f = torch.float64
    B, n, H, dn, dc, page = c["B"], c["n"], c["H"], c["dn"], c["dc"], c["page"]
    o = torch.zeros(B, n, H, c["dv"], dtype=f, device="cuda")
    weights = s["weights"].to(f) if c["scored"] else None
    w = s["w_kv"].to(f)

    def tokens(table, ln):
        at = torch.arange(ln, device="cuda")
        return s["cache"][table.long()[at // page], at % page].to(f)

    fronts = [tokens(s["prefix_table"][g], ln) for g, ln in enumerate(_prefixes(c))]
    for b, ln in enumerate(_owns(c)):
        front = fronts[b // (B // c["G"])]
        P = front.shape[0]
        rows = torch.cat((front, tokens(s["table"][b], ln)))
        if c["scored"]:
            weights[b, max(0, ln - n):ln] = 0
        for t in range(n):
            p = P + ln - n + t
            if p < 0:
                continue
            seen = rows[:p + 1]
            lift = (s["q"][b, t, :, None, :dn].to(f) @ w[:, :dn])[:, 0]
            turned = _turn(s["q"][b, t, :, dn:], torch.full((H,), p, device="cuda"), c["dr"], c["interleaved"],
                           (s["cos"], s["sin"]))
            prob = torch.softmax((lift @ seen[:, :dc].t() + turned @ seen[:, dc:].t()) * s["scale"], -1)
            o[b, t] = (w[:, dn:] @ (prob @ seen[:, :dc])[..., None])[..., 0]
            if c["scored"] and p >= P:
                weights[b, :p + 1 - P] += prob[:, P:].sum(0)
    return {"o": o, "weights": weights} if c["scored"] else {"o": o}


def _exact_evict(c, s):
    keep, page = c["keep"], c["page"]
    cache = s["cache"].to(torch.float64).view(-1, c["dc"] + c["dr"])
    old = cache.clone()
    table = s["table"].cpu().numpy().astype(np.int64)
    before, order = s["weights"].cpu().numpy().astype(np.float64), s["order"].cpu().numpy().astype(np.int64)
    after = np.zeros_like(before)
    for b, ln in enumerate(_owns(c)):
        age = order[b, :ln].copy()
        fresh = np.flatnonzero(age < 0)
        age[fresh] = age.max(initial=-1) + 1 + fresh - (fresh[0] if fresh.size else 0)
        safe = (age < c["sinks"]) | (age > age.max(initial=-1) - c["recent"])
        # the last key sorts first: safe rows, then the weights from the largest, then the rows
        stay = np.sort(np.lexsort((np.arange(ln), -before[b, :ln], ~safe))[:keep])
        went = np.setdiff1d(np.arange(min(ln, keep)), stay)
        came = stay[stay >= keep]
        after[b, :min(ln, keep)] = before[b, :min(ln, keep)]
        after[b, went] = before[b, came]
        at = lambda r: torch.from_numpy(table[b, r // page] * page + r % page).to(cache.device)  # noqa: E731
        cache[at(went)] = old[at(came)]
    return {"cache": cache.view(s["cache"].shape), "kv_lens": None, "source": None,
            "weights": torch.from_numpy(after).cuda(), "order": None}


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_attend(case, s) if case["op"] == "attend" else _exact_evict(case, s)
