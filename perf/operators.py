"""Latent attention and its paged cache, as timed cases.

Attention whose keys and values come from one latent vector a token: the
expanded form (prompts and training, with its gradient), the absorbed form that
reads the latents of a paged cache (single tokens, or a few at once), and the
call that appends to that cache and rotates by position on the way.

``listed()`` gives the named cases, ``draw(rng)`` further ones of the same
ranges, ``prepare`` / ``run`` one pass, ``work`` what the pass cannot do without
and ``exact`` the same results in 64 bits.  ``run`` computes the operators in
plain torch operations in 32 bits, or with ``own`` set through the library.
"""
from __future__ import annotations

import math
import os
import sys

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
# H heads; dn / dr: key width without position and rotated; dv: value width;
# dc: latent width; page: tokens a cache page.
def listed():
    return [
        # serving, one step: the new token of each of 32 sequences enters the cache
        dict(name="append_token", op="append", N=32, H=6, dn=128, dr=64, dc=512, page=64, skip=0, interleaved=False,
             dtype="bf16"),
        # serving, a prompt of 8192 tokens enters the cache
        dict(name="append_prompt", op="append", N=8192, H=16, dn=128, dr=64, dc=512, page=64, skip=0,
             interleaved=False, dtype="bf16"),
        # one user, a short conversation: latency
        dict(name="decode_one", op="decode", B=1, n=1, H=6, L=777, dn=128, dr=64, dv=128, dc=512, page=16,
             ragged=False, empty=False, interleaved=False, dtype="bf16"),
        # a full batch of conversations of all lengths
        dict(name="decode_batch", op="decode", B=64, n=1, H=16, L=8192, dn=128, dr=64, dv=128, dc=512, page=64,
             ragged=True, empty=False, interleaved=False, dtype="bf16"),
        # a few long documents
        dict(name="decode_long", op="decode", B=4, n=1, H=16, L=32768, dn=128, dr=64, dv=128, dc=512, page=64,
             ragged=False, empty=False, interleaved=False, dtype="bf16"),
        # a draft of four tokens checked at once, one slot of the batch idle
        dict(name="decode_draft", op="decode", B=8, n=4, H=16, L=4096, dn=128, dr=64, dv=128, dc=512, page=128,
             ragged=True, empty=True, interleaved=True, dtype="bf16"),
        # the float32 form, as for checking a model before going to bf16
        dict(name="decode_fp32", op="decode", B=3, n=1, H=8, L=1501, dn=64, dr=32, dv=64, dc=256, page=32,
             ragged=True, empty=False, interleaved=False, dtype="fp32"),
        # prefill of a long prompt
        dict(name="prompt", op="fwd", B=1, T=8192, S=8192, H=16, dn=128, dr=64, dv=128, ragged=False, empty=False,
             causal=True, dtype="bf16"),
        # two prompts of odd lengths continued after a cached prefix, in one padded batch
        dict(name="prompt_extend", op="fwd", B=2, T=517, S=4500, H=6, dn=128, dr=64, dv=128, ragged=True, empty=False,
             causal=True, dtype="bf16"),
        # a training step of the model's layer (d_model 768, six heads, micro batch 8 of 4096)
        dict(name="train_model", op="train", B=8, T=4096, S=4096, H=6, dn=128, dr=64, dv=128, ragged=False,
             empty=False, causal=True, dtype="bf16"),
        # a training step at the benchmark's length and heads
        dict(name="train_large", op="train", B=2, T=8192, S=8192, H=16, dn=128, dr=64, dv=128, ragged=False,
             empty=False, causal=True, dtype="bf16"),
        # a float32 training step on a padded batch
        dict(name="train_fp32", op="train", B=2, T=512, S=512, H=4, dn=64, dr=32, dv=64, ragged=True, empty=False,
             causal=True, dtype="fp32"),
    ]


def _log_int(rng, lo, hi):
    return min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "fwd", "train"])
    while True:
        dn, dr, dv = rng.choice([(128, 64, 128), (128, 64, 128), (64, 32, 64), (96, 32, 64), (56, 24, 72), (128, 32, 96)])
        dtype = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        if op == "append":
            c = dict(op=op, N=_log_int(rng, 1, 16384), H=_log_int(rng, 1, 32), dn=dn, dr=dr,
                     dc=rng.choice([128, 256, 512, 448]), page=rng.choice([1, 16, 24, 64, 128, 256]),
                     skip=rng.choice([0, 0, 3]), interleaved=rng.random() < 0.5, dtype=dtype)
            if c["N"] * (c["dc"] + 2 * dr + c["H"] * (dn + dr)) <= 1 << 25:
                return c
        elif op == "decode":
            c = dict(op=op, B=_log_int(rng, 1, 64), n=rng.choice([1, 1, 1, 2, 5, 8]), H=_log_int(rng, 1, 64),
                     L=_log_int(rng, 1, 32768), dn=dn, dr=dr, dv=dv, dc=rng.choice([128, 256, 512, 512, 448]),
                     page=rng.choice([1, 16, 24, 64, 128, 256]), ragged=rng.random() < 0.5, empty=rng.random() < 0.2,
                     interleaved=rng.random() < 0.5, dtype=dtype)
            most = 1 << 27 if dtype == "bf16" else 1 << 23
            if c["B"] * c["n"] * c["H"] * c["L"] <= 1 << 23 and c["B"] * c["L"] * (c["dc"] + dr) <= most:
                return c
        else:
            T = _log_int(rng, 1, 8192)
            S = T if op == "train" or rng.random() < 0.5 else _log_int(rng, 1, 8192)
            c = dict(op=op, B=_log_int(rng, 1, 8), T=T, S=S, H=_log_int(rng, 1, 16), dn=dn, dr=dr, dv=dv,
                     ragged=rng.random() < 0.4, empty=rng.random() < 0.2, causal=rng.random() < 0.8, dtype=dtype)
            most = (1 << 30 if op == "train" else 1 << 29) if dtype == "bf16" else 1 << 26
            if c["B"] * c["H"] * T * S <= most:
                return c


def _lengths(B, most, ragged, empty):
    """The sequences' lengths of a case: the first is whole, the others between half and whole where ragged."""
    n = [most - (b * 7919) % (most // 2 + 1) if ragged else most for b in range(B)]
    if empty:
        n[-1] = 0
    return n


def _attn_lengths(c):
    """(query lengths, key lengths); None where nothing is padded."""
    if not c["ragged"] and not c["empty"]:
        return None, None
    kv = _lengths(c["B"], c["S"], c["ragged"], c["empty"])
    q = list(kv) if c["S"] == c["T"] else _lengths(c["B"], c["T"], c["ragged"], False)
    return q, kv


# ------------------------------------------------------------------ inputs
def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32)


def _tables(rows, dr):
    """cos / sin of the rotation, as a model keeps them."""
    f = 1e4 ** (-torch.arange(0, dr, 2, device="cuda", dtype=torch.float64) / dr)
    a = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * f
    return a.cos().float(), a.sin().float()


def _ints(v, dtype=torch.int32):
    return None if v is None else torch.tensor(v, dtype=dtype, device="cuda")


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[c["dtype"]]
    s = {"case": c}
    if c["op"] == "append":
        N, page = c["N"], c["page"]
        pages = -(-N // page) + 3
        cos, sin = _tables(2 * N + 64, c["dr"])
        # the tokens of one projection: latent and rotated key are slices of its rows
        down = _randn(gen, N, c["dc"] + c["dr"]).to(dt)
        slots = torch.randperm(pages * page, generator=gen, device="cuda")[:N]
        if c["skip"]:
            slots[::c["skip"]] = -1
        s.update(cache=_randn(gen, pages, page, c["dc"] + c["dr"]).to(dt), c_kv=down[:, :c["dc"]],
                 k_pe=down[:, c["dc"]:], slots=slots, cos=cos, sin=sin,
                 positions=torch.randint(0, 2 * N + 64, (N,), generator=gen, device="cuda", dtype=torch.int32),
                 q=_randn(gen, N, c["H"], c["dn"] + c["dr"]).to(dt))
    elif c["op"] == "decode":
        B, page, L = c["B"], c["page"], c["L"]
        per = -(-L // page)
        pages = B * per + 1
        cos, sin = _tables(L + 1, c["dr"])
        s.update(q=_randn(gen, B, c["n"], c["H"], c["dn"] + c["dr"]).to(dt),
                 w_kv=(_randn(gen, c["H"], c["dn"] + c["dv"], c["dc"]) / math.sqrt(c["dc"])).to(dt),
                 cache=_randn(gen, pages, page, c["dc"] + c["dr"]).to(dt),
                 table=torch.randperm(pages, generator=gen, device="cuda")[:B * per].view(B, per).to(torch.int32),
                 kv_lens=_ints(_lengths(B, L, c["ragged"], c["empty"])), cos=cos, sin=sin)
    else:
        B, H = c["B"], c["H"]
        ql, kl = _attn_lengths(c)
        s.update(q=_randn(gen, B, c["T"], H, c["dn"] + c["dr"]).to(dt),
                 kv=_randn(gen, B, c["S"], H, c["dn"] + c["dv"]).to(dt), k_pe=_randn(gen, B, c["S"], c["dr"]).to(dt),
                 q_lens=_ints(ql), kv_lens=_ints(kl))
        if c["op"] == "train":
            s["do"] = _randn(gen, B, c["T"], H, c["dv"]).to(dt)
            for n in ("q", "kv", "k_pe"):
                s[n].requires_grad_(True)
    if c["op"] != "append":
        s["scale"] = (c["dn"] + c["dr"]) ** -0.5
    return s


# ------------------------------------------------------------- plain forms
def _rotated(x, cos, sin, interleaved):
    """x [..., dr] (32 bits) rotated by cos / sin [..., dr / 2]."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    a, b = x.chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _plain_append(s):
    c, dt = s["case"], s["c_kv"].dtype
    p = s["positions"].long()
    cos, sin = s["cos"][p], s["sin"][p]
    k = _rotated(s["k_pe"].float(), cos, sin, c["interleaved"]).to(dt)
    rows = s["cache"].view(-1, c["dc"] + c["dr"])
    row = torch.cat((s["c_kv"], k), -1)
    if c["skip"]:  # a slot below zero: the token does not enter the cache
        keep = s["slots"] >= 0
        rows[s["slots"][keep]] = row[keep]
    else:
        rows[s["slots"]] = row
    q_pe = _rotated(s["q"][..., c["dn"]:].float(), cos[:, None], sin[:, None], c["interleaved"]).to(dt)
    return {"cache": s["cache"], "k": k, "q": torch.cat((s["q"][..., :c["dn"]], q_pe), -1)}


def _softmax(sc, visible):
    """Probabilities over the visible keys (all zero in a row without any) and the log of their sum."""
    sc = sc.masked_fill(~visible, -math.inf)
    m = sc.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = (sc - m).exp_()
    tot = e.sum(-1, keepdim=True)
    lse = (m + tot.log()).squeeze(-1)
    return e.div_(tot.clamp(min=1e-30)), lse


def _plain_decode(s):
    c = s["case"]
    B, n, dn, dc = c["B"], c["n"], c["dn"], c["dc"]
    lat = s["cache"][s["table"].long()].flatten(1, 2).float()     # [B, tokens, dc + dr]
    lens = s["kv_lens"].long()
    pos = lens[:, None] - n + torch.arange(n, device=lens.device)  # [B, n]
    at = pos.clamp(min=0)
    w = s["w_kv"].float()
    q = s["q"].float()
    q_pe = _rotated(q[..., dn:], s["cos"][at][:, :, None], s["sin"][at][:, :, None], c["interleaved"])
    q_lat = torch.matmul(q[..., :dn].unsqueeze(-2), w[:, :dn]).squeeze(-2)   # [B, n, H, dc]
    rows = torch.cat((q_lat, q_pe), -1).flatten(1, 2)
    sc = torch.matmul(rows, lat.transpose(1, 2)) * s["scale"]
    tok = torch.arange(lat.shape[1], device=lens.device)
    visible = (tok <= pos[..., None]).repeat_interleave(c["H"], 1)
    p, _ = _softmax(sc, visible)
    o_lat = torch.matmul(p, lat[..., :dc]).view(B, n, c["H"], dc)
    o = torch.matmul(w[:, dn:], o_lat.unsqueeze(-1)).squeeze(-1)
    return {"o": o.to(s["q"].dtype)}


def _plain_attention(s):
    c = s["case"]
    T, S, dn, H = c["T"], c["S"], c["dn"], c["H"]
    q, kv, k_pe = (s[n].detach().float() for n in ("q", "kv", "k_pe"))
    dev = q.device
    q = q.transpose(1, 2)                                                                     # [B, H, T, d]
    k = torch.cat((kv[..., :dn], k_pe[:, :, None].expand(-1, -1, H, -1)), -1).transpose(1, 2)
    v = kv[..., dn:].transpose(1, 2)
    i, j = torch.arange(T, device=dev)[:, None], torch.arange(S, device=dev)
    ql = s["q_lens"].long().view(-1, 1, 1) if s["q_lens"] is not None else torch.full((1, 1, 1), T, device=dev)
    kl = s["kv_lens"].long().view(-1, 1, 1) if s["kv_lens"] is not None else torch.full((1, 1, 1), S, device=dev)
    visible = (i < ql) & (j < kl)
    if c["causal"]:
        visible = visible & (j <= i + (kl - ql))
    p, lse = _softmax(torch.matmul(q, k.transpose(2, 3)) * s["scale"], visible[:, None])
    o = torch.matmul(p, v)
    out = {"o": o.transpose(1, 2).to(s["q"].dtype), "lse": lse}
    if c["op"] == "fwd":
        return out
    do = s["do"].float().transpose(1, 2)
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = torch.matmul(do, v.transpose(2, 3))
    ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
    dq, dk = torch.matmul(ds, k), torch.matmul(ds.transpose(2, 3), q)
    dt = s["q"].dtype
    return {"o": out["o"], "dq": dq.transpose(1, 2).to(dt),
            "dkv": torch.cat((dk[..., :dn], dv), -1).transpose(1, 2).to(dt), "dk_pe": dk[..., dn:].sum(1).to(dt)}


# -------------------------------------------------------------------- pass
def run(state):
    s, c = state, state["case"]
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "fwd": _plain_attention,
                "train": _plain_attention}[c["op"]](s)
    L = _latent()
    if c["op"] == "append":
        k, q = L.append(s["cache"], s["c_kv"], s["k_pe"], s["slots"], s["positions"], s["cos"], s["sin"], q=s["q"],
                        interleaved=c["interleaved"])
        return {"cache": s["cache"], "k": k, "q": q}
    if c["op"] == "decode":
        return {"o": L.decode(s["q"], s["w_kv"], s["cache"], s["table"], s["kv_lens"], s["scale"], cos=s["cos"],
                              sin=s["sin"], interleaved=c["interleaved"])}
    if c["op"] == "fwd":
        o, lse = L.forward(s["q"], s["kv"], s["k_pe"], s["scale"], causal=c["causal"], q_lens=s["q_lens"],
                           kv_lens=s["kv_lens"])
        return {"o": o, "lse": lse}
    o = L.attention(s["q"], s["kv"], s["k_pe"], s["scale"], causal=c["causal"], q_lens=s["q_lens"],
                    kv_lens=s["kv_lens"])
    dq, dkv, dk = torch.autograd.grad(o, (s["q"], s["kv"], s["k_pe"]), s["do"])
    return {"o": o.detach(), "dq": dq, "dkv": dkv, "dk_pe": dk}


# -------------------------------------------------------------------- work
def _pairs(c):
    """Visible (query, key) pairs of a head over the whole batch."""
    ql, kl = _attn_lengths(c)
    total = 0
    for a, b in zip(ql or [c["T"]] * c["B"], kl or [c["S"]] * c["B"]):
        if not c["causal"]:
            total += a * b
        else:  # query i sees max(0, i + b - a + 1) keys
            first = max(0, a - b)
            total += sum((first + b - a + 1, b)) * (a - first) // 2 if a > first else 0
    return total


def work(case):
    c, es = case, _ES[case["dtype"]]
    d = c["dn"] + c["dr"]
    if c["op"] == "append":
        row = c["dc"] + c["dr"]
        return {"bytes": c["N"] * (es * (2 * row + c["dr"] + 2 * c["H"] * d) + 4 * c["dr"] + 12),
                "flops": 3 * c["N"] * (c["H"] + 1) * c["dr"]}
    if c["op"] == "decode":
        lens = _lengths(c["B"], c["L"], c["ragged"], c["empty"])
        seen = sum(max(0, ln - c["n"] + t + 1) for ln in lens for t in range(c["n"]))
        wide = c["dn"] + c["dv"]
        return {"bytes": es * (sum(lens) * (c["dc"] + c["dr"]) + c["H"] * wide * c["dc"]
                               + c["B"] * c["n"] * c["H"] * (d + c["dv"])) + 4 * sum(-(-ln // c["page"]) for ln in lens),
                "flops": 2 * c["H"] * (seen * (2 * c["dc"] + c["dr"]) + c["B"] * c["n"] * c["dc"] * wide)}
    rows, cols = c["B"] * c["T"], c["B"] * c["S"]
    once = es * (rows * c["H"] * (d + c["dv"]) + cols * (c["H"] * (c["dn"] + c["dv"]) + c["dr"]))
    mults = 2 * c["H"] * _pairs(c) * (d + c["dv"])
    if c["op"] == "fwd":
        return {"bytes": once + 4 * rows * c["H"], "flops": mults}
    return {"bytes": 2 * once + es * rows * c["H"] * c["dv"], "flops": 3 * mults}


# ------------------------------------------------------------------ 64 bits
def _turn(x, pos, dr, interleaved, tables):
    """The pairs of x as complex numbers, each times cos + i sin of its angle."""
    z = x.double().reshape(*x.shape[:-1], dr // 2, 2) if interleaved else \
        x.double().reshape(*x.shape[:-1], 2, dr // 2).transpose(-1, -2)
    turn = torch.complex(tables[0].double()[pos], tables[1].double()[pos])
    while turn.dim() < z.dim() - 1:
        turn = turn.unsqueeze(-2)
    z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn)
    return z.flatten(-2) if interleaved else z.transpose(-1, -2).flatten(-2)


def exact(case, seed):
    c = case
    s = prepare(c, seed)
    f = torch.float64
    dn, dr = c["dn"], c["dr"]
    if c["op"] == "append":
        pos, tab = s["positions"].long(), (s["cos"], s["sin"])
        k = _turn(s["k_pe"], pos, dr, c["interleaved"], tab)
        cache = s["cache"].to(f).view(-1, c["dc"] + dr)
        for t in (s["slots"] >= 0).nonzero().flatten().split(4096):
            cache[s["slots"][t]] = torch.cat((s["c_kv"][t].to(f), k[t]), 1)
        q = s["q"].to(f)
        q[..., dn:] = _turn(s["q"][..., dn:], pos, dr, c["interleaved"], tab)
        return {"cache": cache.view(s["cache"].shape), "k": k, "q": q}
    if c["op"] == "decode":
        o = torch.zeros(c["B"], c["n"], c["H"], c["dv"], dtype=f, device="cuda")
        w = s["w_kv"].to(f)
        for b, ln in enumerate(s["kv_lens"].tolist()):
            if ln == 0:
                continue
            at = torch.arange(ln, device="cuda")
            rows = s["cache"][s["table"][b].long()[at // c["page"]], at % c["page"]].to(f)
            # head by head as the expanded form: keys and values out of the latents
            for t in range(max(0, c["n"] - ln), c["n"]):
                p = ln - c["n"] + t
                qp = _turn(s["q"][b, t, :, dn:], torch.full((c["H"],), p, device="cuda"), dr, c["interleaved"],
                           (s["cos"], s["sin"]))
                seen = rows[:p + 1]
                lift = (s["q"][b, t, :, None, :dn].to(f) @ w[:, :dn])[:, 0]
                sc = (lift @ seen[:, :c["dc"]].t() + qp @ seen[:, c["dc"]:].t()) * s["scale"]
                o[b, t] = (w[:, dn:] @ (torch.softmax(sc, -1) @ seen[:, :c["dc"]])[..., None])[..., 0]
        return {"o": o}
    B, T, S, H = c["B"], c["T"], c["S"], c["H"]
    ql, kl = _attn_lengths(c)
    train = c["op"] == "train"
    o = torch.zeros(B, T, H, c["dv"], dtype=f, device="cuda")
    lse = torch.full((B, H, T), -math.inf, dtype=f, device="cuda")
    dq, dkv = (torch.zeros(s[n].shape, dtype=f, device="cuda") for n in ("q", "kv")) if train else (None, None)
    dk_pe = torch.zeros(s["k_pe"].shape, dtype=f, device="cuda")
    for b in range(B):
        a, e = (ql[b], kl[b]) if ql is not None else (T, S)
        lo = max(0, a - e) if c["causal"] else 0     # the queries before it see nothing
        if e == 0 or lo >= a:
            continue
        for h in range(H):
            q = s["q"][b, lo:a, h].detach().to(f)
            k = torch.cat((s["kv"][b, :e, h, :dn], s["k_pe"][b, :e]), 1).detach().to(f)
            v = s["kv"][b, :e, h, dn:].detach().to(f)
            sc = (q @ k.t()) * s["scale"]
            if c["causal"]:
                sc += torch.full_like(sc, -math.inf).triu_(e - a + lo + 1)
            lse[b, h, lo:a] = torch.logsumexp(sc, 1)
            p = torch.exp(sc - lse[b, h, lo:a, None])
            o[b, lo:a, h] = p @ v
            if train:
                do = s["do"][b, lo:a, h].to(f)
                dp = do @ v.t()
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) * s["scale"]
                dq[b, lo:a, h] = ds @ k
                dk = ds.t() @ q
                dkv[b, :e, h] = torch.cat((dk[:, :dn], p.t() @ do), 1)
                dk_pe[b, :e] += dk[:, dn:]
    return {"o": o, "dq": dq, "dkv": dkv, "dk_pe": dk_pe} if train else {"o": o, "lse": lse}
