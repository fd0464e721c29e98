"""What rounding may cost latent attention, norm by norm and term by term.

A bf16 rounding is off by at most U = 2^-8 of the value.  Where each of many terms
is rounded by itself, the norm of a sum's error is at most U times the root of the
sum of the terms' squares if the errors are independent (0.58 U on average, a uniform
error's deviation, which leaves 1.7 times for what is not).
"""
import pytest
import torch

from _util import banner
from atomic_ops import latent as L
from oracle import latent as ol

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -8


def _two_tokens(H, n, length, page, at_a, at_b, dc, seed):
    """A cache of one sequence in which two tokens weigh nearly the same and the
    others nothing (scores of -16 and below against 0 and -0.03).  Their latents are
    opposite, so o is the small difference of the two probabilities: in column 0
    as one latent, in columns 1 and 2 as two that the value projection adds."""
    g = torch.Generator().manual_seed(seed)
    dn, dr, dv = 64, 32, 64
    per = -(-length // page)
    table = torch.randperm(per + 1, generator=g)[:per].to(torch.int32)[None]
    rows = torch.zeros(per * page, dc + dr)
    rows[:, dc] = -32.0
    rows[at_a, 0], rows[at_b, 0] = 1, -1
    rows[at_a, 1], rows[at_b, 2] = 1, -1
    rows[at_a, dc], rows[at_b, dc] = 0, -0.03125
    cache = torch.full((per + 1, page, dc + dr), float("nan"))
    cache[table[0].long()] = rows.view(per, page, -1)
    q = torch.zeros(1, n, H, dn + dr)
    q[..., dn] = torch.rand(1, n, H, generator=g) + 0.5
    w = torch.randn(H, dn + dv, dc, generator=g) * dc ** -0.5
    w[:, dn:] = 0
    w[:, dn, 0] = 1
    w[:, dn + 1, 1:3] = 1
    return [t.to(BF16) for t in (q, w, cache)], table


@pytest.mark.parametrize("H,n,length,page,a,b,dc", [
    (4, 1, 20, 16, 2, 13, 64),          # one split, up to 16 rows
    (24, 1, 20, 16, 2, 13, 512),        # up to 32
    (64, 1, 60, 64, 2, 13, 512),        # and more
    (32, 2, 60, 64, 40, 13, 128),
    (16, 1, 300, 16, 3, 5, 512),        # splits joined in the last kernel
    (16, 1, 300, 16, 3, 250, 512),
    (16, 1, 6400, 64, 5, 7, 64),        # two hundred splits, joined before it
    (16, 1, 6400, 64, 5, 6000, 512),
    (40, 2, 6400, 64, 6000, 5, 64),
])
def test_decode_weights_have_sixteen_bits(H, n, length, page, a, b, dc):
    """Probabilities and the joined latent enter their products as two bf16 numbers
    each, which leave out 2^-18 of them; fp32 sums and exponentials of arguments below
    0.1 less.  So o, 0.01 to 0.03 as a difference of two halves, is within 2^-16 and
    its own rounding.  One bf16 number (eight bits) in either place is off by 2^-10 of
    a half and does not pass."""
    banner(f"latent decode weights H{H} n{n} length {length} tokens {a} {b} dc {dc}")
    (q, w, cache), table = _two_tokens(H, n, length, page, a, b, dc, seed=H + length)
    e = torch.exp(q[0, :, :, 64].double() * -0.03125)
    want = (1 - e) / (1 + e)
    tol = U * want + 2.0 ** -16
    for eight in ((1 - e.to(BF16).double()) / (1 + e),
                  (1 / (1 + e)).to(BF16).double() - (e / (1 + e)).to(BF16).double()):
        assert ((eight - want).abs() > tol).any()
    ln = torch.tensor([length], dtype=torch.int32)
    o = L.decode(*(t.cuda() for t in (q, w, cache, table, ln)), 1.0).double().cpu()[0]
    for i in range(2):
        assert ((o[..., i] - want).abs() <= tol).all(), (o[..., i] - want).abs().max()
    assert (o[..., 2:] == 0).all()


@pytest.mark.parametrize("H,n", [(4, 1), (24, 2), (16, 4)])
def test_decode_of_hundreds_of_splits(H, n):
    """q_lat and o are rounded once each; with scores of unit spread q_lat's errors
    reach o as o's own do: within 0.82 U of the norm, twice that in a row."""
    banner(f"latent decode splits H{H} n{n}")
    g = torch.Generator().manual_seed(H)
    r = lambda *s: torch.randn(*s, generator=g)
    B, dn, dr, dv, dc, page, lens = 2, 64, 32, 64, 64, 48, [6400, 3]
    per = -(-6400 // page)
    table = torch.randperm(B * per, generator=g).view(B, per).to(torch.int32)
    q, w, cache = r(B, n, H, dn + dr).to(BF16), (r(H, dn + dv, dc) * dc ** -0.5).to(BF16), r(B * per, page, dc + dr).to(BF16)
    o = L.decode(*(t.cuda() for t in (q, w, cache, table, torch.tensor(lens, dtype=torch.int32))), 96 ** -0.5)
    want = ol.decode(q, w, cache, table, lens, 96 ** -0.5)
    off, size = (o.double().cpu() - want).norm(dim=-1), want.norm(dim=-1)
    assert (off <= 2 * U * size).all(), (off / size.clamp(min=1e-30)).max()
    for b in range(B):
        assert off[b].norm() <= U * size[b].norm()


@pytest.mark.parametrize("B,T,S,H,widths,causal,ql,kl,dtype", [
    (1, 1100, 1100, 2, (128, 64, 128), True, None, None, BF16),     # several blocks of 256 rows on kept score gradients
    (2, 700, 900, 1, (128, 64, 128), True, [700, 513], [900, 700], BF16),
    (1, 1030, 520, 1, (64, 32, 64), False, None, None, BF16),
    (1, 40, 5000, 2, (128, 64, 128), True, None, [4800], BF16),
    (1, 600, 600, 1, (128, 64, 128), True, None, None, F32),
    (1, 40, 5000, 1, (64, 32, 64), False, None, None, F32),
])
def test_norms_of_outputs_and_gradients(B, T, S, H, widths, causal, ql, kl, dtype):
    """p and ds are rounded before their products and every result once: per head,
    each within U sqrt(|result|^2 + sum of its terms' squares).  float32: 1e-5 of the
    same (a score's rounding, 3e-6 of its size, in p, and sums of up to 5000 terms)."""
    banner(f"latent norms B{B} T{T} S{S} H{H} {widths} causal={causal} {ql} {kl} {dtype}")
    dn, dr, dv = widths
    g = torch.Generator().manual_seed(T)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    q, kv, k_pe, do = r(B, T, H, dn + dr), r(B, S, H, dn + dv), r(B, S, dr), r(B, T, H, dv)
    scale, u = (dn + dr) ** -0.5, U if dtype == BF16 else 1e-5
    dev = [t.cuda() for t in (q, kv, k_pe)]
    i32 = lambda v: None if v is None else torch.tensor(v, dtype=torch.int32, device="cuda")
    kw = dict(causal=causal, q_lens=i32(ql), kv_lens=i32(kl))
    o, lse, rest = L.forward(*dev, scale, save=True, **kw)
    dq, dkv, dk_pe = L.backward(*dev, o, lse, do.cuda(), scale, rest=rest, **kw)
    o, dq, dkv, dk_pe = (t.double().cpu() for t in (o, dq, dkv, dk_pe))

    def near(got, want, terms, what):
        bound = u * (want.square().sum() + terms).sqrt()
        assert (got - want).norm() <= bound, f"{what}: {(got - want).norm() / want.norm():.2e}, bound {bound / want.norm():.2e}"

    for b in range(B):
        nq, nk = T if ql is None else ql[b], S if kl is None else kl[b]
        see = ol.visible(T, S, nq, nk, causal)
        want_pe, terms_pe = 0, 0
        for h in range(H):
            k, v = torch.cat((kv[b, :, h, :dn], k_pe[b]), 1).double(), kv[b, :, h, dn:].double()
            x, up = q[b, :, h].double(), do[b, :, h].double()
            p, _ = ol._probs(x, k, scale, see)
            near(o[b, :, h], p @ v, (p.square() @ v.square()).sum(), "o")
            dp = up @ v.t()
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
            near(dq[b, :, h], ds @ k, (ds.square() @ k.square()).sum(), "dq")
            near(dkv[b, :, h, dn:], p.t() @ up, (p.square().t() @ up.square()).sum(), "dv")
            dk, terms = ds.t() @ x, ds.square().t() @ x.square()
            near(dkv[b, :, h, :dn], dk[:, :dn], terms[:, :dn].sum(), "dk")
            want_pe, terms_pe = want_pe + dk[:, dn:], terms_pe + terms[:, dn:].sum()
        near(dk_pe[b], want_pe, terms_pe, "dk_pe")
