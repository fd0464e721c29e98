"""Latent attention on the GPU at its edges."""
import pytest
import torch
from torch.autograd import forward_ad

from _util import banner
from atomic_ops import latent as L
from oracle import latent as ol

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
NAN, INF = float("nan"), float("inf")


def _inputs(B, T, S, H, dn, dr, dv, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    return r(B, T, H, dn + dr), r(B, S, H, dn + dv), r(B, S, dr), r(B, T, H, dv)


def _i32(v):
    return None if v is None else torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,T,S,H,widths,causal,ql,kl,alone", [
    # alone: batch row -> the query rows that see one key
    (8, 1, 1, 3, (128, 64, 128), True, None, None, lambda b: range(1)),
    (2, 3, 1, 2, (64, 32, 64), False, None, None, lambda b: range(3)),
    (1, 300, 1, 2, (128, 64, 128), False, None, None, lambda b: range(300)),
    (1, 300, 1, 1, (56, 24, 72), True, None, None, lambda b: [299]),
    (3, 64, 64, 2, (128, 64, 128), True, [1, 40, 64], [1, 1, 1], lambda b: [(0, 39, 63)[b]]),
    (3, 64, 64, 2, (128, 64, 128), False, [1, 40, 64], [1, 1, 1], lambda b: range((1, 40, 64)[b])),
    (2, 300, 300, 2, (128, 64, 128), True, None, None, lambda b: [0]),
    (1, 200, 70, 2, (96, 32, 64), True, None, None, lambda b: [130]),
    (1, 700, 40, 1, (64, 32, 64), True, [690], [33], lambda b: [657]),   # the queries divided over workgroups
])
def test_a_query_of_one_key_gives_its_score_no_gradient(B, T, S, H, widths, causal, ql, kl, alone, dtype):
    """p is 1 whatever the score, so ds is zero: dq of such a query is zero, not a
    rounding, and so are the keys' gradients where no other query sees anything."""
    banner(f"latent one key B{B} T{T} S{S} H{H} {widths} causal={causal} {ql} {kl} {dtype}")
    dn, dr, dv = widths
    q, kv, k_pe, do = (t.cuda() for t in _inputs(B, T, S, H, dn, dr, dv, dtype, seed=T + S))
    kw = dict(causal=causal, q_lens=_i32(ql), kv_lens=_i32(kl))
    o, lse, rest = L.forward(q, kv, k_pe, 0.2, save=True, **kw)
    for r in (rest, None):
        dq, dkv, dk_pe = L.backward(q, kv, k_pe, o, lse, do, 0.2, rest=r, **kw)
        for b in range(B):
            assert (dq[b, list(alone(b))] == 0).all()
            n = T if ql is None else ql[b]
            first = max(0, n - (S if kl is None else kl[b])) if causal else 0   # the first query that sees anything
            if len(list(alone(b))) == n - first:
                assert (dq[b] == 0).all() and (dkv[b, ..., :dn] == 0).all() and (dk_pe[b] == 0).all()
            assert (dkv[b, 0, :, dn:] != 0).any()     # the value's gradient is there all the same
    # a NaN of the output's gradient is not hidden by the zero
    do[0, alone(0)[0]] = NAN
    dq = L.backward(q, kv, k_pe, o, lse, do, 0.2, rest=rest, **kw)[0]
    assert torch.isnan(dq[0, alone(0)[0]]).all()


def test_a_query_of_one_key_where_scores_are_computed_again():
    """As above past the score gradients that are kept (bfloat16, 4 GB)."""
    banner("latent one key, scores again")
    T = 46400
    d = [torch.zeros(1, T, *s, dtype=BF16, device="cuda") for s in ((1, 192), (1, 256), (64,))]
    do = torch.zeros(1, T, 1, 128, dtype=BF16, device="cuda")
    small = _inputs(1, 90, 70, 1, 128, 64, 128, BF16, seed=1)
    for t, x in zip((*d, do), small):
        t[:, :x.shape[1]] = x.cuda()
    for ql, kl, causal, alone in ((90, 70, True, [20]), (90, 1, False, range(90)), (1, 1, True, [0])):
        kw = dict(causal=causal, q_lens=_i32([ql]), kv_lens=_i32([kl]))
        o, lse, rest = L.forward(*d, 0.2, save=True, **kw)
        dq, dkv, dk_pe = L.backward(*d, o, lse, do, 0.2, rest=rest, **kw)
        assert (dq[0, list(alone)] == 0).all()
        assert kl > 1 or ((dkv[..., :128] == 0).all() and (dk_pe == 0).all() and (dkv[..., 128:] != 0).any())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T,S", [(70, 200), (70, 2100)])      # the keys in one part, and in several
def test_rows_past_the_length_are_zero_beside_a_last_query_that_is_not_finite(T, S, dtype):
    banner(f"latent padding beside NaN T{T} S{S} {dtype}")
    n = 40
    for bad in ("q", "v"):
        q, kv, k_pe, _ = (t.cuda() for t in _inputs(2, T, S, 2, 64, 32, 64, dtype, seed=S))
        if bad == "q":
            q[0, n - 1] = NAN
        else:
            kv[0, S - 1, :, 64:] = INF     # the last key, which the last query alone sees
        o, lse, rest = L.forward(q, kv, k_pe, 0.1, q_lens=_i32([n, T]), save=True)
        assert not torch.isfinite(o[0, n - 1]).any()
        assert (o[0, n:] == 0).all() and (lse[0, :, n:] == -INF).all()
        assert rest is None or (rest[0, n:] == 0).all()
        assert torch.isfinite(o[1]).all() and torch.isfinite(o[0, :n - 1]).all() or bad == "v"


def test_one_token_of_a_tensor_laid_out_token_first():
    """Tokens 50 MB apart of which one is taken: the dense tensors' bits."""
    banner("latent one token of far apart ones")
    B, H, dn, dr, dv = 1024, 128, 128, 64, 128
    wide = torch.empty(3, B, H, dn + dr, dtype=BF16, device="cuda")
    q, kv, k_pe, do = (t.cuda() for t in _inputs(B, 1, 2, 1, dn, dr, dv, BF16, seed=3))
    q, kv, do = (t.expand(-1, -1, H, -1) for t in (q, kv, do))
    wide[1] = q[:, 0]
    one = wide.transpose(0, 1)[:, 1:2]
    assert one.stride(1) * 2 > 1 << 25
    o, lse = L.forward(one, kv, k_pe, 0.1)
    o2, lse2 = L.forward(q, kv, k_pe, 0.1)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    for a, b in zip(L.backward(one, kv, k_pe, o, lse, do, 0.1), L.backward(q, kv, k_pe, o, lse, do, 0.1)):
        assert torch.equal(a, b)


def test_forward_mode_is_refused():
    """No tangent is computed, so none may get lost: dual tensors are an error, with and without a graph."""
    banner("latent forward mode")
    q, kv, k_pe, _ = (t.cuda() for t in _inputs(1, 8, 8, 1, 64, 32, 64, BF16, seed=24))
    for i in range(3):
        for graph in (False, True):
            x = [t.clone().requires_grad_(graph) for t in (q, kv, k_pe)]
            with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
                x[i] = forward_ad.make_dual(x[i], torch.ones_like(x[i]))
                L.attention(*x, 0.1)
    with forward_ad.dual_level():      # an open level by itself changes nothing
        o = L.attention(q, kv, k_pe, 0.1)
    assert torch.equal(o, L.attention(q, kv, k_pe, 0.1))


def _tables(rows, dr):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, dr, 2, dtype=torch.float64) / dr)
    return a.cos().float(), a.sin().float()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,H,dn,dr,inter", [(1, 1, 128, 64, False), (37, 3, 56, 24, True), (300, 2, 64, 32, False)])
def test_append_keeps_the_graph(N, H, dn, dr, inter, dtype):
    """k and q of ``append`` against the rotation's own gradient in 64 bits.  Its
    terms are two fp32 products and a sum, rounded once more in bf16 (at most
    three and a half 2^-24 of two terms of up to 6 each, and 2^-8 of itself).
    The unrotated part is passed on as it is; what the cache takes has no gradient."""
    banner(f"latent append graph N{N} H{H} {dn}/{dr} interleaved={inter} {dtype}")
    g = torch.Generator().manual_seed(N)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    k, q, gk, gq, c, cache = r(N, dr), r(N, H, dn + dr), r(N, dr), r(N, H, dn + dr), r(N, 64), r(N, 1, 64 + dr)
    pos = torch.randint(0, 60, (N,), generator=g, dtype=torch.int32)      # some past the tables
    cos, sin = _tables(50, dr)
    kx, qx, cx = (t.cuda().requires_grad_(True) for t in (k, q, c))
    dev, slots = cache.cuda(), torch.arange(N, device="cuda")
    ko, qo = L.append(dev, cx, kx, slots, pos.cuda(), cos.cuda(), sin.cuda(), q=qx, interleaved=inter)
    assert ko.requires_grad and qo.requires_grad and not dev.requires_grad
    with torch.no_grad():      # the same bits as without a graph
        k2, q2 = L.append(dev.clone(), cx, kx, slots, pos.cuda(), cos.cuda(), sin.cuda(), q=qx, interleaved=inter)
    assert torch.equal(ko, k2) and torch.equal(qo, q2) and not k2.requires_grad
    assert torch.equal(dev[:, 0], torch.cat((cx, ko), 1).detach())
    dk, dq, dc = torch.autograd.grad((ko, qo), (kx, qx, cx), (gk.cuda(), gq.cuda()), allow_unused=True)
    assert dc is None
    at = pos.clamp(max=49)
    want = []
    for x, up in ((k, gk), (q[..., dn:], gq[..., dn:])):
        x = x.double().requires_grad_(True)
        y = ol.rotate(x, at, cos, sin, inter)
        want.append(torch.autograd.grad(y, x, up.double())[0])
    tol = lambda x: (2.0 ** -8 if dtype == BF16 else 0.0) * x.abs() + 3.5 * 2.0 ** -24 * 12
    for a, b in ((dk, want[0]), (dq[..., dn:], want[1])):
        assert a.dtype == dtype and ((a.double().cpu() - b).abs() <= tol(b)).all()
    assert torch.equal(dq[..., :dn].cpu(), gq[..., :dn])
    # one of the two outputs by itself, keys without queries, a gradient that is one number broadcast
    ko, qo = L.append(None, None, kx, None, pos.cuda(), cos.cuda(), sin.cuda(), q=qx, interleaved=inter)
    assert torch.equal(torch.autograd.grad(qo, qx, gq.cuda(), retain_graph=True)[0], dq)
    assert torch.equal(torch.autograd.grad(ko, kx, gk.cuda())[0], dk)
    ko, none = L.append(None, None, kx, None, pos.cuda(), cos.cuda(), sin.cuda(), interleaved=inter)
    ones, = torch.autograd.grad(ko.sum(), kx)
    ko, none = L.append(None, None, kx, None, pos.cuda(), cos.cuda(), sin.cuda(), interleaved=inter)
    assert none is None and torch.equal(ones, torch.autograd.grad(ko, kx, torch.ones_like(ko))[0])


def test_gradient_of_append_follows_differences():
    """float32, linear in the inputs: the slope along a direction is the difference
    itself, up to the roundings (2^-24 of each of 2e3 terms' sizes, over a step of 1)."""
    banner("latent append differences")
    g = torch.Generator().manual_seed(7)
    r = lambda *s: torch.randn(*s, generator=g).cuda()
    q, u, up, k = r(9, 2, 96), r(9, 2, 96), r(9, 2, 96), r(9, 32)
    cos, sin = (t.cuda() for t in _tables(50, 32))
    pos = torch.arange(9, dtype=torch.int32, device="cuda") * 5
    f = lambda x: L.append(None, None, k, None, pos, cos, sin, q=x)[1]
    x = q.clone().requires_grad_(True)
    d, = torch.autograd.grad(f(x), x, up)
    slope = ((f(q + u).double() - f(q).double()) * up.double()).sum()
    assert abs(slope - (d.double() * u.double()).sum()) < 1e-3


def test_append_refuses_what_has_no_gradient():
    banner("latent append refusals in a graph")
    z = lambda *s: torch.zeros(*s, device="cuda")
    pos, slots = torch.zeros(5, dtype=torch.int32, device="cuda"), torch.arange(5, device="cuda")
    for i in range(3):
        cache, cos, sin = (z(*s).requires_grad_(i == j) for j, s in enumerate(((5, 1, 96), (9, 16), (9, 16))))
        with pytest.raises(ValueError, match="no gradient"):
            L.append(cache, z(5, 64), z(5, 32), slots, pos, cos, sin)
    k = z(5, 32)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
        L.append(None, None, forward_ad.make_dual(k, torch.ones_like(k)), None, pos, z(9, 16), z(9, 16))
    ko, _ = L.append(None, None, k.requires_grad_(True), None, pos, z(9, 16), z(9, 16))
    d, = torch.autograd.grad(ko.square().sum(), k, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        d.sum().backward()


def test_decode_in_a_graph():
    """The same bits, and an error instead of a gradient that is not there."""
    banner("latent decode graph")
    g = torch.Generator().manual_seed(2)
    r = lambda *s: torch.randn(*s, generator=g).to(BF16).cuda()
    table, ln = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4), _i32([60, 17])
    for i in range(3):
        x = [r(2, 1, 4, 96), r(4, 128, 128), r(8, 16, 160)]
        with torch.no_grad():
            want = L.decode(*x, table, ln, 0.1)
        x[i].requires_grad_(True)
        with torch.no_grad():
            o = L.decode(*x, table, ln, 0.1)
        assert torch.equal(o, want) and not o.requires_grad
        o = L.decode(*x, table, ln, 0.1)
        assert torch.equal(o, want)
        with pytest.raises(RuntimeError, match="no gradient"):
            o.float().sum().backward()
        x = [t.detach() for t in x]
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward mode"):
            x[i] = forward_ad.make_dual(x[i], torch.ones_like(x[i]))
            L.decode(*x, table, ln, 0.1)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_slots_that_occur_twice_mix_their_own_tokens_only(dtype):
    """A slot given to several tokens: every element of its row is one of theirs, all
    other rows are as they would be."""
    banner(f"latent append repeated slots {dtype}")
    g = torch.Generator().manual_seed(11)
    N, dc, dr = 400, 512, 64
    down, cache = (torch.randn(*s, generator=g).to(dtype) for s in ((N, dc + dr), (30, 16, dc + dr)))
    slots = torch.randperm(480, generator=g)[:N]
    slots[100:300] = slots[50]
    slots[399] = slots[0]
    cos, sin = (t.cuda() for t in _tables(50, dr))
    dev, pos = cache.cuda(), torch.arange(N, dtype=torch.int32, device="cuda") % 50
    k, _ = L.append(dev, down.cuda()[:, :dc], down.cuda()[:, dc:], slots.cuda(), pos, cos, sin)
    rows, got = torch.cat((down[:, :dc], k.cpu()), 1), dev.cpu().view(480, -1)
    want = cache.view(480, -1).clone()
    want[slots] = rows
    for s in slots.unique().tolist():
        mine = (slots == s).nonzero().flatten()
        assert (got[s] == rows[mine]).any(0).all()
        want[s] = got[s]
    assert torch.equal(got, want)
