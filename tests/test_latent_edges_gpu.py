"""Latent attention on the GPU at its edges."""
import pytest
import torch
from torch.autograd import forward_ad

from _util import banner
from atomic_ops import latent as L

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
