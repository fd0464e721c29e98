"""Latent attention on the GPU against the float64 oracle.

Bounds, fixed beforehand.  A bf16 rounding is off by at most U16 = 2^-8 of the
value.  In the expanded form p and o are rounded once each, so o is within
U16 (|o| + sum p |v|); a gradient is within U16 of itself plus U16 times the
sum of its terms' sizes, where ds is rounded once and its delta comes from a
rounded o (1.5 covers p (|dp| + 3 sum p |v| |do|) by the oracle's size).  float32:
the same sums with U32 = 2e-5, a score of 192 products being off by up to
192 * 0.64 * 0.07 * sqrt(192) * 2^-24 = 7e-6 and a sum of 4096 terms by
64 * 2^-24 = 4e-6 of its size.  The absorbed form rounds q_lat, p and o; with
scores of unit spread each contributes 0.58 * 2^-8 to a row's 2-norm, together
2^-8: a row may be off by four times that, all rows by twice.
"""
import importlib.util
import os

import pytest
import torch

from _util import banner
from atomic_ops import _lib
from atomic_ops import latent as L
from oracle import latent as ol

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
U = {BF16: 2.0 ** -8, F32: 2e-5}
NAN, INF = float("nan"), float("inf")


def _inputs(B, T, S, H, dn, dr, dv, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    return r(B, T, H, dn + dr), r(B, S, H, dn + dv), r(B, S, dr), r(B, T, H, dv)


def _spoil(ts, lens):
    """The rows past each length as NaN and infinities."""
    for t, ln in zip(ts, lens):
        if ln is not None:
            for b, n in enumerate(ln):
                t[b, n:] = NAN
                t[b, n + 1:] = INF


def _within(got, want, size, u, what):
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    over = (got - want).abs() - u * (want.abs() + size) * 1.01 - 1e-30
    assert over.max() <= 0, f"{what}: {over.max():.3e} over its bound, {(over > 0).sum()} places"


def _i32(v):
    return None if v is None else torch.tensor(v, dtype=torch.int32, device="cuda")


SHAPES = [
    # B, T, S, H, dn, dr, dv, causal, q_lens, kv_lens
    (1, 1, 1, 1, 128, 64, 128, True, None, None),         # one token
    (2, 1, 77, 3, 128, 64, 128, True, None, None),        # one query over a prefix
    (1, 131, 131, 2, 128, 64, 128, True, None, None),     # a block and three rows
    (2, 257, 257, 1, 64, 32, 64, False, None, None),
    (1, 33, 200, 2, 56, 24, 72, True, None, None),        # widths that are padded
    (1, 200, 70, 2, 128, 64, 128, True, None, None),      # the first 130 queries see nothing
    (3, 140, 140, 2, 128, 64, 128, True, [140, 0, 37], [140, 0, 37]),
    (4, 65, 300, 1, 96, 32, 64, True, [65, 64, 1, 33], [300, 0, 128, 20]),
    (2, 40, 129, 5, 8, 8, 8, False, [40, 3], [128, 129]),
    (1, 300, 500, 6, 128, 32, 96, True, [256], [384]),
    (1, 70, 2100, 1, 128, 64, 128, True, None, [2049]),      # the keys divided over eight workgroups
    (1, 2100, 70, 1, 64, 32, 64, False, [2049], None),       # and the queries
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,T,S,H,dn,dr,dv,causal,ql,kl", SHAPES)
def test_expanded_matches_the_formulas(B, T, S, H, dn, dr, dv, causal, ql, kl, dtype):
    banner(f"latent expanded B{B} T{T} S{S} H{H} {dn}/{dr}/{dv} causal={causal} {ql} {kl} {dtype}")
    q, kv, k_pe, do = _inputs(B, T, S, H, dn, dr, dv, dtype, seed=T + S)
    _spoil((q, do, kv, k_pe), (ql, ql, kl, kl))
    scale = (dn + dr) ** -0.5
    qd, kvd, kd, dod = (t.cuda() for t in (q, kv, k_pe, do))
    o, lse = L.forward(qd, kvd, kd, scale, causal=causal, q_lens=_i32(ql), kv_lens=_i32(kl))
    grads = L.backward(qd, kvd, kd, o, lse, dod, scale, causal=causal, q_lens=_i32(ql), kv_lens=_i32(kl))
    torch.cuda.synchronize()
    o_ref, lse_ref, mag = ol.expanded(q, kv, k_pe, scale, causal, ql, kl)
    _within(o, o_ref, mag, U[dtype], "o")
    empty = lse_ref == -INF
    got = lse.double().cpu()
    assert torch.equal(got == -INF, empty)
    assert ((got - lse_ref).abs()[~empty] <= 2e-5 * (1 + lse_ref.abs()[~empty])).all()
    assert (o.cpu()[empty.transpose(1, 2)] == 0).all()
    want, size = ol.expanded_grads(q, kv, k_pe, do, scale, causal, ql, kl)
    for n, a, b, s in zip(("dq", "dkv", "dk_pe"), grads, want, size):
        assert a.dtype == dtype
        _within(a, b, 1.5 * s, U[dtype], n)
    assert (grads[0].cpu()[empty.transpose(1, 2)] == 0).all()


def _against_the_oracle(shape, dtype, seed, scale=None):
    B, T, S, H, dn, dr, dv, causal, ql, kl = shape
    q, kv, k_pe, do = _inputs(B, T, S, H, dn, dr, dv, dtype, seed=seed)
    _spoil((q, do, kv, k_pe), (ql, ql, kl, kl))
    scale = (dn + dr) ** -0.5 if scale is None else scale
    d = [t.cuda() for t in (q, kv, k_pe)]
    kw = dict(causal=causal, q_lens=_i32(ql), kv_lens=_i32(kl))
    o, lse = L.forward(*d, scale, **kw)
    grads = L.backward(*d, o, lse, do.cuda(), scale, **kw)
    torch.cuda.synchronize()
    o_ref, lse_ref, mag = ol.expanded(q, kv, k_pe, scale, causal, ql, kl)
    _within(o, o_ref, mag, U[dtype], "o")
    seen = lse_ref != -INF
    assert torch.equal(lse.cpu() == -INF, ~seen)
    assert ((lse.double().cpu() - lse_ref).abs()[seen] <= 2e-5 * (1 + lse_ref.abs()[seen])).all()
    want, size = ol.expanded_grads(q, kv, k_pe, do, scale, causal, ql, kl)
    for n, a, b, z in zip(("dq", "dkv", "dk_pe"), grads, want, size):
        _within(a, b, 1.5 * z, U[dtype], n)
    _, _, rest = L.forward(*d, scale, save=True, **kw)
    if dtype == BF16:
        _within(o.double() + rest.double(), o_ref, mag, 2.0 ** -8, "o and what its rounding left out")
    for n, a, b, z in zip(("dq", "dkv", "dk_pe"), L.backward(*d, o, lse, do.cuda(), scale, rest=rest, **kw), want, size):
        _within(a, b, 1.5 * z, U[dtype], n)


@pytest.mark.parametrize("causal", [True, False])
def test_many_row_blocks(causal):
    """More row blocks than the card holds at once."""
    banner(f"latent expanded, many row blocks causal={causal}")
    _against_the_oracle((8, 300, 333, 17, 128, 64, 128, causal, [300, 0, 37, 256, 257, 64, 1, 129],
                         [333, 12, 0, 256, 300, 65, 64, 100]), BF16, seed=21)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("scale", [-0.1, 0.0])
def test_negative_and_zero_scale(scale, dtype):
    """With a scale of zero every visible key weighs the same, and q, k have no gradient."""
    banner(f"latent expanded scale {scale} {dtype}")
    _against_the_oracle((2, 90, 150, 2, 64, 32, 64, True, [90, 20], [150, 10]), dtype, seed=22, scale=scale)


def test_more_score_gradients_than_are_kept():
    """Two bytes a pair of the padded lengths pass 4 GB: dq computes its scores again."""
    banner("latent backward past the kept score gradients")
    T, ql, kl = 46400, 200, 230
    q, kv, k_pe, do = _inputs(1, ql, kl, 1, 128, 64, 128, BF16, seed=23)
    pad = lambda t, n: torch.cat((t, t.new_full((1, T - n, *t.shape[2:]), NAN)), 1).cuda()
    d = [pad(q, ql), pad(kv, kl), pad(k_pe, kl)]
    for causal in (True, False):
        kw = dict(causal=causal, q_lens=_i32([ql]), kv_lens=_i32([kl]))
        o, lse = L.forward(*d, 0.07, **kw)
        grads = L.backward(*d, o, lse, pad(do, ql), 0.07, **kw)
        torch.cuda.synchronize()
        want, size = ol.expanded_grads(q, kv, k_pe, do, 0.07, causal)
        for n, x, a, b, z in zip(("dq", "dkv", "dk_pe"), (ql, kl, kl), grads, want, size):
            _within(a[:, :x], b, 1.5 * z, U[BF16], n)
            assert (a[:, x:] == 0).all()


def test_scores_of_one_key_have_no_gradient():
    """A query that sees one key: do . v less do . o is zero.  With what o's
    rounding left out, itself rounded, o is known to 2^-16; the two sums of 128
    products differ by 128 * 2^-24 of their sizes, the difference is rounded (in a
    ratio) and so is its product: within 2^-15 of the terms' sizes."""
    banner("latent expanded one key")
    for T, S, causal, ql, kl in ((3, 1, False, None, None), (64, 64, True, [1], [1])):
        q, kv, k_pe, do = _inputs(1, T, S, 2, 128, 64, 128, BF16, seed=26)
        x = [t.cuda().requires_grad_(True) for t in (q, kv, k_pe)]
        o = L.attention(*x, 0.07, causal=causal, q_lens=_i32(ql), kv_lens=_i32(kl))
        grads = torch.autograd.grad(o, x, do.cuda())
        want, size = ol.expanded_grads(q, kv, k_pe, do, 0.07, causal, ql, kl)
        for i in (0, 2):
            assert (grads[i].double().cpu() - want[i]).abs().sub(2.0 ** -15 * size[i]).max() <= 0
        assert torch.equal(L.forward(*(t.detach() for t in x), 0.07, causal=causal, q_lens=_i32(ql),
                                     kv_lens=_i32(kl))[0], o.detach())


def test_lengths_belong_to_the_graph():
    """Lengths changed after the forward are an error in the backward, as any saved tensor's change is;
    a second derivative is refused."""
    banner("latent expanded saved lengths")
    q, kv, k_pe, _ = (t.cuda() for t in _inputs(1, 8, 8, 1, 64, 32, 64, BF16, seed=24))
    ln = _i32([8])
    o = L.attention(q.requires_grad_(True), kv, k_pe, 0.1, kv_lens=ln)
    ln.fill_(3)
    with pytest.raises(RuntimeError, match="modified"):
        o.float().sum().backward()
    o = L.attention(q, kv, k_pe, 0.1)
    g, = torch.autograd.grad(o.float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()


def test_gradient_follows_differences():
    """float32: the loss along a random direction of each input.  The loss sums
    T H dv = 8e3 products whose rounding (1e-6 of their root sum of squares) is
    divided by the step's 2e-2: 1e-6 * 90 / 2e-2 = 5e-3; the third derivative
    adds a step squared times the slope's scale (about 30): 3e-3 * 30."""
    banner("latent expanded differences")
    q, kv, k_pe, do = (t.cuda() for t in _inputs(1, 50, 60, 2, 64, 32, 64, F32, seed=5))
    scale = 96 ** -0.5
    f = lambda *a: (L.forward(*a, scale)[0].double() * do.double()).sum().item()
    o, lse = L.forward(q, kv, k_pe, scale)
    grads = L.backward(q, kv, k_pe, o, lse, do, scale)
    g = torch.Generator().manual_seed(9)
    for i, d in enumerate(grads):
        u = torch.randn(d.shape, generator=g).cuda()
        hi, lo = [q, kv, k_pe], [q, kv, k_pe]
        hi[i], lo[i] = hi[i] + 1e-2 * u, lo[i] - 1e-2 * u
        slope = (d.double() * u.double()).sum().item()
        assert abs((f(*hi) - f(*lo)) / 2e-2 - slope) < 0.1 + 1e-3 * abs(slope)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strided_inputs_are_read_in_place(dtype):
    """Transposed heads and slices of wider rows give the dense tensors' bits."""
    banner(f"latent expanded strides {dtype}")
    B, T, S, H, dn, dr, dv = 2, 70, 90, 3, 64, 32, 64
    q, kv, k_pe, do = (t.cuda() for t in _inputs(B, T, S, H, dn, dr, dv, dtype, seed=2))
    qt = q.transpose(1, 2).contiguous().transpose(1, 2)
    wide = torch.full((B, S, 16 + H * (dn + dv)), NAN, dtype=dtype, device="cuda")
    wide[..., 16:] = kv.flatten(2)
    kvw = wide[..., 16:].unflatten(2, (H, dn + dv))
    down = torch.full((B, S, 128 + dr), NAN, dtype=dtype, device="cuda")
    down[..., 128:] = k_pe
    gt = do.permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    for a in (qt, kvw, down[..., 128:], gt):
        assert L._strided(a, a.dim() - 1)[0] is a
    odd = torch.empty(k_pe.numel() + 3, dtype=dtype, device="cuda")[3:].view(k_pe.shape)   # off 16 bytes: copied
    odd.copy_(k_pe)
    for kp in (down[..., 128:], odd):
        o, lse = L.forward(qt, kvw, kp, 0.1)
        o2, lse2 = L.forward(q, kv, k_pe, 0.1)
        assert torch.equal(o, o2) and torch.equal(lse, lse2)
        for a, b in zip(L.backward(qt, kvw, kp, o, lse, gt, 0.1), L.backward(q, kv, k_pe, o, lse, do, 0.1)):
            assert torch.equal(a, b)


def test_autograd_broadcast_gradient_and_repeats():
    """A gradient that is one number broadcast (all strides zero); the same call twice gives the same bits."""
    banner("latent expanded autograd")
    q, kv, k_pe, _ = (t.cuda() for t in _inputs(2, 150, 150, 4, 128, 64, 128, BF16, seed=8))
    x = [t.requires_grad_(True) for t in (q, kv, k_pe)]
    runs = []
    for _ in range(2):
        o = L.attention(*x, 0.07)
        runs.append((o.detach(), *torch.autograd.grad(o.sum(), x)))
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    ones = torch.ones_like(runs[0][0])
    with torch.no_grad():
        o, lse, rest = L.forward(*x, 0.07, save=True)
        for a, b in zip(L.backward(*x, o, lse, ones, 0.07, rest=rest), runs[0][1:]):
            assert torch.equal(a, b)


def test_scores_far_apart():
    """Scores of thousands: the softmax picks one key, and nothing overflows."""
    banner("latent expanded large scores")
    q, kv, k_pe, do = _inputs(1, 64, 300, 2, 64, 32, 64, F32, seed=4)
    q = q * 300
    o, lse = L.forward(q.cuda(), kv.cuda(), k_pe.cuda(), 1.0)
    o_ref, lse_ref, mag = ol.expanded(q, kv, k_pe, 1.0)
    # a score of 1e4 is off by 1e4 * 2^-24 * sqrt(96) = 6e-3 at most
    assert (lse.double().cpu() - lse_ref).abs().max() < 2e-2
    assert ((o.double().cpu() - o_ref).abs() <= 2e-2 * mag + 2e-2 * o_ref.abs()).all()
    for g in L.backward(q.cuda(), kv.cuda(), k_pe.cuda(), o, lse, do.cuda(), 1.0):
        assert torch.isfinite(g).all()


def test_rows_further_apart_than_32_bits():
    banner("latent expanded distant rows")
    B, T, H, dn, dr, dv = 2, 20, 1, 64, 32, 64
    q, kv, k_pe, do = (t.cuda() for t in _inputs(B, T, T, H, dn, dr, dv, BF16, seed=6))
    far = torch.empty((1 << 31) + 8192, dtype=BF16, device="cuda")
    kf = far.as_strided((B, T, H, dn + dv), (1 << 31, 128, 128, 1))
    kf.copy_(kv)
    o, lse = L.forward(q, kf, k_pe, 0.1)
    o2, lse2 = L.forward(q, kv, k_pe, 0.1)
    assert torch.equal(o, o2) and torch.equal(lse, lse2)
    for a, b in zip(L.backward(q, kf, k_pe, o, lse, do, 0.1), L.backward(q, kv, k_pe, o2, lse2, do, 0.1)):
        assert torch.equal(a, b)


def test_tokens_further_apart_than_a_tile_reaches():
    """Tokens 33 MB apart (the tokens of a transposed tensor) are copied, in the library's own call refused."""
    banner("latent expanded token strides past the library's")
    B, T, H, dn, dr, dv = 1, 3, 2, 64, 32, 64
    q, kv, k_pe, _ = (t.cuda() for t in _inputs(B, T, T, H, dn, dr, dv, BF16, seed=16))
    ld = (1 << 24) + 8 * H * (dn + dv)
    far = torch.empty(2 * ld + H * (dn + dv), dtype=BF16, device="cuda").as_strided(kv.shape, (8, ld, dn + dv, 1))
    far.copy_(kv)
    for a, b in zip(L.forward(q, far, k_pe, 0.1), L.forward(q, kv, k_pe, 0.1)):
        assert torch.equal(a, b)
    args, _ = L.make_args(q, kv, k_pe, 0.1, True)
    args.kv_stride[1] = ld
    assert _lib.load().atomic_latent_fwd_workspace_size(args) == 0


def _tables(rows, dr):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, dr, 2, dtype=torch.float64) / dr)
    return a.cos().float(), a.sin().float()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N,H,dn,dr,dc,page,inter", [(1, 1, 128, 64, 512, 64, False), (37, 3, 56, 24, 448, 24, True),
                                                     (300, 6, 64, 32, 128, 1, False), (65, 2, 8, 8, 8, 16, True)])
def test_append_writes_its_rows_and_no_others(N, H, dn, dr, dc, page, inter, dtype):
    banner(f"latent append N{N} H{H} {dn}/{dr}/{dc} page {page} interleaved={inter} {dtype}")
    g = torch.Generator().manual_seed(N)
    r = lambda *s: torch.randn(*s, generator=g).to(dtype)
    pages = -(-N // page) + 2
    down, q, cache = r(N, dc + dr), r(N, H, dn + dr), r(pages, page, dc + dr)
    slots = torch.randperm(pages * page, generator=g)[:N]
    slots[1::5], slots[2::7] = -1, pages * page
    pos = torch.randint(0, 50, (N,), generator=g, dtype=torch.int32)
    cos, sin = _tables(50, dr)
    dev = cache.cuda()
    k, qr = L.append(dev, down.cuda()[:, :dc], down.cuda()[:, dc:], slots.cuda(), pos.cuda(), cos.cuda(), sin.cuda(),
                     q=q.cuda(), interleaved=inter)
    torch.cuda.synchronize()
    want = ol.rotate(down[:, dc:], pos, cos, sin, inter)
    # two fp32 products and a sum, rounded once more in bf16
    tol = lambda x: (2.0 ** -8 if dtype == BF16 else 0.0) * x.abs() + 3 * 2.0 ** -23 * 10
    assert ((k.double().cpu() - want).abs() <= tol(want)).all()
    keep = (slots >= 0) & (slots < pages * page)
    rows = cache.view(-1, dc + dr).clone()
    rows[slots[keep]] = torch.cat((down[keep, :dc], k.cpu()[keep]), 1)
    assert torch.equal(dev.cpu().view(-1, dc + dr), rows)
    want = ol.rotate(q[..., dn:], pos, cos, sin, inter)
    assert torch.equal(qr.cpu()[..., :dn], q[..., :dn])
    assert ((qr.double().cpu()[..., dn:] - want).abs() <= tol(want)).all()
    # by itself the rotation gives the same bits; positions past the tables take the last row
    k2, none = L.append(None, None, down.cuda()[:, dc:], None, pos.cuda(), cos.cuda(), sin.cuda(), interleaved=inter)
    assert none is None and torch.equal(k2, k)
    far = L.append(None, None, down.cuda()[:, dc:], None, pos.cuda() * 0 + 99, cos.cuda(), sin.cuda(),
                   interleaved=inter)[0]
    end = L.append(None, None, down.cuda()[:, dc:], None, pos.cuda() * 0 + 49, cos.cuda(), sin.cuda(),
                   interleaved=inter)[0]
    assert torch.equal(far, end)


def _paged(B, H, n, lens, dn, dr, dv, dc, page, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    per = max(1, -(-max(lens) // page))
    pages = B * per + 2
    table = torch.randperm(pages, generator=g)[:B * per].view(B, per).to(torch.int32)
    cache = r(pages, page, dc + dr).to(dtype)
    # whatever no sequence holds is NaN, table entries past a sequence's pages point nowhere
    used = torch.zeros(pages, page, dtype=torch.bool)
    for b, ln in enumerate(lens):
        for j in range(ln):
            used[table[b, j // page], j % page] = True
        table[b, -(-ln // page):] = -12345 if b % 2 else 1 << 30
    cache[~used] = NAN
    return (r(B, n, H, dn + dr).to(dtype), (r(H, dn + dv, dc) * dc ** -0.5).to(dtype), cache, table,
            torch.tensor(lens, dtype=torch.int32))


def _rows_within(got, want, u):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    off, size = (got - want).norm(dim=-1), want.norm(dim=-1)
    assert (off[size == 0] == 0).all()
    assert (off <= 4 * u * size).all(), (off / size.clamp(min=1e-30)).max()
    assert off.norm() <= 2 * u * size.norm() + 1e-30


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H,n,lens,dn,dr,dv,dc,page", [
    (1, 1, [1], 128, 64, 128, 512, 64),
    (6, 1, [777, 0, 64, 65], 128, 64, 128, 512, 16),
    (16, 1, [200, 1, 129], 64, 32, 64, 256, 24),       # pages that end inside a tile
    (8, 4, [130, 3, 0], 56, 24, 72, 448, 1),           # more queries than tokens
    (30, 2, [70, 300], 128, 32, 96, 128, 64),
    (40, 1, [100, 257], 128, 64, 128, 512, 128),
    (64, 2, [190], 8, 8, 8, 8, 256),
    (16, 19, [50, 80], 64, 32, 64, 512, 64),           # more query tokens than a tile of rows
])
def test_decode_matches_the_expanded_formula(H, n, lens, dn, dr, dv, dc, page, dtype):
    banner(f"latent decode H{H} n{n} lens {lens} {dn}/{dr}/{dv}/{dc} page {page} {dtype}")
    B = len(lens)
    q, w, cache, table, ln = _paged(B, H, n, lens, dn, dr, dv, dc, page, dtype, seed=H + n)
    cos, sin = _tables(max(lens) + 1, dr)
    scale = (dn + dr) ** -0.5
    d = [t.cuda() for t in (q, w, cache, table, ln)]
    for rope in (None, False, True):
        kw = {} if rope is None else dict(cos=cos.cuda(), sin=sin.cuda(), interleaved=rope)
        o = L.decode(*d, scale, **kw)
        torch.cuda.synchronize()
        want = ol.decode(q, w, cache, table, lens, scale, *((None, None) if rope is None else (cos, sin)), bool(rope))
        _rows_within(o, want, 2.0 ** -8 if dtype == BF16 else U[F32])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_decode_of_many_sequences(dtype):
    """Splits of many tiles, one of the sequences far longer than the others."""
    banner(f"latent decode many sequences {dtype}")
    lens = [9000] + [137 * i % 2000 for i in range(63)]
    q, w, cache, table, ln = _paged(64, 4, 1, lens, 64, 32, 64, 64, 48, dtype, seed=25)
    for scale in (0.1, -0.1, 0.0):
        o = L.decode(*(t.cuda() for t in (q, w, cache, table, ln)), scale)
        torch.cuda.synchronize()
        _rows_within(o, ol.decode(q, w, cache, table, lens, scale), 2.0 ** -8 if dtype == BF16 else U[F32])


def test_decode_reads_strided_queries_and_lengths_past_the_table():
    banner("latent decode strides")
    q, w, cache, table, ln = (t.cuda() for t in _paged(2, 4, 2, [128, 96], 64, 32, 64, 128, 32, BF16, seed=1))
    wide = torch.full((2, 2, 4 * 96 + 8), NAN, dtype=BF16, device="cuda")
    wide[..., :384] = q.flatten(2)
    o = L.decode(q, w, cache, table, ln, 0.1)
    assert torch.equal(o, L.decode(wide[..., :384].unflatten(2, (4, 96)), w, cache, table, ln, 0.1))
    more = ln.clone()
    more[0] = 1 << 30        # taken as the table's 128 tokens
    assert torch.equal(o, L.decode(q, w, cache, table, more, 0.1))


def test_cache_larger_than_32_bits():
    banner("latent decode and append in a cache of 2^31 elements and more")
    dc, dr, page = 512, 64, 64
    pages = (1 << 31) // (page * (dc + dr)) + 40
    cache = torch.empty(pages, page, dc + dr, dtype=BF16, device="cuda")
    small = torch.randn(4, page, dc + dr, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    cache[-4:] = small
    q, w, _, _, _ = (t.cuda() for t in _paged(1, 8, 1, [200], 64, dr, 64, dc, page, BF16, seed=2))
    ln = torch.tensor([200], dtype=torch.int32, device="cuda")
    at = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    assert torch.equal(L.decode(q, w, cache, at + (pages - 4), ln, 0.1), L.decode(q, w, small, at, ln, 0.1))
    cos, sin = (t.cuda() for t in _tables(8, dr))
    row = torch.randn(1, dc + dr, generator=torch.Generator().manual_seed(3)).to(BF16).cuda()
    k, _ = L.append(cache, row[:, :dc], row[:, dc:], torch.tensor([pages * page - 1], device="cuda"),
                    torch.tensor([3], dtype=torch.int32, device="cuda"), cos, sin)
    assert torch.equal(cache[-1, -1], torch.cat((row[0, :dc], k[0])))


def test_other_streams_and_graph_replays():
    """The calls follow the current stream, and a captured decode step replays
    with new cache contents, eager work in between."""
    banner("latent streams and graphs")
    q, w, cache, table, ln = (t.cuda() for t in _paged(3, 8, 1, [500, 77, 130], 64, 32, 64, 256, 16, BF16, seed=3))
    cos, sin = (t.cuda() for t in _tables(512, 32))
    want = L.decode(q, w, cache, table, ln, 0.1, cos=cos, sin=sin)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    late = torch.empty_like(q)
    with torch.cuda.stream(side):
        torch.empty(1 << 27, device="cuda").normal_()      # keeps the stream busy before the input is there
        late.copy_(q)
        got = L.decode(late, w, cache, table, ln, 0.1, cos=cos, sin=sin)
    side.synchronize()
    assert torch.equal(got, want)
    slots = (table[:, :1].long() * 16).flatten()
    new = torch.randn(3, 288, generator=torch.Generator().manual_seed(4)).to(BF16).cuda()
    pos = torch.zeros(3, dtype=torch.int32, device="cuda")

    def step():
        L.append(cache, new[:, :256], new[:, 256:], slots, pos, cos, sin)
        return L.decode(q, w, cache, table, ln, 0.1, cos=cos, sin=sin)

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for k in range(3):
        new.copy_(torch.randn(3, 288, generator=torch.Generator().manual_seed(10 + k)))
        graph.replay()
        torch.cuda.synchronize()
        replayed = out.clone()
        assert torch.equal(replayed, step())


def test_the_example_layer_agrees_with_itself():
    """examples/latent_layer.py: training steps, a prompt and single tokens of one layer."""
    banner("latent example layer")
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "latent_layer.py")
    spec = importlib.util.spec_from_file_location("latent_layer", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    example.main(B=2, T=80, prompt=65, page=16, steps=2)


def test_nothing_to_do():
    """Dimensions of zero: no queries, no keys, no tokens to append, no pages."""
    banner("latent empty dimensions")
    z = lambda *s, dt=BF16: torch.ones(*s, dtype=dt, device="cuda")
    for B, T, S in ((0, 3, 3), (2, 0, 3), (2, 3, 0)):
        x = [t.requires_grad_(True) for t in (z(B, T, 2, 96), z(B, S, 2, 128), z(B, S, 32))]
        o = L.attention(*x, 0.1)
        assert o.shape == (B, T, 2, 64) and (o == 0).all()
        assert (L.forward(*(t.detach() for t in x), 0.1)[1] == -INF).all()
        for t, g in zip(x, torch.autograd.grad(o.float().sum(), x)):
            assert g.shape == t.shape and (g == 0).all()
    cache, w, cs = z(3, 16, 96), z(2, 128, 64), z(9, 16, dt=F32)
    before = cache.clone()
    k, q = L.append(cache, z(0, 64), z(0, 32), z(0, dt=torch.int64), z(0, dt=torch.int32), cs, cs, q=z(0, 2, 96))
    assert k.shape == (0, 32) and q.shape == (0, 2, 96) and torch.equal(cache, before)
    assert L.decode(z(0, 1, 2, 96), w, cache, z(0, 2, dt=torch.int32), z(0, dt=torch.int32), 0.1).shape == (0, 1, 2, 64)
    none = L.decode(z(2, 1, 2, 96), w, cache, z(2, 0, dt=torch.int32), z(2, dt=torch.int32), 0.1)
    assert none.shape == (2, 1, 2, 64) and (none == 0).all()


def test_refusals():
    banner("latent refusals")
    z = lambda *s, dt=BF16: torch.zeros(*s, dtype=dt, device="cuda")
    q, kv, k_pe = z(1, 4, 2, 96), z(1, 4, 2, 128), z(1, 4, 32)
    with pytest.raises(TypeError, match="dtype"):
        L.forward(q, kv.float(), k_pe, 1.0)
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        L.forward(q.half(), kv.half(), k_pe.half(), 1.0)
    for a in ((q, kv[:, :3], k_pe), (q, kv, z(1, 4, 96)), (q[0], kv, k_pe), (q, z(1, 4, 2, 64), k_pe)):
        with pytest.raises(ValueError):
            L.forward(*a, 1.0)
    with pytest.raises(ValueError, match="kv_lens"):
        L.forward(q, kv, k_pe, 1.0, kv_lens=torch.zeros(1, dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError, match="pieces"):
        L.forward(z(1, 4, 2, 95), z(1, 4, 2, 127), k_pe, 1.0)
    with pytest.raises(_lib.AtomicError, match="SHAPE"):
        L.forward(z(1, 4, 2, 176), z(1, 4, 2, 208), k_pe, 1.0)      # dn 144
    o, lse = L.forward(q, kv, k_pe, 1.0)
    with pytest.raises(ValueError, match="dout"):
        L.backward(q, kv, k_pe, o, lse, o[:, :3], 1.0)
    for ws in (torch.zeros(1 << 20, dtype=torch.uint8), z(1 << 20), z(1 << 20, dt=torch.uint8)[::2]):
        with pytest.raises(ValueError, match="workspace"):
            L.forward(q, kv, k_pe, 1.0, workspace=ws)
        with pytest.raises(ValueError, match="workspace"):
            L.backward(q, kv, k_pe, o, lse, o, 1.0, workspace=ws)
    args, _ = L.make_args(q, kv, k_pe, 1.0, True, o)
    lib, p = _lib.load(), lambda t: t.data_ptr()
    small = z(64, dt=torch.uint8)
    for call in (lambda ws, n: lib.atomic_latent_bwd(args, p(q), p(kv), p(k_pe), None, None, p(o), p(lse), None, p(o), p(q),
                                                     p(kv), p(k_pe), ws, n, None),):
        for ws, n in ((None, 1 << 20), (p(small), 64)):
            with pytest.raises(_lib.AtomicError, match="WORKSPACE"):
                _lib.check(call(ws, n), "atomic_latent_bwd")
    w, cache, table, ln = z(2, 128, 64), z(3, 16, 96), z(1, 2, dt=torch.int32), z(1, dt=torch.int32)
    qd = z(1, 1, 2, 96)
    assert (L.decode(qd, w, cache, table, ln, 1.0) == 0).all()
    cs = z(9, 16, dt=F32)
    for kw in (dict(cos=cs), dict(cos=cs[:, :8], sin=cs[:, :8]), dict(cos=cs.double(), sin=cs.double())):
        with pytest.raises(ValueError, match="cos and sin"):
            L.decode(qd, w, cache, table, ln, 1.0, **kw)
    with pytest.raises(ValueError, match="dense"):
        L.decode(qd, w, z(16, 3, 96).transpose(0, 1), table, ln, 1.0)
    with pytest.raises(ValueError, match="page_table"):
        L.decode(qd, w, cache, table.long(), ln, 1.0)
    with pytest.raises(_lib.AtomicError, match="unsupported shape"):
        L.decode(z(1, 1, 2, 96), z(2, 128, 528), z(3, 16, 560), table, ln, 1.0)      # dc 528
    x, pos = z(5, 96), z(5, dt=torch.int32)
    with pytest.raises(ValueError, match="slot"):
        L.append(cache, x[:, :64], x[:, 64:], None, pos, cs, cs)
    with pytest.raises(ValueError, match="slots"):
        L.append(cache, x[:, :64], x[:, 64:], pos, pos, cs, cs)
    with pytest.raises(ValueError, match="dense"):
        L.append(z(3, 16, 104), x[:, :64], x[:, 64:], pos.long(), pos, cs, cs)
