"""Shared prefixes, gathered weights and eviction on the GPU against the float64 oracle.

Bounds, fixed beforehand.  o: as the absorbed form without a prefix; q_lat and o are
rounded to bf16 (each at most 2^-8 of the value), and p may be: with scores of unit
spread each contributes 0.58 * 2^-8 to a row's 2-norm, together 2^-8, so a row may be
off by four times that and all rows by twice.  float32: 2e-5, by the sums of products.

Gathered weights are float32 in either type.  In bf16 the query enters as two numbers:
what the first leaves out, at most 2^-8 of the value, is rounded to 2^-8 of itself, so a
score of unit spread is off by 0.58 * 2^-16 in the mean, and a weight by as much of
itself.  With the float32 sums' 2e-5: a sequence's weights may be off by
2^-15 + 2e-5 of their 2-norm, a single one by four times that of itself and of their mean.
"""
import pytest
import torch

from _util import banner
from atomic_ops import _lib
from atomic_ops import latent as L
from oracle import latent as ol

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
U = {BF16: 2.0 ** -8, F32: 2e-5}
UW = {BF16: 2.0 ** -15 + 2e-5, F32: 2e-5}
NAN = float("nan")


def _tables(rows, dr):
    a = torch.arange(rows, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(0, dr, 2, dtype=torch.float64) / dr)
    return a.cos().float(), a.sin().float()


def _case(pre, own, n, H, dn, dr, dv, dc, page, dtype, seed):
    """q, w_kv, cache, prefix_table, prefix_lens, page_table, kv_lens on the CPU.  What no sequence
    holds is NaN, and table entries past the needed ones point nowhere."""
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)
    G, B = len(pre), len(own)
    front, per = (max(1, -(-max(x, default=0) // page)) for x in (pre, own))
    pages = G * front + B * per + 2
    ids = torch.randperm(pages, generator=g).to(torch.int32)
    pt, table = ids[:G * front].view(G, front).clone(), ids[G * front:G * front + B * per].view(B, per).clone()
    cache = r(pages, page, dc + dr).to(dtype)
    used = torch.zeros(pages, page, dtype=torch.bool)
    for tab, lens in ((pt, pre), (table, own)):
        for b, ln in enumerate(lens):
            for j in range(ln):
                used[tab[b, j // page], j % page] = True
            tab[b, -(-ln // page):] = -12345 if b % 2 else 1 << 30
    cache[~used] = NAN
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)
    return (r(B, n, H, dn + dr).to(dtype), (r(H, dn + dv, dc) * dc ** -0.5).to(dtype), cache, pt, i32(pre), table,
            i32(own))


def _rows_within(got, want, u):
    got = got.double().cpu()
    assert torch.isfinite(got).all()
    off, size = (got - want).norm(dim=-1), want.norm(dim=-1)
    assert (off[size == 0] == 0).all()
    assert (off <= 4 * u * size).all(), (off / size.clamp(min=1e-30)).max()
    assert off.norm() <= 2 * u * size.norm() + 1e-30


def _weights_within(got, before, add, lens, n, u):
    """Against what stood there and the step's sums; what lies past a length is untouched."""
    want = ol.gathered(before, add, lens, n)
    got = got.double().cpu()
    for b, ln in enumerate(lens):
        assert torch.equal(got[b, ln:], before[b, ln:].double())
        a, x = add[b, :ln], (got - want)[b, :ln].abs()
        if ln:
            # (and the float32 sum with what stood there)
            tol = u * (a + a.mean()) * 4 + 2.0 ** -23 * want[b, :ln].abs()
            assert (x <= tol).all(), (x - tol).max()
            assert x.norm() <= u * a.norm() + 2.0 ** -23 * want[b, :ln].norm()


CASES = [
    # pre, own, n, H, dn, dr, dv, dc, page
    ([1], [1], 1, 1, 128, 64, 128, 512, 64),
    ([130], [0], 1, 6, 128, 64, 128, 512, 64),                    # a prefix by itself
    ([0], [70, 3], 1, 6, 128, 64, 128, 512, 16),                  # no prefix yet
    ([777], [33, 0, 1, 64], 1, 6, 128, 64, 128, 512, 16),
    ([200, 65, 0], [5, 130, 64, 0, 20, 1], 1, 16, 64, 32, 64, 256, 24),
    ([40, 300], [0, 1, 3, 90], 4, 8, 56, 24, 72, 448, 1),         # queries that stand in the prefix
    ([2, 0], [0, 1, 3, 0], 5, 3, 64, 32, 64, 128, 64),            # queries before the first token
    ([513], [31, 32, 33, 7, 0, 100, 64, 65, 1, 12], 1, 30, 128, 32, 96, 128, 64),   # a row tile and a part
    ([1100, 64], [50] * 6, 2, 40, 128, 64, 128, 512, 128),
    ([257], [20] * 33, 1, 4, 8, 8, 8, 8, 256),
    ([90], [17] * 70, 3, 1, 128, 64, 128, 512, 32),               # one head
    ([150], [40, 0], 19, 16, 64, 32, 64, 512, 64),                # more query tokens than a tile of rows
]


# rows enough that a prefix's tokens are bound by matrix instructions (wide latents in bf16,
# tables of 4096 tokens or more, here wider than the prefixes)
MANY = [
    ([256], [0] * 33, 1, 1, 128, 64, 128, 512, 64),                          # 33 rows of one head
    ([300], [0, 40, 2] * 5, 3, 6, 128, 64, 128, 512, 16),                    # queries that stand in the prefix
    ([1, 700, 0, 257], [5, 0, 33, 64] * 3, 1, 20, 56, 24, 72, 448, 24),      # prefixes of one token, none, many
    ([2049], [17 * i % 50 for i in range(9)], 2, 15, 64, 32, 64, 264, 1),    # 270 rows; a token past a split
    ([33, 500], [20] * 8, 4, 40, 128, 32, 96, 320, 128),
    ([256], [3, 0], 19, 16, 64, 32, 64, 512, 256),                           # more queries than own tokens
    ([300], [0, 40, 2] * 5, 3, 6, 64, 32, 64, 256, 16),                      # the same with narrow latents
    ([1, 700, 0, 257], [5, 0, 33, 64] * 3, 1, 20, 56, 24, 72, 200, 24),
    ([33, 500], [20] * 8, 4, 40, 128, 64, 96, 128, 128),
    ([256], [70] * 33, 1, 1, 128, 64, 128, 8, 64),
]


# prefixes and own tokens in one launch and in two: up to some 262144 own tokens, in float32, where
# the two kinds differ in their row tiles, up to 4096
BOTH = [
    ([90], [1024, 3, 700, 0], 1, 6, 64, 32, 64, 64, 128),
    ([90], [1030, 3, 700, 0], 1, 6, 64, 32, 64, 64, 1),
    ([40], [16384] + [7] * 15, 1, 2, 64, 32, 64, 32, 256),
    ([40], [16390] + [7] * 15, 1, 2, 64, 32, 64, 32, 1),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("pre,own,n,H,dn,dr,dv,dc,page,most", [(*c, 0) for c in CASES + BOTH] + [(*c, 4096) for c in MANY])
def test_shared_matches_the_formula(pre, own, n, H, dn, dr, dv, dc, page, most, dtype):
    banner(f"latent shared {pre} {own} n{n} H{H} {dn}/{dr}/{dv}/{dc} page {page} {most} {dtype}")
    q, w, cache, pt, pl, table, ln = _case(pre, own, n, H, dn, dr, dv, dc, page, dtype, seed=H + n + pre[0])
    more = max(0, -(-most // page) - pt.shape[1])
    pt = torch.cat((pt, pt.new_full((len(pre), more), -7)), 1)
    cos, sin = _tables(max(pre) + max(own) + 1, dr)
    scale = (dn + dr) ** -0.5
    d = [t.cuda() for t in (q, w, cache, pt, pl, table, ln)]
    for rope in (None, False, True):
        kw = {} if rope is None else dict(cos=cos.cuda(), sin=sin.cuda(), interleaved=rope)
        o = L.decode_shared(*d, scale, **kw)
        before = torch.rand(len(own), table.shape[1] * page + 3, generator=torch.Generator().manual_seed(1))
        got = before.cuda()
        o2 = L.decode_shared(*d, scale, weights=got, **kw)
        torch.cuda.synchronize()
        want, add = ol.decode_shared(q, w, cache, pt, pl, table, own, scale,
                                     *((None, None) if rope is None else (cos, sin)), bool(rope))
        _rows_within(o, want, U[dtype])
        _rows_within(o2, want, U[dtype])
        _weights_within(got, before, add, own, n, UW[dtype])
    again, twice = before.cuda(), L.decode_shared(*d, scale, **kw)       # the same bits
    assert torch.equal(L.decode_shared(*d, scale, weights=again, **kw), o2) and torch.equal(again, got)
    assert torch.equal(twice, o)


DECODES = [
    # lens, n, H, dn, dr, dv, dc, page
    ([1], 1, 1, 128, 64, 128, 512, 64),
    ([777, 0, 64, 65], 1, 6, 128, 64, 128, 512, 16),
    ([200, 1, 129], 1, 16, 64, 32, 64, 256, 24),
    ([130, 3, 0], 4, 8, 56, 24, 72, 448, 1),               # more queries than tokens
    ([70, 300], 2, 30, 128, 32, 96, 128, 64),
    ([100, 257], 1, 40, 128, 64, 128, 512, 128),
    ([1300] + [31 * i for i in range(20)], 1, 4, 64, 32, 64, 64, 48),
    ([50, 80], 19, 16, 64, 32, 64, 512, 64),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,n,H,dn,dr,dv,dc,page", DECODES)
def test_decode_gathers_the_weights(lens, n, H, dn, dr, dv, dc, page, dtype):
    banner(f"latent decode weights {lens} n{n} H{H} {dn}/{dr}/{dv}/{dc} page {page} {dtype}")
    q, w, cache, _, _, table, ln = _case([], lens, n, H, dn, dr, dv, dc, page, dtype, seed=H + n)
    d = [t.cuda() for t in (q, w, cache, table, ln)]
    scale = (dn + dr) ** -0.5
    want, add = ol.decode_shared(q, w, cache, None, None, table, lens, scale)
    # rows of a wider state, what stands there far larger than a step's share
    wide = 3.0 * torch.rand(len(lens), table.shape[1] * page + 9, generator=torch.Generator().manual_seed(2))
    dev = wide.cuda()
    view, before = dev[:, 2:-1], wide[:, 2:-1]
    o = L.decode(*d, scale, weights=view)
    torch.cuda.synchronize()
    _rows_within(o, want, U[dtype])
    _weights_within(view, before, add, lens, n, UW[dtype])
    assert torch.equal(dev[:, :2].cpu(), wide[:, :2]) and torch.equal(dev[:, -1:].cpu(), wide[:, -1:])
    # once more into zeros: the same sums, bit for bit
    a, b = (torch.zeros_like(before).cuda() for _ in range(2))
    assert torch.equal(L.decode(*d, scale, weights=a), o) and torch.equal(L.decode(*d, scale, weights=b), o)
    assert torch.equal(a, b)
    _weights_within(a, torch.zeros_like(before), add, lens, n, UW[dtype])


@pytest.mark.parametrize("dc,H", [(128, 4), (512, 18), (128, 18)])
@pytest.mark.parametrize("scale", [-0.1, 0.0, 3.0])
def test_other_scales(scale, dc, H):
    """Negative, zero, and large enough that single tokens carry a row and its reference moves often
    (a score of spread s is off by s times what one of unit spread is)."""
    banner(f"latent shared scale {scale} {dc} {H}")
    pre, own = [300, 77], [40, 1, 0, 90]
    q, w, cache, pt, pl, table, ln = _case(pre, own, 2, H, 64, 32, 64, dc, 32, BF16, seed=31)
    if H == 18:
        pt = torch.cat((pt, pt.new_full((2, 120), 1 << 30)), 1)     # room for 4160 tokens
    if scale == 3.0:
        o = L.decode_shared(*(t.cuda() for t in (q, w, cache, pt, pl, table, ln)), scale)
        want, _ = ol.decode_shared(q, w, cache, pt, pl, table, own, scale)
        spread = scale * (64 + 32) ** 0.5      # dn + dr products of unit spread
        assert torch.isfinite(o).all()
        assert (o.double().cpu() - want).norm() <= 2 * U[BF16] * spread * want.norm()
        return
    weights = torch.zeros(4, 96, device="cuda")
    o = L.decode_shared(*(t.cuda() for t in (q, w, cache, pt, pl, table, ln)), scale, weights=weights)
    want, add = ol.decode_shared(q, w, cache, pt, pl, table, own, scale)
    _rows_within(o, want, U[BF16])
    _weights_within(weights, torch.zeros(4, 96), add, own, 2, UW[BF16])


@pytest.mark.parametrize("dc", [256, 512])
def test_many_rows_behind_one_prefix(dc):
    """Twelve row blocks and a prefix of many splits."""
    banner(f"latent shared many rows {dc}")
    pre, own = [2600], [3 + 5 * i % 40 for i in range(48)]
    q, w, cache, pt, pl, table, ln = _case(pre, own, 1, 32, 64, 32, 64, dc, 64, BF16, seed=32)
    pt = torch.cat((pt, pt.new_full((1, 30), -7)), 1)
    o = L.decode_shared(*(t.cuda() for t in (q, w, cache, pt, pl, table, ln)), 0.1)
    want, _ = ol.decode_shared(q, w, cache, pt, pl, table, own, 0.1)
    _rows_within(o, want, U[BF16])


def test_wider_tables_and_lengths_past_them():
    banner("latent shared wide tables")
    pre, own = [64, 40], [32, 20, 7, 1]
    d = [t.cuda() for t in _case(pre, own, 1, 8, 64, 32, 64, 128, 32, BF16, seed=33)]
    q, w, cache, pt, pl, table, ln = d
    want = L.decode_shared(*d, 0.1)
    more = lambda t, k: torch.cat((t, t.new_full((t.shape[0], k), -7)), 1)
    wide = L.decode_shared(q, w, cache, more(pt, 60), pl, more(table, 33), ln, 0.1)
    assert ((wide.float() - want.float()).norm() <= 4 * U[BF16] * want.float().norm()).item()
    far = pl.clone(), ln.clone()
    far[0][0], far[1][0] = 1 << 30, 1 << 30      # the tables' 64 and 32 tokens
    assert torch.equal(L.decode_shared(q, w, cache, pt, far[0], table, far[1], 0.1), want)
    # no own pages at all, no prefix pages at all
    none = table[:, :0]
    a = L.decode_shared(q, w, cache, pt, pl, none, ln * 0, 0.1)
    assert torch.equal(a, L.decode_shared(q, w, cache, pt, pl, none, ln, 0.1))
    b = L.decode_shared(q, w, cache, pt[:, :0], pl, table, ln, 0.1)
    c = L.decode(q, w, cache, table, ln, 0.1)
    assert ((b.float() - c.float()).norm() <= 4 * U[BF16] * c.float().norm()).item()
    assert (L.decode_shared(q, w, cache, pt[:, :0], pl, none, ln, 0.1) == 0).all()


@pytest.mark.parametrize("most", [96, 4096])
def test_weights_of_no_own_pages(most):
    """A prefix by itself where weights are asked for: there are none to gather, and o is that of the call
    whose sequences have pages without tokens."""
    banner(f"latent shared weights of nothing {most}")
    q, w, cache, pt, pl, table, ln = (t.cuda() for t in _case([90], [0] * 5, 1, 8, 64, 32, 64, 512, 32, BF16, seed=39))
    pt = torch.cat((pt, pt.new_full((1, most // 32 - 3), -7)), 1)
    some = torch.ones(5, 32, device="cuda")
    want = L.decode_shared(q, w, cache, pt, pl, table, ln, 0.1, weights=some)
    for wide in (0, 7):
        weights = torch.ones(5, wide, device="cuda")
        o = L.decode_shared(q, w, cache, pt, pl, table[:, :0], ln, 0.1, weights=weights)
        assert ((o.float() - want.float()).norm() <= 4 * U[BF16] * want.float().norm()).item()
        assert (weights == 1).all()
    assert (some == 1).all()


def test_strided_queries_and_another_stream():
    banner("latent shared strides and streams")
    d = [t.cuda() for t in _case([150], [40, 9, 0], 2, 4, 64, 32, 64, 128, 16, BF16, seed=34)]
    q, rest = d[0], d[1:]
    cos, sin = (t.cuda() for t in _tables(200, 32))
    want = L.decode_shared(q, *rest, 0.1, cos=cos, sin=sin)
    wide = torch.full((3, 2, 4 * 96 + 8), NAN, dtype=BF16, device="cuda")
    wide[..., :384] = q.flatten(2)
    assert torch.equal(L.decode_shared(wide[..., :384].unflatten(2, (4, 96)), *rest, 0.1, cos=cos, sin=sin), want)
    odd = torch.empty(q.numel() + 1, dtype=BF16, device="cuda")[1:].view_as(q).copy_(q)     # off a 16-byte address
    assert torch.equal(L.decode_shared(odd, *rest, 0.1, cos=cos, sin=sin), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    late = torch.empty_like(q)
    with torch.cuda.stream(side):
        torch.empty(1 << 27, device="cuda").normal_()      # keeps the stream busy before the input is there
        late.copy_(q)
        got = L.decode_shared(late, *rest, 0.1, cos=cos, sin=sin)
    side.synchronize()
    assert torch.equal(got, want)


def test_calls_that_share_a_workspace_and_a_dirty_one():
    banner("latent shared workspace")
    d = [t.cuda() for t in _case([150, 70], [40, 9, 0, 3], 1, 4, 64, 32, 64, 128, 16, BF16, seed=35)]
    want = L.decode_shared(*d, 0.1)
    w0 = torch.zeros(4, 48, device="cuda")
    o0 = L.decode_shared(*d, 0.1, weights=w0)
    ws = torch.full((1 << 22,), 255, dtype=torch.uint8, device="cuda")     # NaN in every part
    w1 = torch.zeros(4, 48, device="cuda")
    assert torch.equal(L.decode_shared(*d, 0.1, workspace=ws), want)
    assert torch.equal(L.decode_shared(*d, 0.1, weights=w1, workspace=ws), o0) and torch.equal(w0, w1)


def test_cache_larger_than_32_bits():
    """Pages behind 2^31 elements: read as a prefix and as own tokens, and moved."""
    banner("latent shared and evict in a cache of 2^31 elements and more")
    row, page = 576, 64
    pages = (1 << 31) // (page * row) + 40
    cache = torch.empty(pages, page, row, dtype=BF16, device="cuda")
    q, w, small, pt, pl, table, ln = (t.cuda() for t in _case([300], [100, 90], 1, 8, 64, 64, 64, 512, page, BF16, seed=36))
    cache[-small.shape[0]:] = small
    at = pages - small.shape[0]
    pt, table = pt.clamp(0, small.shape[0] - 1), table.clamp(0, small.shape[0] - 1)
    assert torch.equal(L.decode_shared(q, w, cache, pt + at, pl, table + at, ln, 0.1),
                       L.decode_shared(q, w, small, pt, pl, table, ln, 0.1))
    weights = torch.rand(2, 128, generator=torch.Generator().manual_seed(6)).cuda()
    order = torch.full((2, 128), -1, dtype=torch.int32, device="cuda")
    a = L.evict(cache, table + at, ln, weights, order, 60, recent=5)
    b = L.evict(small, table, ln, weights, order, 60, recent=5)
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    x, y = cache[at:], small
    assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))


def test_in_a_graph_of_gradients():
    banner("latent shared gradients")
    d = [t.cuda() for t in _case([70], [20, 3], 1, 4, 64, 32, 64, 128, 16, BF16, seed=37)]
    o = L.decode_shared(d[0].requires_grad_(True), *d[1:], 0.1)
    with pytest.raises(RuntimeError, match="no gradient"):
        o.float().sum().backward()
    weights = torch.zeros(2, 32, device="cuda")
    o = L.decode(d[0], d[1], d[2], d[5], d[6], 0.1, weights=weights)
    assert weights[0, :20].sum() > 0
    with pytest.raises(RuntimeError, match="no gradient"):
        o.float().sum().backward()


def test_nothing_to_do():
    banner("latent shared empty dimensions")
    z = lambda *s, dt=BF16: torch.ones(*s, dtype=dt, device="cuda")
    i = lambda *s: z(*s, dt=torch.int32)
    w, cache = z(2, 128, 64), z(3, 16, 96)
    for B, n in ((0, 1), (2, 0)):
        o = L.decode_shared(z(B, n, 2, 96), w, cache, i(1, 2), i(1), i(B, 2), i(B), 0.1)
        assert o.shape == (B, n, 2, 64)
    assert L.decode_shared(z(0, 1, 2, 96), w, cache, i(0, 2), i(0), i(0, 2), i(0), 0.1).shape == (0, 1, 2, 64)
    weights = z(2, 32, dt=F32)
    L.decode(z(2, 1, 2, 96), w, cache, i(2, 2), i(2) * 0, 0.1, weights=weights)
    L.decode(z(2, 1, 2, 96), w, cache, i(2, 0), i(2) * 0, 0.1, weights=weights)
    assert (weights == 1).all()


def test_refusals():
    banner("latent shared refusals")
    d = [t.cuda() for t in _case([70, 9], [20, 3], 1, 4, 64, 32, 64, 128, 16, BF16, seed=38)]
    q, w, cache, pt, pl, table, ln = d
    for a in ((pt[:1].repeat(3, 1), pl[:1].repeat(3)), (pt[:0], pl[:0])):
        with pytest.raises(ValueError, match="divide"):
            L.decode_shared(q, w, cache, *a, table, ln, 0.1)
    for a in ((pt[0], pl), (pt, pl[:1]), (pt.long(), pl), (pt, pl.long()), (pt.cpu(), pl), (pt, pl[None])):
        with pytest.raises(ValueError, match="prefix"):
            L.decode_shared(q, w, cache, *a, table, ln, 0.1)
    f = lambda *s, dt=F32: torch.zeros(*s, dtype=dt, device="cuda")
    for bad in (f(2, 31), f(3, 32), f(2, 32, dt=BF16), f(2, 32).cpu(), f(32), f(2, 32).requires_grad_(True), f(32, 2).t(),
                f(1, 32).expand(2, 32)):
        with pytest.raises(ValueError, match="weights"):
            L.decode(q, w, cache, table, ln, 0.1, weights=bad)
        with pytest.raises(ValueError, match="weights"):
            L.decode_shared(*d, 0.1, weights=bad)
    with pytest.raises(_lib.AtomicError, match="unsupported shape"):
        L.decode_shared(f(2, 1, 4, 176, dt=BF16), f(4, 208, 128, dt=BF16), cache, pt, pl, table, ln, 0.1)     # dn 144
    with pytest.raises(ValueError, match="workspace"):
        L.decode_shared(*d, 0.1, workspace=torch.zeros(1 << 22, dtype=torch.uint8))
