"""Eviction from the latent cache on the GPU against the oracle (everything is exact), and
the serving loop that it belongs to: append, decode behind a shared prefix, evict."""
import pytest
import torch

from _util import banner
from atomic_ops import _lib
from atomic_ops import latent as L
from oracle import latent as ol
from test_latent_shared_gpu import BF16, F32, U, UW, _rows_within, _tables, _weights_within

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def _state(lens, page, row, dtype, seed, settled=0, width=3, per=None):
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    per = max(1, -(-max(lens) // page)) if per is None else per
    pages = B * per + 2
    cache = torch.randn(pages, page, row, generator=g).to(dtype)
    table = torch.randperm(pages, generator=g)[:B * per].view(B, per).to(torch.int32)
    W = per * page + width
    weights = torch.randn(B, W, generator=g).exp() * (torch.rand(B, W, generator=g) > 0.2)
    order = torch.full((B, W), -1, dtype=torch.int32)
    for b in range(B):
        order[b, :settled] = torch.randperm(3 * settled, generator=g)[:settled].to(torch.int32)
    return cache, table, torch.tensor(lens, dtype=torch.int32), weights, order


def _check(state, keep, sinks, recent, **kw):
    cache, table, lens, weights, order = state
    page, most = cache.shape[1], table.shape[1] * cache.shape[1]
    real = [min(max(int(x), 0), most) for x in lens]
    n, w, o, source = ol.evict(real, weights, order, keep, sinks, recent)
    dev = [t.cuda() for t in state]
    at = [t.clone() for t in dev]
    got = L.evict(*dev, keep, sinks=sinks, recent=recent, **kw)
    torch.cuda.synchronize()
    want = cache.clone()
    B, W = weights.shape
    assert got[0].tolist() == n and got[3].shape == (B, keep) and got[1].shape == got[2].shape == (B, W)
    gw, go, gs = (t.cpu() for t in got[1:])
    for b in range(B):
        k = n[b]
        assert gs[b, :k].tolist() == source[b] and (gs[b, k:] == -1).all()
        assert go[b, :k].tolist() == o[b] and (go[b, k:] == -1).all()
        assert torch.equal(gw[b, :k].nan_to_num(-5.0), weights[b, source[b]].nan_to_num(-5.0)) and (gw[b, k:] == 0).all()
        slot = lambda j: (int(table[b, j // page]), j % page)
        for j, s in enumerate(source[b]):
            want[slot(j)] = cache[slot(s)]
    assert torch.equal(dev[0].cpu(), want)
    return at, dev, got


CASES = [
    # lens, page, row, keep, sinks, recent, settled
    ([1], 64, 576, 1, 0, 1, 0),
    ([2], 64, 576, 1, 0, 0, 0),
    ([2, 2], 1, 576, 1, 1, 0, 1),
    ([65, 0, 64, 130], 16, 576, 64, 4, 8, 64),            # one token over, none, just fitting, many over
    ([300, 299, 20], 24, 280, 100, 1, 99, 50),            # only sinks and the newest
    ([500, 77, 1000, 1001], 64, 96, 333, 0, 0, 200),      # by weight alone
    ([2050, 1025, 1024, 1023], 128, 16, 1024, 4, 100, 0),
    ([90, 91], 16, 576, 91, 2, 3, 80),                    # nothing to do
    ([90, 91], 16, 576, 5000, 2, 3, 80),                  # more than the table holds
    ([5001, 2500, 4000], 24, 288, 3001, 1, 100, 1500),
]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens,page,row,keep,sinks,recent,settled", CASES)
def test_evict_keeps_what_the_oracle_keeps(lens, page, row, keep, sinks, recent, settled, dtype):
    banner(f"latent evict {lens} page {page} row {row} keep {keep} {sinks} {recent} settled {settled} {dtype}")
    _check(_state(lens, page, row, dtype, seed=keep + row, settled=settled), keep, sinks, recent)


@pytest.mark.parametrize("most,keep", [(2048, 1900), (2049, 1900), (4096, 3000), (4097, 4000), (8192, 8063), (8192, 8064),
                                       (8192, 8095), (8192, 8096),
                                       (8193, 5000), (8193, 8100), (10240, 2048), (10240, 6144), (12000, 11999), (9000, 1)])
def test_around_the_limits_of_table_and_budget(most, keep):
    """Tables that one workgroup takes and longer ones, few and many rows to move, budgets that end at a chunk's end."""
    banner(f"latent evict table {most} keep {keep}")
    _check(_state([most, most - 1, keep, keep + 1, most // 2], 1, 16, BF16, seed=most + keep, settled=min(keep, 700)), keep,
           min(3, keep), min(keep - min(3, keep), 150))


def test_long_tables():
    """Many workgroups a sequence, ties across them, sequences that fit among those that do not."""
    banner("latent evict long tables")
    _check(_state([40000, 33000, 500], 128, 16, BF16, seed=3, settled=2000), 20000, 4, 700)
    _check(_state([32768, 100, 0], 128, 16, BF16, seed=4), 32000, 4, 700)
    _check(_state([300, 100], 64, 16, BF16, seed=5, per=1000), 200, 4, 70)
    _check(_state([300, 100], 64, 16, BF16, seed=5, per=1000), 70000, 4, 70)
    cache, table, lens, w, order = _state([30000, 20001, 12345], 64, 16, BF16, seed=13, settled=300)
    w[0] = 1.0
    w[1] = (torch.arange(w.shape[1]) % 3).float()
    for keep, recent in ((15000, 0), (20000, 100), (5000, 4000)):
        _check((cache, table, lens, w, order), keep, 5, recent)


def test_ties_and_what_is_no_number():
    banner("latent evict ties")
    cache, table, lens, _, order = _state([700, 650, 700, 700], 32, 96, BF16, seed=6)
    w = torch.zeros(4, order.shape[1])
    w[0] = 1.0                                                # all alike
    w[1, ::3], w[1, 1::7] = 2.5, -0.0                         # three values, zeros of both signs
    w[2] = torch.linspace(-3, 3, w.shape[1])
    w[2, 5:600:11], w[2, 6:600:50], w[2, 7:600:60] = NAN, INF, -INF
    w[3] = 1.0 + (torch.arange(w.shape[1]) % 7) * 2.0 ** -23  # that differ in the last bits only
    for keep, sinks, recent in ((100, 0, 0), (333, 7, 50), (649, 0, 649)):
        _check((cache, table, lens, w, order), keep, sinks, recent)


def test_only_nan_and_orders_at_the_end_of_their_range():
    banner("latent evict extremes")
    cache, table, lens, w, order = _state([200, 130], 32, 96, BF16, seed=7)
    order[0, :3] = torch.tensor([2 ** 31 - 2 - 196, 4, 9])    # the newest ends at 2^31 - 1
    _check((cache, table, lens, torch.full_like(w, NAN), order), 60, 5, 20)


def test_the_same_call_again_and_in_place():
    banner("latent evict twice")
    at, dev, got = _check(_state([500, 77, 300], 16, 576, BF16, seed=8, settled=30), 120, 4, 16)
    cache = dev[0].clone()
    again = L.evict(*dev, 120, sinks=4, recent=16)            # the same state: the same again
    assert all(torch.equal(x, y) for x, y in zip(got, again)) and torch.equal(cache, dev[0])
    place = [t.clone() for t in at]
    res = L.evict(*place, 120, sinks=4, recent=16, in_place=True)
    assert all(x is y for x, y in zip(res, place[2:]))
    assert all(torch.equal(x, y) for x, y in zip(got, res)) and torch.equal(cache, place[0])
    # what is left fits: nothing changes, every row is its own source
    more = L.evict(*place, 120, sinks=4, recent=16, in_place=True)
    assert torch.equal(more[3][0], torch.arange(120, device="cuda", dtype=torch.int32))
    assert all(torch.equal(x, y) for x, y in zip(got[:3], more)) and torch.equal(cache, place[0])


def test_strided_states_and_lengths_past_the_table():
    banner("latent evict strides")
    cache, table, lens, w, o = _state([200, 96, 150], 32, 96, BF16, seed=9, settled=10, width=0)
    wide = torch.full((3, 2, w.shape[1] + 5), 9.0, device="cuda")
    ages = torch.full((3, w.shape[1] + 8), 77, dtype=torch.int32, device="cuda")
    wv, ov = wide[:, 1, 2:-3], ages[:, 8:]
    wv.copy_(w)
    ov.copy_(o)
    a, b = cache.cuda(), cache.cuda()
    dev = [t.cuda() for t in (table, lens)]
    want = L.evict(a, *dev, w.cuda(), o.cuda(), 64, recent=9)
    got = L.evict(b, *dev, wv, ov, 64, recent=9, in_place=True)
    assert all(torch.equal(x, y) for x, y in zip(want, got)) and torch.equal(a, b)
    assert (wide[:, 0] == 9).all() and (wide[:, 1, :2] == 9).all() and (wide[:, 1, -3:] == 9).all()
    assert (ages[:, :8] == 77).all()
    far = lens.clone()
    far[0], far[1] = 1 << 30, -4                              # the table's tokens, none
    _check((cache, table, far, w, o), 64, 2, 9)


def test_other_streams_and_graph_replays():
    """A captured eviction in place, with new weights for every replay."""
    banner("latent evict graphs")
    state = _state([300, 40, 170], 16, 96, BF16, seed=10)
    first = [t.cuda() for t in state]
    live = [t.clone() for t in first]
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    L.evict(*[t.clone() for t in first], 50, recent=4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        source = L.evict(*live, 50, recent=4, in_place=True, workspace=ws)[3]
    for k in range(3):
        for x, y in zip(live, first):
            x.copy_(y)
        live[3].copy_(torch.rand(live[3].shape, generator=torch.Generator().manual_seed(k)))
        want = [t.clone() for t in live]
        graph.replay()
        torch.cuda.synchronize()
        s = L.evict(*want, 50, recent=4, in_place=True)[3]
        assert torch.equal(s, source) and all(torch.equal(x, y) for x, y in zip(want, live))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    late = torch.empty_like(first[3])
    a, b = first[0].clone(), first[0].clone()
    want = L.evict(a, *first[1:], 50, recent=4)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.empty(1 << 27, device="cuda").normal_()         # keeps the stream busy before the weights are there
        late.copy_(first[3])
        got = L.evict(b, first[1], first[2], late, first[4], 50, recent=4)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(want, got)) and torch.equal(a, b)


def _serve(cache, table, pt, pl, lens, weights, order, tokens, keep, w_kv, cos, sin, pos, recent, sinks):
    """A step of a serving loop on a full cache: the new tokens enter it, are answered, and what is over goes."""
    c, k_pe, q = tokens
    page = cache.shape[1]
    rows = lens.long()
    lens += 1
    slots = table.gather(1, (rows // page)[:, None])[:, 0].long() * page + rows % page
    # rows say nothing of the positions any more: the queries are rotated with the keys
    _, q = L.append(cache, c, k_pe, slots, pos, cos, sin, q=q)
    o = L.decode_shared(q[:, None], w_kv, cache, pt, pl, table, lens, 0.1, weights=weights)
    source = L.evict(cache, table, lens, weights, order, keep, sinks=sinks, recent=recent, in_place=True)[3]
    return o, source


def test_serving_loop():
    """Append, decode behind two shared prefixes, evict: each step against the oracle on lists
    of tokens.  The oracle evicts by the kernel's weights (its own are within the bound above)."""
    banner("latent serving loop")
    g = torch.Generator().manual_seed(11)
    r = lambda *s: torch.randn(*s, generator=g)
    B, H, dn, dr, dv, dc, page, keep, sinks, recent = 4, 6, 64, 32, 64, 128, 8, 13, 2, 4
    pre = [37, 20]
    cos, sin = _tables(128, dr)
    w_kv = (r(H, dn + dv, dc) * dc ** -0.5).to(BF16)
    per = 2
    ids = torch.randperm(2 * 5 + B * per, generator=g).to(torch.int32)
    pt, table = ids[:10].view(2, 5), ids[10:].view(B, per)
    cache = r(len(ids), page, dc + dr).to(BF16)
    lens, weights = torch.zeros(B, dtype=torch.int32), torch.zeros(B, per * page)
    order = torch.full((B, per * page), -1, dtype=torch.int32)
    dev = [t.cuda() for t in (cache, table, pt, torch.tensor(pre, dtype=torch.int32), lens, weights, order)]
    consts = w_kv.cuda(), cos.cuda(), sin.cuda()
    held = [[] for _ in range(B)]                   # each sequence's rows, in the order of its cache
    ages = [[] for _ in range(B)]
    gathered = torch.zeros(B, per * page, dtype=torch.float64)
    for step in range(30):
        c, k_pe, q = r(B, dc).to(BF16), r(B, dr).to(BF16), r(B, H, dn + dr).to(BF16)
        pos = torch.tensor([pre[b // 2] + step for b in range(B)], dtype=torch.int32)
        before = dev[5].cpu()
        o, source = _serve(*dev, [t.cuda() for t in (c, k_pe, q)], keep, *consts, pos.cuda(), recent, sinks)
        torch.cuda.synchronize()
        k_rot = ol.rotate(k_pe, pos, cos, sin, False).to(BF16)
        q_rot = torch.cat((q[..., :dn], ol.rotate(q[..., dn:], pos, cos, sin, False).to(BF16)), -1)
        for b in range(B):
            held[b].append(torch.cat((c[b], k_rot[b])))
            ages[b].append(step)
        n = [len(h) for h in held]
        rows = torch.zeros(B, max(n), dc + dr, dtype=BF16)
        for b in range(B):
            rows[b, :n[b]] = torch.stack(held[b])
        # the sequences' rows as pages of their own, behind the prefixes'
        width = -(-max(n) // page)
        paged = torch.zeros(B, width * page, dc + dr, dtype=BF16)
        paged[:, :max(n)] = rows
        both = torch.cat((cache, paged.view(-1, page, dc + dr)))
        own = torch.arange(B * width).view(B, width) + len(cache)
        want, add = ol.decode_shared(q_rot[:, None], w_kv, both, pt, pre, own, n, 0.1)
        _rows_within(o, want, U[BF16])
        # the kernel's weights before the eviction, by where its rows went
        after, src = dev[5].cpu(), source.cpu()
        for b in range(B):
            full = ol.gathered(before[b:b + 1], add[b:b + 1], [n[b]], 1)[0, :n[b]]
            kept = [s for s in src[b].tolist() if s >= 0]
            assert len(kept) == min(n[b], keep)
            off = (after[b, :len(kept)].double() - full[kept]).abs()
            a = add[b, :n[b]]
            assert (off <= 4 * UW[BF16] * (a[kept] + a.mean()) + 2.0 ** -22 * full[kept]).all()
            if n[b] > keep:
                out = next(j for j in range(n[b]) if j not in kept)
                safe = [j for j in range(n[b]) if ages[b][j] < sinks or ages[b][j] > step - recent]
                assert out not in safe
                slack = 4 * UW[BF16] * (a.max() + a.mean()) + 2.0 ** -22 * full.max()
                assert all(full[out] <= full[j] + 2 * slack for j in kept if j not in safe)
            held[b] = [held[b][s] for s in kept]
            ages[b] = [ages[b][s] for s in kept]
            assert dev[6][b, :len(kept)].tolist() == ages[b]
    assert dev[4].tolist() == [keep] * B
    for b in range(B):      # the cache holds what the lists say
        at = torch.arange(keep)
        assert torch.equal(dev[0].cpu()[table[b].long()[at // page], at % page][:, :dc], torch.stack(held[b])[:, :dc])


def test_serving_step_in_a_graph():
    """The step of the loop above as a captured graph, replayed with new tokens and eager work in between."""
    banner("latent serving graph")
    g = torch.Generator().manual_seed(21)
    r = lambda *s: torch.randn(*s, generator=g).to(BF16).cuda()
    B, H, dn, dr, dv, dc, page, keep, per = 6, 20, 64, 32, 64, 512, 16, 40, 3
    cos, sin = (t.cuda() for t in _tables(6000, dr))
    w_kv = (torch.randn(H, dn + dv, dc, generator=g) * dc ** -0.5).to(BF16).cuda()
    front = 4096 // page
    ids = torch.randperm(front + B * per, generator=g).to(torch.int32).cuda()
    pt, table = ids[:front].view(1, front), ids[front:].view(B, per)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    state = [r(len(ids), page, dc + dr), table, pt, i32(4090), i32(*[keep] * B), torch.rand(B, per * page, generator=g).cuda(),
             torch.full((B, per * page), -1, dtype=torch.int32, device="cuda")]
    tokens = [r(B, dc), r(B, dr), r(B, H, dn + dr)]
    pos = i32(*[4090 + keep] * B)
    rest = (keep, w_kv, cos, sin, pos, 8, 2)
    step = lambda s: _serve(*s, tokens, *rest)
    twin = [t.clone() for t in state]
    step([t.clone() for t in state])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(state)
    for k in range(4):
        for t in tokens:
            t.copy_(torch.randn(t.shape, generator=g))
        pos += 1
        graph.replay()
        torch.cuda.synchronize()
        want = step(twin)
        assert all(torch.equal(a, b) for a, b in zip(out, want))
        assert all(torch.equal(a, b) for a, b in zip(state, twin))


def test_nothing_to_do():
    banner("latent evict empty dimensions")
    z = lambda *s, dt=F32: torch.ones(*s, dtype=dt, device="cuda")
    i = lambda *s: z(*s, dt=torch.int32)
    cache = z(3, 16, 96, dt=BF16)
    for B, per in ((0, 2), (2, 0)):
        lens, w, o, s = L.evict(cache, i(B, per), i(B), z(B, 40), i(B, 40), 7)
        assert lens.shape == (B,) and s.shape == (B, 7) and (lens == 0).all() and (s == -1).all()
        assert w.shape == o.shape == (B, 40) and (w == 0).all() and (o == -1).all()


def test_refusals():
    banner("latent evict refusals")
    cache, table, lens, w, o = (t.cuda() for t in _state([50, 20], 16, 96, BF16, seed=12))
    W = w.shape[1]
    for keep, sinks, recent in ((0, 0, 0), (-1, 0, 0), ((1 << 32) + 10, 0, 0), (5, 6, 0), (5, 0, 6), (5, 3, 3), (5, -1, 0), (5, 0, -1)):
        with pytest.raises(ValueError, match="sinks and recent"):
            L.evict(cache, table, lens, w, o, keep, sinks=sinks, recent=recent)
    for bad in (w[:1], w.double(), w[:, :-4], w.cpu(), w[0], w.t().contiguous().t(), w[:1].expand(2, W)):
        with pytest.raises(ValueError, match="weights"):
            L.evict(cache, table, lens, bad, o, 10)
    for bad in (o[:1], o.long(), o[:, :-4], o.cpu(), o[:, :-1]):
        with pytest.raises(ValueError, match="order"):
            L.evict(cache, table, lens, w, bad, 10)
    for bad in (lens.long(), lens[:1], lens.cpu()):
        with pytest.raises(ValueError, match="kv_lens"):
            L.evict(cache, table, bad, w, o, 10)
    for bad in (table.long(), table[0], table.cpu()):
        with pytest.raises(ValueError, match="page_table"):
            L.evict(cache, bad, lens, w, o, 10)
    with pytest.raises(ValueError, match="in place"):
        L.evict(cache, table, torch.stack((lens, lens), 1)[:, 0], w, o, 10, in_place=True)
    with pytest.raises(ValueError, match="dense"):
        L.evict(cache.transpose(0, 1), table, lens, w, o, 10)
    with pytest.raises(ValueError, match="gradient"):
        L.evict(cache.clone().requires_grad_(True), table, lens, w, o, 10)
    with pytest.raises(TypeError, match="bfloat16 or float32"):
        L.evict(cache.half(), table, lens, w, o, 10)
    with pytest.raises(ValueError, match="HIP"):
        L.evict(cache.cpu(), table, lens, w, o, 10)
    with pytest.raises(ValueError, match="workspace"):
        L.evict(cache, table, lens, w, o, 10, workspace=torch.zeros(1 << 20, dtype=torch.uint8))
    with pytest.raises(_lib.AtomicError, match="SHAPE"):
        L.evict(torch.zeros(9, 16, 600, dtype=BF16, device="cuda"), table, lens, w, o, 10)
