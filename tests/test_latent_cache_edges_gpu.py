"""Shared prefixes, gathered weights and eviction on the GPU at the edges that the kernels' plans
have: what a part holds that has nothing else in it, and calls that reach few of the paths."""
import pytest
import torch
from torch.autograd import forward_ad

from _util import banner
from atomic_ops import latent as L
from oracle import latent as ol
from test_latent_evict_gpu import _state
from test_latent_shared_gpu import BF16, F32, _case

pytestmark = pytest.mark.gpu

NAN = float("nan")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("where,at,most", [("own", 32, 0), ("own", 64, 0), ("own", 0, 0), ("prefix", 64, 0),
                                           ("prefix", 0, 0), ("prefix", 64, 4096), ("prefix", 96, 4096)])
def test_a_nan_that_is_alone_in_its_part_stays_one(where, at, most, dtype):
    """Parts are of 32 or 64 tokens here, so the last token is a part by itself: a score that is no number
    makes the softmax of its row none, and with it what every token of the sequence gathers."""
    banner(f"latent weights behind a NaN {where} {at} {most} {dtype}")
    n, H = 1, 18
    pre, own = ([at + 1], [20, 0, 33]) if where == "prefix" else ([50], [at + 1, 20, 33])
    q, w, cache, pt, pl, table, ln = _case(pre, own, n, H, 64, 32, 64, 64, 16, dtype, seed=at + n)
    tab = pt[0] if where == "prefix" else table[0]
    cache[tab[at // 16], at % 16, :64] = NAN
    d = [t.cuda() for t in (q, w, cache, torch.cat((pt, pt.new_full((1, max(0, most // 16 - pt.shape[1])), -7)), 1), pl,
                            table, ln)]
    before = torch.zeros(3, table.shape[1] * 16)
    got = before.cuda()
    o = L.decode_shared(*d, 0.1, weights=got)
    want, add = ol.decode_shared(q, w, cache, pt, pl, table, own, 0.1)
    want_w = ol.gathered(before, add, own, n)
    assert torch.equal(torch.isnan(o.cpu()), torch.isnan(want))
    assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want_w))
    assert torch.isnan(want_w[0, :own[0]]).all() and not torch.isnan(want_w[0, own[0]:]).any()


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("which", ["cache", "weights"])
def test_evict_refuses_tangents(which, in_place):
    """A row that moves would leave its tangent with another token's row."""
    banner(f"latent evict tangents {which} {in_place}")
    state = {"cache": torch.randn(4, 16, 96, device="cuda"),
             "table": torch.arange(4, dtype=torch.int32, device="cuda").view(2, 2),
             "lens": torch.tensor([32, 20], dtype=torch.int32, device="cuda"), "weights": torch.rand(2, 32, device="cuda"),
             "order": torch.full((2, 32), -1, dtype=torch.int32, device="cuda")}
    before = {k: t.clone() for k, t in state.items()}
    with forward_ad.dual_level():
        given = {**state, which: forward_ad.make_dual(state[which], torch.ones_like(state[which]))}
        with pytest.raises(NotImplementedError, match="forward mode"):
            L.evict(*given.values(), 8, in_place=in_place)
    assert all(torch.equal(state[k], before[k]) for k in state)
    assert L.evict(*state.values(), 8, in_place=in_place)[0].tolist() == [8, 8]


@pytest.mark.parametrize("call", ["forward", "backward", "attention", "append", "decode", "decode_shared", "evict"])
def test_tensors_of_another_device_than_the_current_one(call, monkeypatch):
    """The library launches on the current device: each call makes the tensors' device it for that
    long.  (With one card the current one is said to be another.)"""
    banner(f"latent on another device {call}")
    r = lambda *s: torch.randn(*s, dtype=BF16, device="cuda")
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
    qkv = r(1, 5, 2, 96), r(1, 5, 2, 128), r(1, 5, 32)
    q, w, cache, table, lens = r(1, 1, 2, 96), r(2, 128, 64), r(4, 16, 96), i(0, 1)[None], i(20)
    o, lse, rest = L.forward(*qkv, 0.1, save=True)
    dout = r(1, 5, 2, 64)
    cos, sin = torch.rand(9, 16, device="cuda"), torch.rand(9, 16, device="cuda")
    calls = {
        "forward": lambda: L.forward(*qkv, 0.1),
        "backward": lambda: L.backward(*qkv, o, lse, dout, 0.1, rest=rest),
        "attention": lambda: torch.autograd.grad(L.attention(*[t.requires_grad_(True) for t in qkv], 0.1), qkv, dout),
        "append": lambda: L.append(cache, r(3, 64) * 0, r(3, 32) * 0, i(2, 3, 4).long(), i(0, 1, 2), cos, sin),
        "decode": lambda: (L.decode(q, w, cache, table, lens, 0.1),),
        "decode_shared": lambda: (L.decode_shared(q, w, cache, table, lens, table + 2, lens, 0.1),),
        "evict": lambda: L.evict(cache.clone(), table, lens, torch.ones(1, 32, device="cuda"), i(*[-1] * 32)[None], 9),
    }
    want = calls[call]()
    current, entered = [7], []

    class Device:
        def __init__(self, device):
            self.to = torch.device(device).index

        def __enter__(self):
            entered.append(self.to)
            self.was, current[0] = current[0], self.to

        def __exit__(self, *_):
            current[0] = self.was

    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "current_device", lambda: current[0])
        m.setattr(torch.cuda, "device", Device)
        got = calls[call]()
    assert entered and set(entered) == {0} and current == [7]
    assert all(torch.equal(a, b) for a, b in zip(got, want) if a is not None)


def _evict_in_place(lens, page, keep, sinks, recent, seed, settled=0, strided=False, per=None):
    state = [t.cuda() for t in _state(lens, page, 16, BF16, seed=seed, settled=settled, per=per)]
    other = [t.clone() for t in state]
    if strided:      # rows of wider buffers
        wide = torch.full((len(lens), state[3].shape[1] + 9), 7.0, device="cuda")
        ages = torch.full((len(lens), state[4].shape[1] + 4), 77, dtype=torch.int32, device="cuda")
        wide[:, 2:-7], ages[:, 4:] = state[3], state[4]
        other[3], other[4] = wide[:, 2:-7], ages[:, 4:]
    want = L.evict(*state, keep, sinks=sinks, recent=recent)
    got = L.evict(*other, keep, sinks=sinks, recent=recent, in_place=True)
    assert all(a is b for a, b in zip(got, other[2:]))
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(other[0], state[0])
    if strided:
        assert (wide[:, :2] == 7).all() and (wide[:, -7:] == 7).all() and (ages[:, :4] == 77).all()


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("lens,page,keep,sinks,recent,settled,per", [
    ([40000, 33000, 500], 128, 20000, 4, 700, 2000, None),       # movers and holes of many workgroups
    ([32768, 100, 0], 128, 32000, 4, 700, 0, None),
    ([9000, 8193], 1, 1, 0, 0, 30, None),
    ([12000, 12000], 24, 11999, 0, 11000, 500, None),
    ([300, 100], 64, 70000, 4, 70, 0, 1000),                     # more than the table holds
])
def test_long_tables_in_place(lens, page, keep, sinks, recent, settled, per, strided):
    """The launches after the selection read the state that the call writes over."""
    banner(f"latent evict long in place {lens} page {page} keep {keep} {strided}")
    _evict_in_place(lens, page, keep, sinks, recent, 14, settled, strided, per)


def test_a_long_table_as_a_replayed_graph():
    """A captured eviction of long tables in place, replayed on new states with eager work between."""
    banner("latent evict long graph")
    states = [[t.cuda() for t in _state([30000, 20001, 123], 64, 16, BF16, seed=s, settled=100 * s)] for s in range(4)]
    held = [t.clone() for t in states[0]]
    kw = dict(sinks=4, recent=500)
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        L.evict(*[t.clone() for t in held], 9000, **kw)
    torch.cuda.current_stream().wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        source = L.evict(*held, 9000, **kw, in_place=True)[3]
    for state in states[1:] + states:
        for a, b in zip(held, state):
            a.copy_(b)
        graph.replay()
        cache = state[0].clone()
        want = L.evict(cache, *state[1:], 9000, **kw)
        assert all(torch.equal(a, b) for a, b in zip((*held[2:], source, held[0]), (*want, cache)))


@pytest.mark.parametrize("rows", [100, 9000])
def test_evict_with_a_state_of_nearly_2_to_the_31(rows):
    """What lies past the length is cleared up to the last element, by steps that would not fit 32 bits."""
    banner(f"latent evict wide state {rows}")
    W = (1 << 31) - 1
    cache = torch.randn(-(-rows // 64), 64, 16, device="cuda").to(BF16)
    table = torch.arange(cache.shape[0], dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([rows], dtype=torch.int32, device="cuda")
    weights = torch.ones(1, W, device="cuda")
    order = torch.full((1, W), -1, dtype=torch.int32, device="cuda")
    order[0, rows:] = 5
    got = L.evict(cache, table, lens, weights, order, rows // 2, sinks=3, recent=7, in_place=True)
    assert got[0].tolist() == [rows // 2]
    assert (weights[0, :rows // 2] == 1).all() and (order[0, :rows // 2] >= 0).all()
    for i in range(rows // 2, W, 1 << 28):
        assert not weights[0, i:i + (1 << 28)].any() and (order[0, i:i + (1 << 28)] == -1).all()
