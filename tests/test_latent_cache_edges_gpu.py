"""Shared prefixes, gathered weights and eviction on the GPU at the edges that the kernels' plans
have: what a part holds that has nothing else in it, and calls that reach few of the paths."""
import pytest
import torch
from torch.autograd import forward_ad

from _util import banner
from atomic_ops import latent as L
from oracle import latent as ol
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
