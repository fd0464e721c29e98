"""The oracle of shared prefixes, gathered weights and eviction against its other forms and closed ones (CPU)."""
import math

import pytest
import torch

from oracle import latent as ol

F = torch.float64


def _case(G, S, n, H, pre, own, page, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=F)
    dn, dr, dv, dc = 8, 8, 16, 24
    B = G * S
    front, per = -(-max(pre) // page), -(-max(own) // page)
    ids = torch.randperm(G * front + B * per, generator=g)
    cache = r(G * front + B * per, page, dc + dr)
    return (r(B, n, H, dn + dr), r(H, dn + dv, dc), cache, ids[:G * front].view(G, front), pre,
            ids[G * front:].view(B, per), own, 0.2)


@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("pre,own", [([8, 4], [3, 0, 5, 1]), ([0, 8], [4, 2, 0, 6])])
def test_shared_is_decode_over_both_tables(pre, own, n):
    """Prefixes of whole pages: the two tables as one."""
    page = 4
    q, w, cache, pt, pl, table, ln, scale = _case(2, 2, n, 2, pre, own, page, seed=sum(pre) + n)
    o, weights = ol.decode_shared(q, w, cache, pt, pl, table, ln, scale)
    for b in range(4):
        P = pre[b // 2]
        joint = torch.cat((pt[b // 2, :P // page], table[b]))[None]
        want = ol.decode(q[b:b + 1], w, cache, joint, [P + own[b]], scale)
        assert (o[b] - want[0]).abs().max() < 1e-12
        # a row's probabilities sum to one: over its own tokens to what the prefix leaves
        assert (weights[b, own[b]:] == 0).all()
        if P == 0:
            assert abs(weights[b].sum() - 2 * min(n, own[b])) < 1e-12


def test_gathered_weights_begin_with_the_newest():
    add = torch.tensor([[1.0, 2, 3, 0], [4, 0, 0, 0]], dtype=F)
    before = torch.full((2, 4), 10.0)
    got = ol.gathered(before, add, [3, 1], 2)
    assert got.tolist() == [[11, 2, 3, 10], [4, 10, 10, 10]]


def test_evict_by_hand():
    nan, inf = math.nan, math.inf
    w = torch.tensor([[0.0, 5, 1, 1, nan, 2, 1, 0], [9, 9, 9, 0, 0, 0, 0, 0], [1, -inf, inf, 0.5, -0.0, 0, 3, 4]])
    o = torch.full((3, 8), -1)
    ln, wt, od, src = ol.evict([8, 3, 8], w, o, 4, 1, 1)
    # kept: the sink 0, the newest 7, then 5.0 and 2.0
    assert ln == [4, 3, 4]
    assert src[0] == [0, 1, 5, 7] and wt[0] == [0, 5, 2, 0] and od[0] == [0, 1, 5, 7]
    assert src[1] == [0, 1, 2] and od[1] == [0, 1, 2]
    assert src[2] == [0, 6, 2, 7] and od[2] == [0, 6, 2, 7]
    # ties go to the lowest rows; rows that an eviction has seen keep their order
    w = torch.tensor([[1.0, 1, 1, 1, 1, 1]])
    o = torch.tensor([[4, 0, 7, 2, -1, -1]])
    assert ol.evict([6], w, o, 3, 0, 1)[1:] == ([[1, 1, 1]], [[4, 0, 9]], [[0, 1, 5]])
    assert ol.evict([6], w, o, 3, 3, 0)[3] == [[0, 1, 3]]
    assert ol.evict([6], w, o, 3, 0, 3)[3] == [[4, 5, 2]]
