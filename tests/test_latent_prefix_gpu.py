"""Sequences behind prefixes that are bound by matrix instructions (bf16, more than 32 rows,
tables of 4096 tokens or more) against the float64 oracle."""
import pytest
import torch

from _util import banner
from atomic_ops import latent as L
from oracle import latent as ol
from test_latent_shared_gpu import BF16, U, UW, _case, _rows_within, _weights_within

pytestmark = pytest.mark.gpu


def _exact_queries(pre, own, n, H, dn, dr, dv, dc, page, seed, most):
    """A case whose q_lat has no rounding: each key without position is one latent."""
    q, w, cache, pt, pl, table, ln = _case(pre, own, n, H, dn, dr, dv, dc, page, BF16, seed)
    w[:, :dn] = torch.eye(dc)[:dn]
    return q, w, cache, torch.cat((pt, pt.new_full((len(pre), max(0, -(-most // page) - pt.shape[1])), -7)), 1), pl, table, ln


@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("dc,dr", [(512, 64), (256, 32)])
@pytest.mark.parametrize("P", [1, 2])
def test_a_row_that_looks_at_one_token_has_its_length(P, dc, dr, scored):
    """A probability's rounding may not stay in o as a factor of its row.

    Each of the dv outputs of a row is off by its own rounding, evenly up to 2^-8 of itself, so
    the row's length along the exact one by 2^-8 / sqrt(3) * sqrt(sum o^4) / sum o^2, for normal
    numbers 2^-8 / sqrt(dv) in the mean; four times that is allowed.  (With two tokens scores
    far apart leave one.)"""
    banner(f"latent prefix length of a row {P} {dc} {scored}")
    d = _exact_queries([P], [0] * 40, 1, 2, 64, dr, 128, dc, 64, 50, 4096)
    scale = 0.1 if P == 1 else 40.0
    weights = torch.zeros(40, 64, device="cuda") if scored else None
    o = L.decode_shared(*(t.cuda() for t in d), scale, weights=weights).double().cpu()
    want, _ = ol.decode_shared(*d[:5], d[5], [0] * 40, scale)
    along = (o * want).sum(-1) / (want * want).sum(-1)
    assert ((along - 1).abs() <= 4 * 2.0 ** -8 * 128 ** -0.5).all(), (along - 1).abs().max()


def _rounded_once(o, want, share=0.03):
    """All but a share of o are the bf16 numbers nearest to the exact ones.

    An error of e times an output's terms moves its rounding in a share of e / ulp of the
    cases, ulp at least 2^-8 of an output; over outputs that are normal numbers of the
    terms' size the mean of their inverses, as far as the error is the smaller one, is
    0.8 * 2 ln(2^-8 / e).  float32 sums and the two bf16 numbers that p and o_lat each enter
    as leave e below 2^-16: a share of 0.8 * 2^-8 * 0.8 * 2 * ln(2^8) = 0.03."""
    assert torch.isfinite(o).all()
    other = (o.cpu() != want.to(BF16)).double().mean().item()
    assert other <= share, other


@pytest.mark.parametrize("dc,dr", [(512, 64), (256, 32)])
@pytest.mark.parametrize("P", [1, 40, 4200])
def test_tokens_of_one_latent(P, dc, dr):
    """Every token of the prefix carries one latent and a key of its own: whatever the
    probabilities, o is that latent's value.  So nothing but the parts' sums and o's
    rounding is left, at any length."""
    banner(f"latent prefix of one latent {P} {dc}")
    d = _exact_queries([P], [0] * 40, 1, 2, 64, dr, 128, dc, 64, 51, 4096)
    cache = d[2]
    cache[..., :dc] = torch.randn(dc, generator=torch.Generator().manual_seed(P)).to(BF16)
    o = L.decode_shared(*(t.cuda() for t in d), 0.1)
    _rounded_once(o, ol.decode_shared(*d[:5], d[5], [0] * 40, 0.1)[0])


@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("dc,dr", [(512, 64), (256, 32), (72, 24)])
@pytest.mark.parametrize("most", [0, 4096])
def test_a_short_prefix_in_a_wide_table(most, dc, dr, scored):
    """p enters as two bf16 numbers behind a prefix of fewer than 2048 tokens, however many its table has
    room for, so o has no other rounding than its own in either table (the queries having none)."""
    banner(f"latent prefix short in a table of {most} {dc} {scored}")
    pre, own = [33, 64, 1, 300, 0, 700], [17 * i % 50 for i in range(30)]
    d = _exact_queries(pre, own, 1, 8, 64, dr, 128, dc, 16, 52, most)
    weights = torch.zeros(30, d[5].shape[1] * 16, device="cuda") if scored else None
    o = L.decode_shared(*(t.cuda() for t in d), 0.1, weights=weights)
    _rounded_once(o, ol.decode_shared(*d[:5], d[5], own, 0.1)[0])


def _in_64_bits(q, w, cache, pt, pre, table, own, scale):
    """(o, weights) for one query token a sequence, every prefix row at once (the sizes below are too much
    for the oracle)."""
    f = torch.float64
    B, _, H, d = q.shape
    dc, page, S = w.shape[2], cache.shape[1], q.shape[0] // len(pre)
    dn = d - (cache.shape[2] - dc)
    rows = lambda tab, ln: cache[tab[torch.arange(ln, device="cuda") // page].long(),
                                 torch.arange(ln, device="cuda") % page].to(f)
    k, v, x = w[:, :dn].to(f), w[:, dn:].to(f), q[:, 0].to(f)
    x = torch.cat((torch.stack([x[:, h, :dn] @ k[h] for h in range(H)], 1), x[..., dn:]), -1)
    o_lat, weights = torch.zeros(B, H, dc, dtype=f, device="cuda"), torch.zeros(B, table.shape[1] * page, dtype=f)
    for g, P in enumerate(pre):
        front = rows(pt[g], P)
        sf = (x[g * S:(g + 1) * S].flatten(0, 1) @ front.t() * scale).view(S, H, P)
        for b in range(S):
            at = g * S + b
            mine = rows(table[at], own[at])
            p = torch.softmax(torch.cat((sf[b], x[at] @ mine.t() * scale), 1), 1)
            o_lat[at] = p[:, :P] @ front[:, :dc] + p[:, P:] @ mine[:, :dc]
            weights[at, :own[at]] = p[:, P:].sum(0).cpu()
    o = torch.stack([o_lat[:, h] @ v[h].t() for h in range(H)], 1)[:, None]
    return o.cpu(), weights


LARGE = [
    # prefixes, tokens of their table, own tokens of the longest, sequences, heads, widths, page
    # splits of 1024 tokens, a prefix workgroup for every CU and own ones before them, row blocks dealt to the XCDs
    ([31 * 1024 - 1], 32768, 512, 64, 16, (64, 64, 64, 512), 64),
    ([31 * 1024], 32768, 512, 64, 16, (64, 64, 64, 512), 64),
    ([30 * 1024 + 1], 32768, 512, 64, 16, (64, 32, 64, 256), 128),
    # splits of 1216, rounds and a part of one, row blocks that are not dealt
    ([53 * 1216 - 1], 65536, 64, 66, 16, (32, 32, 64, 512), 256),
    ([53 * 1216 + 1], 65536, 64, 130, 8, (32, 24, 64, 264), 256),
    # one workgroup's row block, more own splits than one turn of the join takes: 32 and 64
    ([4096], 4096, 8192, 8, 8, (64, 64, 64, 512), 64),
    ([2500], 4096, 16384, 4, 16, (64, 32, 64, 200), 128),
    # splits of 832 of two prefixes
    ([19 * 832 + 1, 16384], 16384, 64, 96, 16, (32, 64, 32, 512), 64),
]


@pytest.mark.parametrize("scored", [False, True])
@pytest.mark.parametrize("pre,most,longest,B,H,dims,page", LARGE)
def test_prefixes_of_many_long_splits(pre, most, longest, B, H, dims, page, scored):
    banner(f"latent prefix large {pre} of {most} own {longest} B{B} H{H} {dims} page {page} {scored}")
    dn, dr, dv, dc = dims
    own = [longest] + [longest * i * 37 // B % (longest + 1) for i in range(1, B)]
    q, w, cache, pt, pl, table, ln = _case(pre, own, 1, H, dn, dr, dv, dc, page, BF16, seed=B + pre[0])
    pt = torch.cat((pt, pt.new_full((len(pre), most // page - pt.shape[1]), -7)), 1)
    d = [t.cuda() for t in (q, w, cache, pt, pl, table, ln)]
    scale = (dn + dr) ** -0.5
    before = torch.rand(B, table.shape[1] * page, generator=torch.Generator().manual_seed(1))
    weights = before.cuda() if scored else None
    o = L.decode_shared(*d, scale, weights=weights)
    want, add = _in_64_bits(d[0], d[1], d[2], d[3], pre, d[5], own, scale)
    _rows_within(o, want, U[BF16])
    if scored:
        _weights_within(weights, before, add, own, 1, UW[BF16])
    else:
        assert torch.equal(L.decode_shared(*d, scale), o)      # the same bits


@pytest.mark.parametrize("mul", [1.0, 4.0, 10.0])
@pytest.mark.parametrize("dc,P,most", [(512, 300, 0), (512, 300, 4160), (512, 3000, 4160), (128, 3000, 4160)])
def test_weights_of_scores_of_a_large_spread(dc, P, most, mul):
    """A score of spread s is off by s times what one of unit spread is, 0.58 * 2^-16 s by the query's two
    numbers.  Behind a prefix of many rows the rest of q_lat's rounding is in the row's sum by its first
    order; what is left is half the variance of the rounding's scores, 0.58 * 2^-9 s each at most, in a
    sum that every weight of the row has as a factor."""
    banner(f"latent prefix weights of spread {mul} {dc} {P} {most}")
    pre, own = [P, 77], [40, 1, 0, 90]
    q, w, cache, pt, pl, table, ln = _case(pre, own, 1, 18, 64, 32, 64, dc, 32, BF16, seed=53)
    pt = torch.cat((pt, pt.new_full((2, max(0, most // 32 - pt.shape[1])), 1 << 30)), 1)
    scale = mul * (64 + 32) ** -0.5
    weights = torch.zeros(4, table.shape[1] * 32, device="cuda")
    d = [t.cuda() for t in (q, w, cache, pt, pl, table, ln)]
    L.decode_shared(*d, scale, weights=weights)
    _, add = _in_64_bits(d[0], d[1], d[2], d[3], pre, d[5], own, scale)
    u = mul * 2.0 ** -15 + 2e-5 + (0.58 * 2.0 ** -9 * mul) ** 2 / 2
    _weights_within(weights, torch.zeros(4, table.shape[1] * 32), add, own, 1, u)
