"""Sequences behind prefixes that are bound by matrix instructions (bf16, more than 32 rows,
tables of 4096 tokens or more) against the float64 oracle."""
import pytest
import torch

from _util import banner
from atomic_ops import latent as L
from oracle import latent as ol
from test_latent_shared_gpu import BF16, _case

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
