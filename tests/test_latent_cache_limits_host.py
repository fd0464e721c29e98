"""Sizes at the ends of what the C entries of shared prefixes take: no GPU is needed, nothing is launched."""
import ctypes

import pytest
import torch

from atomic_ops import _lib, latent
from test_latent_cache_host import _shared


def _size(**kw):
    return _lib.load().atomic_latent_decode_shared_workspace_size(ctypes.byref(_shared(**kw)))


def test_positions_behind_a_prefix_fit_32_bits():
    """A query's position is below the tokens that both tables hold together; at 2^31 the last one's
    number of tokens would not fit a 32-bit integer."""
    wide = dict(batch=1, heads=1, prefixes=1, page=1 << 20)
    assert _size(prefix_pages=1 << 10, table_pages=1, **wide) > 0
    assert _size(prefix_pages=1 << 10, table_pages=(1 << 10) - 1, **wide) > 0
    assert _size(prefix_pages=1 << 10, table_pages=1 << 10, **wide) == 0


@pytest.mark.parametrize("which", [0, 1])
def test_a_prefix_table_without_lengths_is_refused(which):
    i = torch.zeros(1, 1, dtype=torch.int32)
    pair = [i, i[0]]
    pair[which] = None
    with pytest.raises(ValueError, match="come together"):
        latent.decode_shared(torch.zeros(1, 1, 1, 16), torch.zeros(1, 16, 8), torch.zeros(1, 1, 16), *pair, i, i[0], 1.0)
