"""The host layer of latent attention where no GPU is needed: what it hands to the library."""
import ctypes

import pytest
import torch

from atomic_ops import _lib, latent

BF16 = torch.bfloat16


@pytest.mark.parametrize("B", [1, 3])
@pytest.mark.parametrize("which", ["q", "kv", "k_pe"])
def test_one_token_of_a_tensor_with_tokens_far_apart(which, B):
    """A dimension of one is never stepped along, so its stride (here 32 MB and more,
    a token of a tensor laid out token first) is no reason for a refusal."""
    far = (1 << 24) + 8
    shapes = {"q": (B, 1, 2, 96), "kv": (B, 1, 2, 128), "k_pe": (B, 1, 32)}
    t = {n: torch.zeros(s, dtype=BF16) for n, s in shapes.items()}
    x = t[which]
    t[which] = x.as_strided(x.shape, (x.stride(0), far, *x.stride()[2:]))
    args, ops = latent.make_args(t["q"], t["kv"], t["k_pe"], 0.1, True, torch.zeros(B, 1, 2, 64, dtype=BF16))
    lib = _lib.load()
    assert lib.atomic_latent_fwd_workspace_size(ctypes.byref(args)) > 0
    assert lib.atomic_latent_bwd_workspace_size(ctypes.byref(args)) > 0
    assert ops[("q", "kv", "k_pe").index(which)].data_ptr() == x.data_ptr()      # read in place
