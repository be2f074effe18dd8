"""Calls of the token path that the documentation allows, at its edges, on the GPU: against plain 64-bit forms, or refused.

Bounds as in test_gpu_token_ops.py: a rounding to type t is off by at most half a step (eps / 2 relative), a chain of n
fp32 additions by n * 2^-24 of what it adds up.
"""

import pytest
import torch

from difflut_b200.utils import group_norm, sample_logits

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _normal(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


# ---------------------------------------------------------------------------------------------- sampling
@pytest.mark.parametrize("V", [300, 2000])
def test_sampling_counts_per_row_past_32_bits(V):
    """Their low words alone would be 5, 1 and 2^31 - 1."""
    x, u = _normal(4, V), torch.tensor([0.1, 0.5, 0.9, 0.3], device=DEV)
    k = torch.tensor([-2 ** 32 + 5, -2 ** 33 + 1, -2 ** 31 - 1, 2 ** 32 + 1], device=DEV)
    assert torch.equal(sample_logits(x, u, top_k=k), sample_logits(x, u))
    assert torch.equal(sample_logits(x, u, top_k=k.clamp(min=0).to(torch.uint64)), sample_logits(x, u))


# ---------------------------------------------------------------------------------------------- group norm
@pytest.mark.parametrize("shape,groups", [((0, 8), 2), ((0, 1, 8), 2), ((0, 1024), 1), ((0, 3, 8), 8)])
def test_group_norm_of_no_samples(shape, groups):
    x = torch.empty(*shape, device=DEV, requires_grad=True)
    w, b = (torch.ones(shape[-1], device=DEV, requires_grad=True) for _ in range(2))
    y = group_norm(x, groups, w, b, activation="silu")
    gx, gw, gb = torch.autograd.grad(y, (x, w, b), torch.empty_like(y))
    assert y.shape == gx.shape == shape and not bool(gw.any()) and not bool(gb.any())
    with torch.no_grad():
        assert group_norm(x, groups, w, b).shape == shape
