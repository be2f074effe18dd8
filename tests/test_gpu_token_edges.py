"""Calls of the token path that the documentation allows, at its edges, on the GPU: against plain 64-bit forms, or refused.

Bounds as in test_gpu_token_ops.py: a rounding to type t is off by at most half a step (eps / 2 relative), a chain of n
fp32 additions by n * 2^-24 of what it adds up.
"""

import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from difflut_b200.encoder import embedding_lookup
from difflut_b200.utils import dropout, group_norm, sample_logits

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


# ---------------------------------------------------------------------------------------------- differentiation
def test_forward_mode_differentiation_is_refused():
    """No operator has a forward derivative: none may answer a dual tensor as if its tangent were zero."""
    x, w, ids = _normal(6, 16), _normal(16, seed=1), torch.arange(6, device=DEV)
    calls = [lambda t: dropout(t, 0.5, seed=1), lambda t: group_norm(t, 4), lambda t: embedding_lookup(ids, t),
             lambda t: group_norm(x, 4, t[0])]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in calls:
            with pytest.raises(NotImplementedError, match="jvp"):
                call(dual)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="jvp"):
                call(dual)
        inside = [call(x) for call in calls]  # tensors without a tangent are taken as ever
    assert all(torch.equal(call(x), y) for call, y in zip(calls, inside))


def test_gradient_with_a_forward_mode_tangent_is_refused():
    """Forward over reverse: the operator's input has no tangent, what comes back to it has one."""
    ids = torch.arange(6, device=DEV)
    for call in (lambda t: dropout(t, 0.5), lambda t: embedding_lookup(ids, t), lambda t: group_norm(t, 4)):
        x = torch.ones(6, 16, device=DEV, requires_grad=True)
        y = call(x)
        with forward_ad.dual_level():
            g = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(NotImplementedError, match="jvp"):
                torch.autograd.grad(y, x, g, retain_graph=True)
            with pytest.raises(NotImplementedError, match="jvp"):
                torch.autograd.grad(y, x, g, retain_graph=True, create_graph=True)
            torch.autograd.grad(y, x, torch.ones_like(y))
