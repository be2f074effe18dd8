"""Calls of the token path that the documentation allows, at its edges, on the GPU: against plain 64-bit forms, or refused.

Bounds as in test_gpu_token_ops.py: a rounding to type t is off by at most half a step (eps / 2 relative), a chain of n
fp32 additions by n * 2^-24 of what it adds up.
"""

import copy

import numpy as np
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.utils.checkpoint import checkpoint

from difflut_b200 import _native
from difflut_b200.encoder import embedding_lookup
from difflut_b200.utils import Dropout, dropout, group_norm, sample_logits
from token_util import half_step, philox

pytestmark = pytest.mark.gpu
DEV = "cuda"
U32 = 2.0 ** -24


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


def _variance_bound(values, width, threads):
    """Relative error of the variance of groups whose threads hold `values` values each, `width` per row.

    A thread takes its values by runs, squares relative to the mean of what came before the run: these add up to no more
    than twice the squares around the thread's mean (the first run's to nine times, its centre being the mean of one of
    eight rows), and a run is at most 32 rows.  Runs are joined by one addition each, then the threads of a block, a
    lane of a warp after the other."""
    return (2 * 32 * width + 9 * 8 * width + values / (32 * width) + 8 + threads / 32 + 16) * U32


@pytest.mark.parametrize("dtype,S,C", [(torch.float32, 524288, 4), (torch.bfloat16, 262144, 8), (torch.float32, 1048576, 2)])
def test_group_norm_value_far_from_all_that_follow(dtype, S, C):
    """Thousands of values per thread, the first one far away: the variance is what the other ones make it.

    So many samples that each is one block of 256 threads, 8192 values a thread; the samples looked at have an outlier in
    their first row and zeros behind it, small noise behind it, and noise without it."""
    N, width = 600, C
    x = torch.zeros(N, S, C, device=DEV, dtype=dtype)
    noise = torch.randn(S, C, device=DEV, generator=torch.Generator(DEV).manual_seed(3))
    x[0, 0, 0] = 1003.7
    x[1] = (noise * 0.05).to(dtype)
    x[1, 0, 0] = 1003.7
    x[2] = noise.to(dtype)
    y = group_norm(x, 1)
    bound = _variance_bound(8192, width, 256)
    for n in range(3):
        v = x[n].double()
        mean = v.mean()
        var = (v - mean).square().mean()
        want = (v - mean) / torch.sqrt(var + 1e-5)
        # half the variance's error for its root, roundings of the linear form, the mean off by its roundings and the
        # block's share of a thread's (one of 256 threads has the outlier)
        off = bound / 2 + 8 * U32
        size = v[0].abs().max() / torch.sqrt(var + 1e-5)
        limit = want.abs() * (off + half_step(dtype) * 1.01) + 2 * U32 * (1 + size)
        err = (y[n].double() - want).abs()
        assert bool((err <= limit).all()), (n, float((err / limit).max()), float(err.max()))
    assert float(y[3:].abs().max()) == 0.0


# ---------------------------------------------------------------------------------------------- dropout
def test_dropout_module_recomputed_while_capturing_is_refused():
    """A captured mask is drawn on the device: a recomputation would draw another one than the forward pass used."""
    drop, x = Dropout(0.5).train(), torch.ones(4096, device=DEV, requires_grad=True)
    with torch.no_grad():
        drop(x)
    torch.cuda.synchronize()
    graph, refused = torch.cuda.CUDAGraph(), None
    with torch.cuda.graph(graph):
        y = checkpoint(lambda v: drop(v) * v, x, use_reentrant=False, preserve_rng_state=False)
        try:
            torch.autograd.grad(y.sum(), x)
        except RuntimeError as e:
            refused = str(e)
    assert refused is not None and "recomputed" in refused
    graph.replay()
    torch.cuda.synchronize()
    kept = y.detach() != 0
    assert 1700 < int(kept.sum()) < 2400 and torch.equal(y.detach(), torch.where(kept, 2.0, 0.0))
    with torch.no_grad():
        assert 1700 < int((drop(x) != 0).sum()) < 2400


# ---------------------------------------------------------------------------------------------- what is kept
def _training_calls():
    ids = torch.randint(0, 500, (20000,), generator=torch.Generator().manual_seed(0)).to(DEV)
    table, x = _normal(500, 8).requires_grad_(True), _normal(64, 3000, 8).requires_grad_(True)
    counter = torch.zeros(1, device=DEV, dtype=torch.int64)
    return {"embedding": (lambda: embedding_lookup(ids, table), table),
            "group norm": (lambda: group_norm(x, 2), x),
            "dropout": (lambda: dropout(x, 0.5, seed=1, counter=counter), x)}


@pytest.mark.parametrize("name", ["embedding", "group norm", "dropout"])
def test_second_backward_pass_needs_a_kept_graph(name):
    call, leaf = _training_calls()[name]
    y = call()
    g = torch.ones_like(y)
    first = torch.autograd.grad(y, leaf, g, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(y, leaf, g)[0], first)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, leaf, g)


@pytest.mark.parametrize("name", ["embedding", "group norm"])
def test_what_the_backward_pass_needs_is_let_go_behind_it(name):
    call, leaf = _training_calls()[name]
    y = call()  # keeps the graph
    g = torch.ones_like(y)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    torch.autograd.grad(y, leaf, g)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() < held


@pytest.mark.parametrize("name", ["embedding", "group norm", "dropout"])
def test_what_the_backward_pass_needs_goes_through_saved_tensor_hooks(name):
    call, leaf = _training_calls()[name]
    plain = call()
    want = torch.autograd.grad(plain, leaf, torch.ones_like(plain))[0]
    with torch.autograd.graph.save_on_cpu():
        y = call()
    assert torch.equal(torch.autograd.grad(y, leaf, torch.ones_like(y))[0], want)


def test_dropout_module_masks_repeat_under_a_seed():
    x = torch.ones(4096, device=DEV)
    called = Dropout(0.5).train()
    called(x)  # has a counter from here on
    for module in (Dropout(0.5).train(), called, copy.deepcopy(called)):
        masks = []
        for _ in range(2):
            torch.manual_seed(11)
            masks.append((module(x), module(x), module(x)))
        for a, b in zip(*masks):
            assert torch.equal(a, b)
        assert not torch.equal(masks[0][0], masks[0][1]) and not torch.equal(masks[0][1], masks[0][2])
    torch.manual_seed(11)
    assert torch.equal(copy.deepcopy(called)(x), masks[0][0])
    assert called._counters and not copy.deepcopy(called)._counters


def test_dropout_elements_past_2_34():
    """There the counter's second word, the high one of element index / 4, is no longer zero."""
    behind = 4096 + 8 * 123 + 5
    count = (1 << 34) + behind
    if torch.cuda.mem_get_info()[0] < 2 * count + (8 << 30):
        pytest.skip("needs 42 GB of free device memory")
    x = torch.empty(count, device=DEV, dtype=torch.bfloat16)
    first = (1 << 34) - 4096
    x[first:] = 1.0
    _native.call("dl_dropout", x, x, count, 1, 0.5, 5, 3, None)  # in place
    got = x[first:].float().cpu()
    del x
    q = np.arange(first // 4, (count + 3) // 4, dtype=np.uint64)
    low, high = q & np.uint64(0xFFFFFFFF), q >> np.uint64(32)
    assert high[0] == 0 and high[-1] == 1
    words = philox(np.stack([low, high, np.full_like(q, 3), np.zeros_like(q)], axis=1), (5, 0)).reshape(-1)
    want = torch.from_numpy(np.where(words[:count - first] < 2 ** 31, 0.0, 2.0).astype(np.float32))
    assert torch.equal(got, want)
