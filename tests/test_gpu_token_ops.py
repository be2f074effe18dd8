"""Token-path operators on the GPU against plain 64-bit forms, at the sizes and values where they can go wrong.

Bounds: a rounding to type t is off by at most half a step (eps / 2 relative); fp32 sums of n terms by at most
n * 2^-24 of the sum of absolute terms.
"""

import copy
import math

import numpy as np
import pytest
import torch

from difflut_b200.encoder import EmbeddingEncoder, ThermometerEncoder, embedding_lookup
from difflut_b200.layers import ConvolutionalLayer, ConvolutionConfig, RandomLayer
from difflut_b200.network import DWNNetwork
from difflut_b200.nodes import DWNNode, NodeConfig, ProbabilisticNode
from difflut_b200.utils import Dropout, GroupNorm, GroupSum, dropout, group_norm, sample_logits
from parity_util import close_normwise
from token_util import (TYPES, check, dropped, embedding_grad, half_step, kept_weights, norm_reference, sample_row,
                        smallest)

pytestmark = pytest.mark.gpu
DEV = "cuda"
U32 = 2.0 ** -24


def _normal(*shape, dtype=torch.float32, seed=0):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype).to(DEV)


# ---------------------------------------------------------------------------------------------- dropout
def _check_dropout(y, x, p, seed, offset, what):
    gone = dropped(x.numel(), p, seed, offset).view(x.shape)
    scale = 1.0 / (1.0 - p) if p < 1.0 else 0.0
    ref = torch.where(gone, torch.zeros((), dtype=torch.float64), x.detach().double().cpu() * scale)
    # scale and product are rounded to fp32, the result to the type
    check(y, ref, ref.abs() * (half_step(x.dtype) + 2 * U32 * 1.01) + smallest(x.dtype), what)
    assert bool((y.detach().cpu()[gone] == 0).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("numel", [1, 3, 4, 5, 31, 255, 2048, 2049, 4096 + 7, 100003])
def test_dropout_forward_and_gradient(dtype, numel):
    x = _normal(numel, dtype=dtype, seed=numel).requires_grad_(True)
    seed, offset = 0x1234567890ABCDEF, (3 << 32) + 5
    y = dropout(x, 0.3, seed=seed, offset=offset)
    _check_dropout(y, x, 0.3, seed, offset, "forward")
    g = _normal(numel, dtype=dtype, seed=numel + 1)
    (gx,) = torch.autograd.grad(y, x, g)
    _check_dropout(gx, g, 0.3, seed, offset, "gradient")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shift", [1, 2, 3, 5])
def test_dropout_at_any_alignment(dtype, shift):
    """The mask belongs to the element's index in the tensor, not to its address."""
    x = _normal(1000 + shift, dtype=dtype)[shift:]
    _check_dropout(dropout(x, 0.5, seed=9), x, 0.5, 9, 0, "shifted")


@pytest.mark.parametrize("p", [0.0, 2.0 ** -34, 1e-9, 0.999999, 1.0 - 2.0 ** -40, 1.0])
def test_dropout_extreme_probabilities(p):
    x = _normal(4099).requires_grad_(True)
    y = dropout(x, p, seed=1)
    _check_dropout(y, x, p, 1, 0, f"p={p}")
    (gx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    _check_dropout(gx, torch.ones(4099), p, 1, 0, f"gradient p={p}")


def test_dropout_of_values_that_are_not_numbers():
    """Dropped positions are exactly 0 whatever they held; kept ones keep infinities and NaN."""
    x = torch.tensor([float("inf"), float("-inf"), float("nan"), 1.0], device=DEV).repeat(256)
    y = dropout(x, 0.5, seed=3).cpu()
    gone = dropped(1024, 0.5, 3, 0)
    assert bool((y[gone] == 0).all())
    kept = torch.tensor([float("inf"), float("-inf"), float("nan"), 2.0]).repeat(256)[~gone]
    assert torch.equal(torch.nan_to_num(y[~gone], nan=7.0), torch.nan_to_num(kept, nan=7.0))


def test_dropout_strides_and_empty():
    x = _normal(64, 48)
    _check_dropout(dropout(x.t(), 0.25, seed=2), x.t().contiguous(), 0.25, 2, 0, "transposed")
    e = torch.empty(0, 5, device=DEV, requires_grad=True)
    assert torch.autograd.grad(dropout(e, 0.5), e, e.detach())[0].shape == (0, 5)
    xg = x.clone().requires_grad_(True)  # an expanded gradient
    (gx,) = torch.autograd.grad(dropout(xg, 0.25, seed=2).sum(), xg)
    _check_dropout(gx, torch.ones(64, 48), 0.25, 2, 0, "expanded gradient")


def test_dropout_second_derivative_is_the_same_mask():
    x = _normal(500).requires_grad_(True)
    (gx,) = torch.autograd.grad(dropout(x, 0.5, seed=4).pow(2).sum(), x, create_graph=True)
    (gg,) = torch.autograd.grad(gx.sum(), x)
    gone = dropped(500, 0.5, 4, 0)
    assert torch.equal(gg.cpu(), torch.where(gone, 0.0, 8.0))


def test_dropout_word_index_past_32_bits():
    """The high counter word: elements from 2^34 on take other words than the ones 2^34 below (bytes would be 32 GB, so
    the counter is moved instead: the offset's words sit beside it in the same block)."""
    x = torch.ones(4096, device=DEV)
    a, b = dropout(x, 0.5, seed=5, offset=1), dropout(x, 0.5, seed=5, offset=1 << 32)
    assert not torch.equal(a, b)
    _check_dropout(b, x, 0.5, 5, 1 << 32, "high offset")


def test_dropout_counter_on_the_device():
    x = _normal(4096).requires_grad_(True)
    counter = torch.tensor([7], device=DEV, dtype=torch.int64)
    y = dropout(x, 0.5, seed=6, offset=10, counter=counter)
    _check_dropout(y, x, 0.5, 6, 17, "counter")
    (gx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    _check_dropout(gx, torch.ones(4096), 0.5, 6, 17, "counter gradient")
    with pytest.raises(TypeError):
        dropout(x, 0.5, counter=counter.int())
    z = dropout(x, 0.5, seed=6, counter=counter)
    counter.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(z, x, torch.ones_like(z))


def test_dropout_module_draws_a_mask_per_call_and_repeats_under_a_seed():
    d, x = Dropout(0.5).train(), torch.ones(4096, device=DEV)
    torch.manual_seed(11)
    a, b = d(x), d(x)
    assert not torch.equal(a, b)
    torch.manual_seed(11)
    e = copy.deepcopy(Dropout(0.5).train())
    first = e(x)  # also creates the counter, from a draw of its own
    assert 0.4 < float((a == 0).float().mean()) < 0.6 and 0.4 < float((first == 0).float().mean()) < 0.6


def test_dropout_module_in_a_captured_graph_draws_a_mask_per_replay():
    d, x = Dropout(0.5).train(), torch.ones(4096, device=DEV, requires_grad=True)
    fresh = Dropout(0.5).train()
    d(x)
    with torch.no_grad():
        fresh_error = None
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        try:
            fresh(x)
        except RuntimeError as e:
            fresh_error = str(e)
        y = d(x)
        (gx,) = torch.autograd.grad(y, x, torch.ones_like(y))
    assert "before capturing" in fresh_error
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal((y == 0), (gx == 0))
        seen.append(y.detach().clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_dropout_module_in_a_checkpointed_block_recomputes_its_mask():
    from torch.utils.checkpoint import checkpoint

    drop = Dropout(0.5).train()
    x = torch.full((4096,), 3.0, device=DEV, requires_grad=True)
    y = checkpoint(lambda v: drop(v) * v, x, use_reentrant=False)
    kept = y.detach() != 0
    (g,) = torch.autograd.grad(y.sum(), x)
    assert 1700 < int(kept.sum()) < 2400 and torch.equal(g, torch.where(kept, 12.0, 0.0))


def test_dropout_on_another_stream():
    x = _normal(1 << 20)
    want = dropout(x, 0.5, seed=8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = dropout(x, 0.5, seed=8)
    s.synchronize()
    assert torch.equal(got, want)


# ---------------------------------------------------------------------------------------------- embedding
def _ids(T, V, seed, kind="zipf"):
    g = torch.Generator().manual_seed(seed)
    if kind == "one":
        return torch.full((T,), V // 2)
    if kind == "runs":  # segments of many lengths
        return (torch.arange(T) * torch.arange(T) // max(1, T)) % V
    u = torch.rand(T, generator=g, dtype=torch.float64)
    if kind == "uniform":
        return (u * V).long()
    return (torch.exp(u * torch.log(torch.tensor(V + 1.0, dtype=torch.float64))) - 1).long().clamp(0, V - 1)


def _check_embedding(T, V, D, dtype, kind="zipf", scale=1.7, padding=None, ids=None, ids_dtype=torch.int64):
    ids = (_ids(T, V, T + V, kind) if ids is None else ids).to(ids_dtype).to(DEV)
    W = _normal(V, D, dtype=dtype, seed=1).requires_grad_(True)
    g = _normal(*ids.shape, D, dtype=dtype, seed=2)
    s32 = float(torch.tensor(scale, dtype=torch.float32))
    out = embedding_lookup(ids, W, scale=scale, padding_idx=padding)
    ok = (ids >= 0) & (ids < V)
    ref = W.detach().double()[torch.where(ok, ids, 0).long()] * s32
    check(out[ok], ref[ok], ref[ok].abs().cpu() * (half_step(dtype) + U32 * 1.01) + smallest(dtype), "lookup")
    assert bool(torch.isnan(out[~ok]).all())
    (gW,) = torch.autograd.grad(out, W, g)
    want, size, n = embedding_grad(ids, g, V, s32, padding)
    # n additions and one product in fp32, then the rounding to the type
    check(gW, want, size * (n + 1) * U32 * 1.01 + want.abs() * half_step(dtype) * 1.01 + smallest(dtype), "table gradient")
    assert bool((gW.cpu()[(n == 0).reshape(-1)] == 0).all())
    return ids, W, g, gW


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T,V,D", [(1, 1, 1), (1, 7, 8), (2, 300, 3), (33, 5, 16), (257, 1000, 36), (1000, 255, 130),
                                   (1000, 256, 64), (5000, 65535, 24), (700, 40, 515), (37, 10, 1100)])
def test_embedding_sizes(T, V, D, dtype):
    _check_embedding(T, V, D, dtype)


@pytest.mark.parametrize("kind", ["one", "runs", "uniform"])
@pytest.mark.parametrize("T", [31, 4096, 4097, 9001, 33000])
def test_embedding_distributions(kind, T):
    """One id for all tokens (a segment over every range), segments of many lengths, and mostly single tokens; one
    sorting block, two, and the whole cluster with several tiles per block."""
    _check_embedding(T, 700, 16, torch.float32, kind)


@pytest.mark.parametrize("T", [65536, 65537, 140000])
def test_embedding_more_tokens_than_the_chip_sorts_in_place(T):
    """Up to 65536 tokens stay in distributed shared memory between the passes, more go through the workspace."""
    ids = _ids(T, 300000, 5, "uniform").to(DEV)
    W = torch.zeros(300000, 1, device=DEV, requires_grad=True)
    g = torch.ones(T, 1, device=DEV)
    (gW,) = torch.autograd.grad(embedding_lookup(ids, W), W, g)
    assert torch.equal(gW[:, 0], torch.bincount(ids, minlength=300000).float())


def test_embedding_long_ranges_of_one_id():
    """So many tokens that a range holds more than 32 of them."""
    _check_embedding(60000, 3, 520, torch.bfloat16, "uniform")


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
def test_embedding_ids_that_do_not_exist(ids_dtype):
    """They give NaN rows, take no gradient, and nothing else changes; padding keeps its row and takes none either."""
    ids = torch.tensor([3, -1, 0, 10, 9, 2147483647, -2147483648, 3, 0, 5])
    _check_embedding(0, 10, 12, torch.float32, ids=ids, padding=0, ids_dtype=ids_dtype)
    _check_embedding(0, 10, 12, torch.float32, ids=torch.full((50,), -7), ids_dtype=ids_dtype)
    if ids_dtype == torch.int64:
        _check_embedding(0, 10, 12, torch.float32, ids=torch.tensor([1 << 32, (1 << 32) + 3, 3, -(1 << 40)]))


def test_embedding_no_tokens():
    W = _normal(5, 4).requires_grad_(True)
    out = embedding_lookup(torch.empty(2, 0, device=DEV, dtype=torch.int64), W)
    assert out.shape == (2, 0, 4)
    assert torch.equal(torch.autograd.grad(out, W, out.detach())[0], torch.zeros_like(W))


def test_embedding_strided_inputs_and_shifted_table():
    ids = _ids(600, 50, 3).view(20, 30).t().to(DEV)
    big = _normal(50, 33)
    table = big[:, 1:]  # rows that start at odd offsets
    out = embedding_lookup(ids, table, scale=2.0)
    assert torch.equal(out, table[ids] * 2.0)
    flat = _normal(50 * 16 + 1)
    shifted = flat[1:].view(50, 16)  # contiguous, 4-byte aligned only
    assert torch.equal(embedding_lookup(ids, shifted), shifted[ids])
    W = big.clone().requires_grad_(True)
    (gW,) = torch.autograd.grad(embedding_lookup(ids, W).sum(), W)  # an expanded gradient
    count = torch.bincount(ids.reshape(-1), minlength=50).float()
    assert torch.equal(gW, count[:, None].expand(50, 33))


@pytest.mark.parametrize("dtype", TYPES)
def test_embedding_gradient_is_the_same_on_every_run(dtype):
    ids, W, g, first = _check_embedding(20000, 900, 72, dtype)
    for _ in range(3):
        (again,) = torch.autograd.grad(embedding_lookup(ids, W, scale=1.7), W, g)
        assert torch.equal(first, again)


def test_embedding_gradient_against_differences():
    """The lookup is linear in the table: a step in one entry moves the loss by gradient * step exactly."""
    ids = _ids(200, 30, 1).to(DEV)
    W = (_normal(30, 8) * 8).round().requires_grad_(True)
    g = (_normal(200, 8, seed=3) * 8).round()
    (gW,) = torch.autograd.grad(embedding_lookup(ids, W, scale=0.5), W, g)
    with torch.no_grad():
        base = (embedding_lookup(ids, W, scale=0.5).double() * g).sum()
        for v, d in ((0, 0), (3, 5), (29, 7)):
            W2 = W.clone()
            W2[v, d] += 1.0
            assert float((embedding_lookup(ids, W2, scale=0.5).double() * g).sum() - base) == float(gW[v, d])


def test_embedding_captured_and_replayed():
    ids, W = _ids(3000, 400, 5).to(DEV), _normal(400, 40).requires_grad_(True)
    g = _normal(3000, 40, seed=6)

    def step():
        out = embedding_lookup(ids, W, scale=1.5)
        return out, torch.autograd.grad(out, W, g)[0]

    want = [t.detach().clone() for t in step()]
    torch.cuda.synchronize()
    graphs, results = [], []
    for _ in range(2):  # two graphs, each with a workspace of its own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step())
        graphs.append(graph)
    for graph in graphs + graphs:
        graph.replay()
    torch.cuda.synchronize()
    for out, gW in results:
        assert torch.equal(out, want[0]) and torch.equal(gW, want[1])
    ids.copy_(ids.flip(0))  # new ids in place: the replay reads them
    new = [t.detach().clone() for t in step()]
    graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(results[0][0], new[0]) and torch.equal(results[0][1], new[1])


def test_embedding_two_streams_at_once():
    ids, W = _ids(20000, 4000, 5).to(DEV), _normal(4000, 64).requires_grad_(True)
    g = _normal(20000, 64, seed=6)
    want = torch.autograd.grad(embedding_lookup(ids, W), W, g)[0]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            got.append(torch.autograd.grad(embedding_lookup(ids, W), W, g)[0])
    torch.cuda.synchronize()
    for x in got:
        assert torch.equal(x, want)


def test_embedding_encoder_trains():
    enc = EmbeddingEncoder(20, num_bits=6, scale=3.0, padding_idx=0).to(DEV)
    ids = torch.randint(0, 20, (5, 7), device=DEV)
    x = enc(ids)
    assert x.shape == (5, 42) and EmbeddingEncoder(20, num_bits=6, flatten=False).to(DEV)(ids).shape == (5, 7, 6)
    assert enc(ids[0]).shape == (42,)
    x.sum().backward()
    assert float(enc.weight.grad[0].abs().max()) == 0.0 and float(enc.weight.grad[1:].abs().max()) > 0.0


# ---------------------------------------------------------------------------------------------- group norm
def _rounded(pair, dtype):
    ref, bound = pair
    return bound + ref.abs() * half_step(dtype) * 1.01 + smallest(dtype)


def _check_norm(N, S, C, G, dtype, act="silu", affine=True, param_dtype=torch.float32, eps=1e-5, shift=0.0, x=None, seed=0):
    if x is None:
        x = _normal(N, S, C, seed=seed) * 1.5 + _normal(C, seed=seed + 1) + shift
    x = x.to(dtype).requires_grad_(True)
    w = (1 + 0.3 * _normal(C, seed=seed + 2)).to(param_dtype).requires_grad_(True) if affine else None
    b = (0.2 * _normal(C, seed=seed + 3)).to(param_dtype).requires_grad_(True) if affine else None
    g = _normal(N, S, C, seed=seed + 4)
    z = norm_reference(x, G, w, b, eps, act)["z"].to(DEV)
    g = torch.where(z.abs() < 1e-3, 0.0, g).to(dtype) if act == "relu" else g.to(dtype)  # away from relu's corner
    ref = norm_reference(x, G, w, b, eps, act, g)
    y = group_norm(x, G, w, b, eps=eps, activation=act)
    check(y, ref["y"][0], _rounded(ref["y"], dtype), "y")
    with torch.no_grad():
        assert torch.equal(group_norm(x, G, w, b, eps=eps, activation=act), y)
    wanted = [t for t in (x, w, b) if t is not None]
    grads = torch.autograd.grad(y, wanted, g, retain_graph=True)
    check(grads[0], ref["gx"][0], _rounded(ref["gx"], dtype), "gx")
    if affine:
        check(grads[1], ref["gw"][0], _rounded(ref["gw"], param_dtype), "gweight")
        check(grads[2], ref["gb"][0], _rounded(ref["gb"], param_dtype), "gbias")
    for first, again in zip(grads, torch.autograd.grad(y, wanted, g)):
        assert torch.equal(first, again)
    return x, w, b, g, y, grads


NORM_SIZES = [(1, 1, 16, 1), (3, 1, 30, 3), (300, 1, 96, 12), (5, 1, 1024, 32), (700, 1, 64, 2), (9, 1, 513, 9), (4, 1, 2048, 2),
              (2, 7, 12, 4), (2, 100, 6, 6), (3, 65, 40, 4), (2, 576, 32, 8), (1, 1517, 120, 12), (2, 333, 8, 8),
              (1, 4097, 64, 4), (2, 50, 1000, 1), (1, 3, 1, 1), (1, 40, 3, 1), (2, 19, 1030, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N,S,C,G", NORM_SIZES)
def test_group_norm_sizes(N, S, C, G, dtype):
    _check_norm(N, S, C, G, dtype, seed=N + S + C)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "sigmoid"])
@pytest.mark.parametrize("N,S,C,G", [(64, 1, 128, 8), (3, 130, 48, 6)])
def test_group_norm_activations(N, S, C, G, act):
    for dtype in TYPES:
        _check_norm(N, S, C, G, dtype, act=act)
        _check_norm(N, S, C, G, dtype, act=act, affine=False)
        _check_norm(N, S, C, G, dtype, act=act, param_dtype=dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,S,C,G", [
    (1, 9000, 64, 2),       # a sample over many chunks of rows
    (1, 30000, 128, 1),     # and more of them
    (2, 3, 8192, 1),        # a group over several blocks of channels
    (1, 2, 5000, 1),        # the same with lanes left over
    (3, 1, 9001, 1),        # and without positions
    (1, 40, 12000, 1),      # chunks and blocks of channels
    (600, 3, 64, 4),        # samples enough: one launch
    (2, 70, 2080, 65),      # the last block of channels has fewer groups
])
def test_group_norm_large_units(N, S, C, G, dtype):
    _check_norm(N, S, C, G, dtype, act="sigmoid")


@pytest.mark.parametrize("S", [1, 37, 5000])
def test_group_norm_far_from_zero(S):
    """A mean a thousand times the spread: squares are taken around the mean."""
    _check_norm(3, S, 32, 2, torch.float32, shift=1500.0)


def test_group_norm_constant_group():
    """No spread at all: the output is act(bias), the gradient is finite."""
    x = torch.full((2, 33, 16), 3.0, device=DEV)
    _check_norm(2, 33, 16, 4, torch.float32, x=x)
    _check_norm(2, 1, 16, 4, torch.float32, x=x[:, :1].contiguous())


@pytest.mark.parametrize("S", [1, 50])
def test_group_norm_values_that_are_not_numbers_stay_in_their_group(S):
    x = _normal(4, S, 32)
    x[1, 0, 3], x[2, S - 1, 20] = float("nan"), float("inf")
    want = torch.nn.functional.group_norm(x.transpose(1, 2).double(), 4).transpose(1, 2)
    y = group_norm(x, 4)
    assert torch.equal(torch.isnan(y), torch.isnan(want))
    ok = ~torch.isnan(want)
    assert float((y[ok] - want[ok]).abs().max()) < 1e-5
    clean = group_norm(torch.nan_to_num(x, nan=0.0, posinf=0.0), 4)
    assert torch.equal(y[0], clean[0]) and torch.equal(y[3], clean[3])


@pytest.mark.parametrize("dtype", TYPES)
def test_group_norm_alignment_and_strides(dtype):
    flat = _normal(2 * 50 * 24 + 1, dtype=dtype)
    shifted, plain = flat[1:].view(2, 50, 24), flat[1:].clone().view(2, 50, 24)
    a, b = group_norm(shifted, 3, activation="silu"), group_norm(plain, 3, activation="silu")
    assert float((a.float() - b.float()).abs().max()) <= 4 * half_step(dtype) * float(b.float().abs().max())
    strided = _normal(2, 24, 50, dtype=dtype).transpose(1, 2)
    assert torch.equal(group_norm(strided, 3), group_norm(strided.contiguous(), 3))
    x = plain.float().requires_grad_(True)  # an expanded gradient
    (gx,) = torch.autograd.grad(group_norm(x, 3).sum(), x)
    assert float(gx.abs().max()) < 1e-4  # a constant on every element of a group has no effect


def test_group_norm_gradient_against_differences():
    x = _normal(2, 9, 12).requires_grad_(True)
    w, b = (1 + 0.1 * _normal(12, seed=1)).requires_grad_(True), _normal(12, seed=2).requires_grad_(True)
    g = _normal(2, 9, 12, seed=3)
    grads = torch.autograd.grad(group_norm(x, 3, w, b, activation="sigmoid"), (x, w, b), g)
    for t, grad in zip((x, w, b), grads):
        d = _normal(*t.shape, seed=7)
        h = 1e-2
        with torch.no_grad():
            def loss(step):
                args = [v + step * d if v is t else v for v in (x, w, b)]
                return (group_norm(args[0], 3, args[1], args[2], activation="sigmoid").double() * g).sum()
            # fourth-order differences: error h^4 times the fifth derivative (below 10) plus rounding / h
            slope = (8 * (loss(h) - loss(-h)) - (loss(2 * h) - loss(-2 * h))) / (12 * h)
        want = float((grad.double() * d).sum())
        assert abs(float(slope) - want) <= 2e-3 * max(1.0, abs(want))


def test_group_norm_empty_batch():
    x = torch.empty(0, 5, 8, device=DEV, requires_grad=True)
    w = torch.ones(8, device=DEV, requires_grad=True)
    gx, gw = torch.autograd.grad(group_norm(x, 2, w), (x, w), torch.empty(0, 5, 8, device=DEV))
    assert gx.shape == (0, 5, 8) and torch.equal(gw, torch.zeros_like(w))
    with pytest.raises(ValueError, match="position"):
        group_norm(torch.empty(2, 0, 8, device=DEV), 2)


def test_group_norm_partial_gradients():
    x, w, b = _normal(3, 20, 16), torch.ones(16, device=DEV, requires_grad=True), torch.zeros(16, device=DEV)
    (gw,) = torch.autograd.grad(group_norm(x, 4, w, b, activation="silu").sum(), w)
    xg, bg = x.clone().requires_grad_(True), b.clone().requires_grad_(True)
    both = torch.autograd.grad(group_norm(xg, 4, w, bg, activation="silu").sum(), (xg, w, bg))
    assert torch.equal(gw, both[1])
    (gx,) = torch.autograd.grad(group_norm(xg, 4, w.detach(), b, activation="silu").sum(), xg)
    assert torch.equal(gx, both[0])


def test_group_norm_captured_and_replayed():
    x, w, b = (t.requires_grad_(True) for t in (_normal(4, 700, 64), _normal(64, seed=1), _normal(64, seed=2)))
    g = _normal(4, 700, 64, seed=3)

    def step():
        y = group_norm(x, 8, w, b, activation="silu")
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), g)

    want = step()
    torch.cuda.synchronize()
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            results.append(step())
        graphs.append(graph)
    for graph in graphs + graphs:
        graph.replay()
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_group_norm_streams_at_once():
    x, g = _normal(8, 2000, 64).requires_grad_(True), _normal(8, 2000, 64, seed=1)
    want = torch.autograd.grad(group_norm(x, 4), x, g)[0]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        with torch.cuda.stream(torch.cuda.Stream()):
            got.append(torch.autograd.grad(group_norm(x, 4), x, g)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in got)


def test_group_norm_module_behind_a_convolutional_layer():
    """(B, C, H, W) over the layer's channels-last memory: no copy in, the same view out."""
    torch.manual_seed(0)
    conv = ConvolutionalLayer(ConvolutionConfig(tree_depth=1, in_channels=2, out_channels=8, receptive_field=3),
                              ProbabilisticNode, NodeConfig(input_dim=4, output_dim=1), RandomLayer,
                              n_inputs_per_node=4, flip_probability=0.0).to(DEV)
    norm = GroupNorm(2, 8, activation="sigmoid", channel_dim=1).to(DEV)
    h = conv(torch.rand(3, 2, 9, 9, device=DEV))
    assert h.movedim(1, -1).is_contiguous()
    y = norm(h)
    want = torch.sigmoid(torch.nn.functional.group_norm(h.detach().double(), 2))
    assert y.shape == h.shape and y.movedim(1, -1).is_contiguous()
    assert float((y - want).abs().max()) < 1e-5
    y.square().sum().backward()
    assert float(norm.weight.grad.abs().max()) > 0 and float(conv.first_layer_chunks[0].raw_weights.grad.abs().max()) > 0
    rows = GroupNorm(2, 8).to(DEV)
    assert rows(torch.rand(5, 8, device=DEV)).shape == (5, 8)


# ---------------------------------------------------------------------------------------------- sampling
def _check_samples(x, u, T=1.0, k=0, p=1.0, m=0.0):
    """Every id equals the plain 64-bit form's, with numbers or per-row tensors as settings."""
    got = sample_logits(x, u, temperature=T, top_k=k, top_p=p, min_p=m).cpu().tolist()
    rows, us = x.double().cpu().numpy(), u.double().cpu().numpy()
    per = [v.cpu().tolist() if isinstance(v, torch.Tensor) else [v] * len(rows) for v in (T, k, p, m)]
    want = [sample_row(rows[r], us[r], *(v[r] for v in per)) for r in range(len(rows))]
    assert got == want, [(r, a, b) for r, (a, b) in enumerate(zip(got, want)) if a != b][:5]
    return got


def _logits(R, V, dtype, seed=0, spread=2.5):
    x = _normal(R, V, seed=seed) * spread
    g = torch.Generator().manual_seed(seed + 1)
    return (x + 6.0 * (torch.rand(R, V, generator=g) < min(0.5, 4.0 / V)).to(DEV)).to(dtype)


def _u(R, seed=0):
    return torch.rand(R, generator=torch.Generator().manual_seed(seed + 77)).to(DEV)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (0.8, 50, 0.95, 0.02),
            (0.0, 0, 1.0, 0.0), (1.0, 1, 0.5, 0.5), (2.0, 3, 0.3, 0.0), (1.0, 1000, 0.999, 0.0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 3, 31, 32, 33, 64, 65, 200, 256, 257, 511, 512, 513, 1000, 4097, 8192, 16384, 40003])
def test_sampling_sizes(V, dtype):
    R = 24 if V < 5000 else 6
    for i, (T, k, p, m) in enumerate(SETTINGS):
        _check_samples(_logits(R, V, dtype, seed=V + i), _u(R, i), T, k, p, m)


@pytest.mark.parametrize("R,V", [(1, 131072), (700, 700), (1, 600), (130, 9000)])
def test_sampling_rows_and_clusters(R, V):
    """One row over the largest cluster, many rows over one block each."""
    for i, (T, k, p, m) in enumerate(SETTINGS[:5]):
        _check_samples(_logits(R, V, torch.float32, seed=i), _u(R, i), T, k, p, m)


@pytest.mark.parametrize("V", [5, 300, 513, 3000, 30000])
@pytest.mark.parametrize("levels", [1, 2, 7])
def test_sampling_equal_logits(V, levels):
    """Few distinct values: the cuts fall inside runs of equal logits and go by index."""
    x = torch.randint(0, levels, (8, V), generator=torch.Generator().manual_seed(V)).float().to(DEV)
    for i, (T, k, p, m) in enumerate([(1.0, 0, 1.0, 0.0), (1.0, 3, 1.0, 0.0), (1.0, V // 2, 1.0, 0.0), (1.0, 0, 0.31, 0.0),
                                      (0.5, V // 3, 0.77, 0.0), (1.0, 0, 0.6, 0.5), (0.0, 0, 1.0, 0.0), (1.0, 0, 1.0, 1.0)]):
        _check_samples(x, _u(8, i), T, k, p, m)


@pytest.mark.parametrize("V", [400, 3000, 30000])
@pytest.mark.parametrize("spread", [1e-3, 1e-6, 1e-30])
def test_sampling_logits_close_together(V, spread):
    """All logits within one step of the histogram: their keys are narrowed down bit by bit."""
    x = _normal(6, V, seed=V) * spread
    x[3] += 8.0  # here most of them become equal
    x[4, ::2] *= -1e-8
    for i, (T, k, p, m) in enumerate([(1.0, V // 3, 1.0, 0.0), (1.0, 0, 0.4, 0.0), (0.9, V // 2, 0.9, 0.0), (1.0, 0, 1.0, 0.0)]):
        _check_samples(x, _u(6, i), T, k, p, m)


@pytest.mark.parametrize("V", [7, 300, 2000, 20000])
def test_sampling_masked_and_extreme_logits(V):
    low, big = torch.finfo(torch.float32).min, 3.0e38
    x = _logits(12, V, torch.float32, seed=V)
    x[0] = -math.inf                       # nothing left
    x[1] = math.nan
    x[2, 1:] = -math.inf                   # one left
    x[3, : V - 1] = low                    # masked by the type's lowest value
    x[4] = low                             # every logit is that value
    x[5, ::2] = math.nan
    x[6, V // 2] = math.inf
    x[7, ::3] = math.inf
    x[8, 0], x[8, V - 1] = big, -big
    x[9, ::2] = 0.0
    x[9, 1::2] = -0.0
    x[10] = -math.inf
    x[10, V - 1] = -5.0
    x[11, : V // 2] = -math.inf
    for i, (T, k, p, m) in enumerate(SETTINGS):
        got = _check_samples(x, _u(12, i), T, k, p, m)
        assert got[0] == got[1] == -1 and got[2] == 0 and got[10] == V - 1


@pytest.mark.parametrize("V", [200, 3000])
@pytest.mark.parametrize("T", [1e-30, 1e-3, 50.0, 1e30, math.inf, 5e-324])
def test_sampling_extreme_temperatures(V, T):
    x, u = _logits(10, V, torch.float32), _u(10)
    if T == 5e-324:  # 1 / T is not a number of the type: the largest logit
        assert sample_logits(x, u, temperature=T).tolist() == x.argmax(1).tolist()
        return
    for k, p in ((0, 1.0), (20, 1.0), (0, 0.9), (20, 0.5)):
        _check_samples(x, u, T, k, p)


@pytest.mark.parametrize("V", [300, 3000, 40000])
def test_sampling_logits_of_any_size(V):
    """Differences beyond the type's range, weighed by a temperature as large."""
    x = (_normal(8, V) * 1e38).clamp(-3.4e38, 3.4e38)
    for T in (1.0, 1e37, 1e38, 3e38):
        for k, p in ((0, 1.0), (20, 1.0), (2000, 0.9), (0, 0.9), (20, 0.5)):
            _check_samples(x, _u(8), T, k, p)


@pytest.mark.parametrize("V", [300, 3000])
def test_sampling_ends_of_the_random_numbers(V):
    """u = 0 takes the first kept class, the largest u below 1 the last; numbers outside [0, 1) and NaN are pulled in."""
    x = _logits(6, V, torch.float32)
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 7.0, -1.0, math.nan], device=DEV)
    got = sample_logits(x, u, top_p=0.9).tolist()
    for r, (id, first) in enumerate(zip(got, (True, False, False, False, True, True))):
        ids, w = kept_weights(x[r].cpu().numpy(), p=0.9)
        assert id == (ids[0] if first else ids[-1])
    u64 = torch.tensor([1.0 - 2.0 ** -53, 2.0 ** -60] * 3, device=DEV, dtype=torch.float64)
    _check_samples(x, u64, 1.0, 0, 0.9)


@pytest.mark.parametrize("V", [100, 2000])
def test_sampling_settings_per_row(V):
    R = 40
    x, u = _logits(R, V, torch.bfloat16), _u(R)
    i = torch.arange(R, device=DEV)
    T = torch.where(i % 5 == 3, 0.0, 0.5 + 0.1 * (i % 7)).float()
    k = torch.where(i % 4 == 1, 0, 1 + i * 3).int()
    p = torch.where(i % 3 == 2, 1.0, 0.3 + 0.015 * i).float()
    m = torch.where(i % 6 == 0, 0.1, 0.0).float()
    _check_samples(x, u, T, k, p, m)
    # what numbers may not be, per row: not positive temperatures and counts, shares outside (0, 1], ratios outside [0, 1]
    T[0], k[1], p[2], p[3], m[4], m[5] = -1.0, -5, 0.0, 2.0, 3.0, -1.0
    got = sample_logits(x, u, temperature=T, top_k=k, top_p=p, min_p=m).tolist()
    rows = x.double().cpu().numpy()
    for r in range(R):
        a = [float(v[r]) for v in (T, k, p, m)]
        a[2] = 1e-12 if a[2] <= 0 else a[2]
        assert got[r] == sample_row(rows[r], float(u[r]), a[0], max(int(a[1]), 0), a[2], min(max(a[3], 0.0), 1.0))
    assert sample_logits(x, u, temperature=T.double(), top_k=k.long(), top_p=p, min_p=m).tolist() == got


@pytest.mark.parametrize("V", [300, 2000])
def test_sampling_settings_per_row_far_outside_their_range(V):
    """A share far below 0 keeps the first class like 0 does, a count past 32 bits keeps all."""
    x, u = _logits(4, V, torch.float32), _u(4)
    p = torch.tensor([-1e9, -3e38, -math.inf, -0.5], device=DEV)
    assert sample_logits(x, u, top_p=p).tolist() == x.argmax(1).tolist()
    k = torch.tensor([2 ** 32 + 1, 2 ** 31, 2 ** 62, -2 ** 40], device=DEV)
    assert sample_logits(x, u, top_k=k).tolist() == sample_logits(x, u).tolist()


@pytest.mark.parametrize("V", [9000, 24600, 70000])
@pytest.mark.parametrize("heavy", [1, 40, 512, 513, 1500, 2047, 2100, 5000, 8800])
def test_sampling_candidates_around_the_lengths_of_the_lists(V, heavy):
    """`heavy` logits stand out: equal ones, ones within a step of the histogram, ones over many steps.  Borders fall among
    them, in lists that hold them in one block, only in several, or not at all."""
    g = torch.Generator().manual_seed(V + heavy)
    x = _normal(3, V, seed=V) - 30.0
    places = torch.stack([torch.randperm(V, generator=g)[:heavy] for _ in range(3)]).to(DEV)
    spread = torch.tensor([0.0, 0.02, 3.0], device=DEV)[:, None]
    x.scatter_(1, places, spread * _normal(3, heavy, seed=heavy))
    for i, (T, k, p, m) in enumerate([(1.0, 0, 0.63, 0.0), (1.0, 0, 0.999, 0.4), (1.0, 0, 1.0, 0.01), (1.0, 1000, 0.7, 0.0),
                                      (1.0, 2048, 1.0, 0.0), (1.0, 2049, 0.9, 0.1), (0.9, 0, 1.0 - 1e-12, 0.0)]):
        _check_samples(x, _u(3, i), T, k, p, m)


@pytest.mark.parametrize("V", [200, 2000, 20000])
def test_sampling_frequencies(V):
    """Random numbers on an even grid: every class comes up as often as its weight says, give or take one at each end."""
    n = 4096
    x = (_normal(1, V, seed=V) * 2).expand(n, V)  # rows at distance zero
    u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).to(DEV)
    got = np.bincount(sample_logits(x, u, temperature=0.8, top_p=0.95).cpu().numpy(), minlength=V)
    ids, w = kept_weights(x[0].cpu().numpy(), 0.8, 0, 0.95)
    want = np.zeros(V)
    want[ids] = w / w.sum() * n
    assert np.abs(got - want).max() <= 1.0 + 1e-6


def test_sampling_strided_rows_and_views():
    big = _logits(10, 900, torch.float32)
    u = _u(10)
    view = big[:, 100:801]  # rows 900 apart, odd start
    assert sample_logits(view, u, top_p=0.9).tolist() == sample_logits(view.contiguous(), u, top_p=0.9).tolist()
    last = big.view(5, 2, 900)[:, -1]
    assert sample_logits(last, u[:5]).tolist() == sample_logits(last.contiguous(), u[:5]).tolist()
    t = big[:, :10].t()
    assert sample_logits(t, u).tolist() == sample_logits(t.contiguous(), u).tolist()
    assert sample_logits(big, u.expand(2, 10).t()[:, 0]).tolist() == sample_logits(big, u).tolist()
    assert sample_logits(big[:0], u[:0]).shape == (0,)


def test_sampling_captured_and_on_streams():
    x, u = _logits(20, 5000, torch.float32), _u(20)
    want = sample_logits(x, u, temperature=0.9, top_k=100, top_p=0.9)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sample_logits(x, u, temperature=0.9, top_k=100, top_p=0.9)
    graph.replay()
    assert torch.equal(got, want)
    u.copy_(_u(20, 5))
    graph.replay()
    assert torch.equal(got, sample_logits(x, u, temperature=0.9, top_k=100, top_p=0.9))
    torch.cuda.synchronize()
    outs = []
    for _ in range(3):
        with torch.cuda.stream(torch.cuda.Stream()):
            outs.append(sample_logits(x, u, temperature=0.9, top_k=100, top_p=0.9))
    torch.cuda.synchronize()
    assert all(torch.equal(o, got) for o in outs)


# ---------------------------------------------------------------------------------------------- all of them together
class _TokenModel(torch.nn.Module):
    """ids (B, T) -> embedding -> group norm + sigmoid -> dropout -> LUT layer -> GroupSum logits (B, k)."""

    def __init__(self, vocabulary, tokens, width, nodes, classes, p):
        super().__init__()
        self.encoder = EmbeddingEncoder(vocabulary, num_bits=width, scale=2.0, padding_idx=0, flatten=False)
        self.norm = GroupNorm(4, width, activation="sigmoid")
        self.dropout = Dropout(p)
        self.layer = RandomLayer(tokens * width, nodes, ProbabilisticNode, NodeConfig(input_dim=4, output_dim=1), seed=3)
        self.head = GroupSum(k=classes, tau=2.0, use_randperm=False)

    def features(self, ids):
        return self.norm(self.encoder(ids)).reshape(ids.shape[0], -1)

    def forward(self, ids, mask=None):
        x = self.features(ids)
        x = self.dropout(x) if mask is None else dropout(x, self.dropout.p, **mask)
        return self.head(self.layer(x))


def _token_model(p=0.25):
    torch.manual_seed(0)
    model = _TokenModel(50, 6, 16, 60, 10, p).to(DEV).train()
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 50, (33, 6), generator=g).to(DEV)
    labels = torch.randint(0, 10, (33,), generator=g).to(DEV)
    return model, ids, labels


def test_token_model_equals_its_plain_form():
    """Logits, loss and every gradient against the same LUT layer behind 64-bit plain forms of the operators."""
    model, ids, labels = _token_model()
    logits = model(ids, dict(seed=11, offset=4))
    loss = torch.nn.functional.cross_entropy(logits, labels)
    loss.backward()
    table = model.encoder.weight.detach().double().requires_grad_(True)
    w, b = (t.detach().double().requires_grad_(True) for t in (model.norm.weight, model.norm.bias))
    x = table[ids] * 2.0
    x = torch.sigmoid(torch.nn.functional.group_norm(x.transpose(1, 2), 4, w, b)).transpose(1, 2).reshape(33, -1)
    gone = dropped(x.numel(), 0.25, 11, 4).view(x.shape).to(DEV)
    x = torch.where(gone, 0.0, x / 0.75).float()
    names = [n for n, _ in model.layer.named_parameters()]
    before = {n: p.grad.clone() for n, p in model.layer.named_parameters()}
    model.layer.zero_grad()
    want = model.head(model.layer(x))
    want_loss = torch.nn.functional.cross_entropy(want, labels)
    want_loss.backward()
    # inputs differ in the last bits of fp32; the layer's outputs are sums of 16 products of four such inputs
    assert float((logits - want).abs().max()) <= 1e-5 * float(want.abs().max())
    assert abs(float(loss - want_loss)) <= 1e-5
    close_normwise(before[names[0]], dict(model.layer.named_parameters())[names[0]].grad, "layer")
    table.grad[0] = 0.0  # padding
    close_normwise(model.encoder.weight.grad, table.grad, "embedding table")
    close_normwise(model.norm.weight.grad, w.grad, "norm weight")
    close_normwise(model.norm.bias.grad, b.grad, "norm bias")


def test_embedding_elements_past_32_bits():
    """The last rows of a table of 2.3e9 elements, and as many tokens' elements as that."""
    V, D = 140001, 16384
    w = torch.zeros(V, D, device=DEV, dtype=torch.bfloat16)
    ids = torch.tensor([V - 1, 0, V - 2, V - 1], device=DEV)
    w[V - 2], w[V - 1] = 2.0, 3.0
    w.requires_grad_()
    out = embedding_lookup(ids, w, 2.0)
    assert out[:, ::4095].tolist() == [[v] * 5 for v in (6.0, 0.0, 4.0, 6.0)]
    (g,) = torch.autograd.grad(out, w, torch.ones_like(out))
    assert g[[0, 1, V - 3, V - 2, V - 1], 7].tolist() == [2.0, 0.0, 0.0, 2.0, 4.0] and float(g[V - 1].sum()) == 4.0 * D
    assert float(g[1: V - 2: 997].abs().max()) == 0.0
    del w, g, out
    small = _normal(9, D, dtype=torch.bfloat16).requires_grad_()
    ids = torch.arange(V, device=DEV) % 9
    out = embedding_lookup(ids, small)
    assert all(torch.equal(out[t], small[t % 9]) for t in (0, 131071, 131072, V - 1))
    g = torch.zeros_like(out)
    g[V - 1] = 1.0
    (gw,) = torch.autograd.grad(out, small, g)
    assert float(gw[(V - 1) % 9].min()) == 1.0 and float(gw.sum()) == D


def test_group_norm_elements_past_32_bits():
    """Two samples of 1.2e9 values: the second one as if it stood alone (behind a short pass over the first)."""
    S, C, G = 1200001, 1024, 8
    x = torch.zeros(2, S, C, device=DEV, dtype=torch.bfloat16)
    x[1, S - 5000:] = _normal(5000, C, dtype=torch.bfloat16)
    g = torch.zeros_like(x)
    g[1, S - 1] = 1.0
    w = torch.ones(C, device=DEV, requires_grad=True)
    x.requires_grad_()
    y = group_norm(x, G, w)
    tail = x.detach()[1, S - 5000:].double().view(5000, G, -1)
    m = S * (C // G)
    mean = tail.sum(dim=(0, 2)) / m
    var = (tail * tail).sum(dim=(0, 2)) / m - mean * mean
    want = ((tail[-1] - mean[:, None]) * torch.rsqrt(var + 1e-5)[:, None]).reshape(-1)
    got = y.detach()[1, S - 1].double()
    # one rounding to bf16's 8 significant bits (half a step is up to 2^-8 of the value: eps = 2^-7), and the statistics'
    # fp32 sums: a thread adds up some 16000 values of a chunk, each addition off by 2^-24 of the sum at most: 2^-10 of the
    # variance, 2^-11 of its root, and as much again for the mean and what joins the chunks
    rounding = half_step(torch.bfloat16) + 2.0 ** -10
    assert bool(((got - want).abs() <= want.abs() * rounding + 1e-5).all())
    assert float(y.detach()[0].abs().max()) == 0.0
    gx, gw = torch.autograd.grad(y, (x, w), g)
    assert bool(((gw.double() - want).abs() <= want.abs() * 2.0 ** -10 + 1e-5).all())
    rstd = torch.rsqrt(var + 1e-5)[:, None]
    xh = (tail[-1] - mean[:, None]) * rstd
    s2 = xh.sum(dim=1, keepdim=True) / m
    last = (rstd * (1.0 - (C // G) / m - xh * s2)).reshape(-1)
    assert bool(((gx[1, S - 1].double() - last).abs() <= last.abs() * rounding).all())


def test_sampling_rows_past_32_bits():
    R, V = 70001, 32768
    x = torch.full((R, V), -40.0, device=DEV, dtype=torch.bfloat16)
    hot = (torch.arange(R, device=DEV) * 7919) % V
    x[torch.arange(R, device=DEV), hot] = 10.0
    u = torch.rand(R, device=DEV, generator=torch.Generator(DEV).manual_seed(1))
    for kw in ({"temperature": 0.0}, {"top_p": 0.9}, {"top_k": 5, "min_p": 0.5}):
        assert torch.equal(sample_logits(x, u, **kw), hot)


def test_token_block_recomputed_expanded_and_repeated():
    """The same gradients with checkpointing, from an expanded gradient of the output, and a second time from a kept graph."""
    from torch.utils.checkpoint import checkpoint

    emb = EmbeddingEncoder(50, num_bits=16, padding_idx=3, flatten=False).to(DEV)
    norm, drop = GroupNorm(4, 16, activation="silu").to(DEV), Dropout(0.25).train()
    ids = torch.randint(0, 50, (6, 40), generator=torch.Generator().manual_seed(5)).to(DEV)
    leaves = [emb.weight, norm.weight, norm.bias]

    def block(ids):
        return drop(norm(emb(ids)))

    def grads(y, g, **kwargs):
        return torch.autograd.grad(y, leaves, g, **kwargs)

    g = torch.full((1, 1, 1), 0.5, device=DEV).expand(6, 40, 16)
    torch.manual_seed(11)
    y = block(ids)
    want = grads(y, g.contiguous(), retain_graph=True)
    assert all(float(w.abs().max()) > 0 for w in want) and float(want[0][3].abs().max()) == 0.0
    again, expanded = grads(y, g.contiguous(), retain_graph=True), grads(y, g)
    torch.manual_seed(11)
    recomputed = checkpoint(block, ids, use_reentrant=False)
    assert torch.equal(recomputed, y)
    for other in (again, expanded, grads(recomputed, g)):
        assert all(torch.equal(a, b) for a, b in zip(want, other))


def test_token_model_trains_captured_and_samples():
    """A captured step draws a new mask per replay and moves the parameters; ids are then sampled from the logits."""
    model, ids, labels = _token_model(p=0.5)
    optimizer = torch.optim.SGD(model.parameters(), lr=0.5)

    def step():
        optimizer.zero_grad(set_to_none=True)
        loss = torch.nn.functional.cross_entropy(model(ids), labels)
        loss.backward()
        optimizer.step()
        return loss.detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = step()
    start = [p.detach().clone() for p in model.parameters()]
    losses = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        losses.append(float(loss))
    assert len(set(losses)) == 3 and all(math.isfinite(v) for v in losses)
    assert all(not torch.equal(a, p) for a, p in zip(start, model.parameters()))
    model.eval()
    with torch.no_grad():
        assert model.dropout(ids) is ids
        logits = model.head(model.layer(model.features(ids)))
    _check_samples(logits, _u(33), 0.5, 4, 0.9)


def test_network_samples_from_its_logits():
    x = torch.rand(300, 12, generator=torch.Generator().manual_seed(0))
    enc = ThermometerEncoder(num_bits=4).fit(x)
    layers = [RandomLayer(48, 40, DWNNode, NodeConfig(input_dim=6, output_dim=1), seed=0).to(DEV),
              RandomLayer(40, 30, DWNNode, NodeConfig(input_dim=6, output_dim=1), seed=1).to(DEV)]
    net = DWNNetwork(enc, layers, GroupSum(k=10, tau=1.0, use_randperm=False))
    x, u = x.to(DEV), _u(300)
    logits = net.logits(x)
    assert torch.equal(net.sample(x, u, temperature=0.7, top_k=3), sample_logits(logits, u, temperature=0.7, top_k=3))
    assert torch.equal(net.sample(x, temperature=0.0), logits.argmax(dim=1))
    ids = net.sample(x)
    assert ids.shape == (300,) and int(ids.min()) >= 0 and int(ids.max()) < 10
