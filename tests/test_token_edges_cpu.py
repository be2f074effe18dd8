"""Calls of the token path that the documentation allows, at its edges, without a GPU.

Where a call would launch, the launches are replaced by functions that do nothing: what is looked at here is which
calls are refused, what autograd is told and what reaches the entry points.
"""

import contextlib
import subprocess
import sys

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch.utils.checkpoint import checkpoint

from difflut_b200 import _native
from difflut_b200.build import LIB_PATH
from difflut_b200.encoder import EmbeddingEncoder, embedding_lookup
from difflut_b200.network import DWNNetwork
from difflut_b200.utils import Dropout, GroupSum, dropout, group_norm
from difflut_b200.utils import sampling


@pytest.fixture
def no_launches(monkeypatch):
    """CPU tensors pass and nothing is launched; yields the names of the entry points called."""
    called = []

    def entry(name):
        return lambda *args: called.append(name)

    monkeypatch.setattr(_native, "require_cuda", lambda what, *tensors: None)
    monkeypatch.setattr(_native, "entry", entry)
    monkeypatch.setattr(_native, "call", lambda name, *args, **kwargs: called.append(name))
    monkeypatch.setattr(_native, "device_of", lambda t: contextlib.nullcontext())
    yield called


# ---------------------------------------------------------------------------------------------- sampling
@pytest.mark.parametrize("dtype", [torch.int64, torch.uint64, torch.uint32])
def test_top_k_per_row_of_any_size_keeps_its_meaning(dtype):
    """A count that is not positive or not below the number of classes keeps all, also past the 32 bits of the kernel."""
    counts = {torch.int64: [-2 ** 32 + 5, -2 ** 33 + 1, -2 ** 31 - 1, -2 ** 63, -1, 0, 3, 2 ** 31, 2 ** 32 + 2, 2 ** 63 - 1],
              torch.uint64: [0, 3, 2 ** 31, 2 ** 32 + 2, 2 ** 63, 2 ** 64 - 3],
              torch.uint32: [0, 3, 2 ** 31, 2 ** 32 - 2]}[dtype]
    rows, scalar = sampling._setting("top_k", torch.tensor(counts, dtype=dtype), len(counts), torch.int32, 0, 2 ** 62)
    assert scalar is None and rows.dtype == torch.int32
    V = 1 << 29  # more classes than this are refused
    for count, row in zip(counts, rows.tolist()):
        assert (row if 0 < row < V else 0) == (count if 0 < count < V else 0), (count, row)


# ---------------------------------------------------------------------------------------------- group norm
@pytest.mark.parametrize("S", [1, 2, 1000])
@pytest.mark.parametrize("C,G", [(8, 2), (1024, 1), (64, 64), (1, 1)])
def test_group_norm_workspaces_of_no_samples(S, C, G):
    """In a process of its own: a division by zero in a size function ends it."""
    code = (f"import ctypes; lib = ctypes.CDLL({LIB_PATH!r})\n"
            "for f in (lib.dl_group_norm_scratch_bytes, lib.dl_group_norm_bwd_scratch_bytes):\n"
            "    f.argtypes, f.restype = [ctypes.c_int64] * 5, ctypes.c_int64\n"
            f"    assert all(f(0, {S}, {C}, {G}, dtype) == 0 for dtype in range(3))\n")
    done = subprocess.run([sys.executable, "-S", "-c", code], capture_output=True, text=True)
    assert done.returncode == 0, done.stderr


# ---------------------------------------------------------------------------------------------- differentiation
def test_forward_mode_differentiation_is_refused(no_launches):
    x, w, ids = torch.ones(6, 16), torch.ones(16), torch.arange(6)
    calls = [lambda t: dropout(t, 0.5), lambda t: embedding_lookup(ids, t), lambda t: group_norm(t, 4),
             lambda t: group_norm(x, 4, t[0]), lambda t: group_norm(x, 4, w, t[0])]
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in calls:
            with pytest.raises(NotImplementedError, match="jvp"):
                call(dual)
            with torch.no_grad(), pytest.raises(NotImplementedError, match="jvp"):
                call(dual)
        no_launches.clear()
        for call in calls:  # tensors without a tangent are taken as ever
            assert not call(x).requires_grad
        assert len(no_launches) == len(calls)
    assert not _native.followed(x, None) and _native.followed(None, w.clone().requires_grad_())


def test_gradient_with_a_forward_mode_tangent_is_refused(no_launches):
    """Forward over reverse: the operator's input has no tangent, what comes back to it has one."""
    ids = torch.arange(6)
    for call in (lambda t: dropout(t, 0.5), lambda t: embedding_lookup(ids, t), lambda t: group_norm(t, 4)):
        x = torch.ones(6, 16, requires_grad=True)
        y = call(x)
        with forward_ad.dual_level():
            g = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(NotImplementedError, match="jvp"):
                torch.autograd.grad(y, x, g, retain_graph=True)
            with pytest.raises(NotImplementedError, match="jvp"):
                torch.autograd.grad(y, x, g, retain_graph=True, create_graph=True)
            torch.autograd.grad(y, x, torch.ones_like(y))


# ---------------------------------------------------------------------------------------------- dropout
@pytest.mark.parametrize("use_reentrant", [False, True])
def test_dropout_module_recomputed_while_capturing_is_refused(no_launches, monkeypatch, use_reentrant):
    """A captured mask is drawn on the device: a recomputation would draw another one than the forward pass used."""
    drop, x = Dropout(0.5).train(), torch.ones(64, requires_grad=True)

    def gradient():
        y = checkpoint(lambda v: drop(v) * v, x, use_reentrant=use_reentrant, preserve_rng_state=False)
        y.sum().backward()

    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    gradient()  # eager: also makes the counter
    assert no_launches.count("dl_dropout") == 3
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="recomputed"):
        gradient()
    (drop(x) * x).sum().backward()  # without recomputation
    assert no_launches.count("dl_counter_draw") == 2


# ---------------------------------------------------------------------------------------------- what is kept
@pytest.mark.parametrize("saved,call", [
    (1, lambda x: embedding_lookup(torch.arange(4), x)),
    (2, lambda x: group_norm(x, 4)),  # and the statistics
    (1, lambda x: dropout(x, 0.5, counter=torch.zeros(1, dtype=torch.int64)))])
def test_what_the_backward_pass_needs_is_kept_by_autograd(no_launches, saved, call):
    """Saved-tensor hooks see it, and it goes with the first backward pass that does not keep the graph."""
    x, packed = torch.ones(8, 16, requires_grad=True), []

    def pack(t):
        packed.append(t)
        return t

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        y = call(x)
    assert len(packed) == saved
    torch.autograd.grad(y, x, torch.ones_like(y), retain_graph=True)
    torch.autograd.grad(y, x, torch.ones_like(y))
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, x, torch.ones_like(y))


# ---------------------------------------------------------------------------------------------- embedding encoder
@pytest.mark.parametrize("shape,flat", [((0, 5), (0, 20)), ((3, 0), (3, 0)), ((0,), (0,)), ((0, 2, 5), (0, 40)), ((3, 5), (3, 20)),
                                        ((3, 2, 5), (3, 40)), ((5,), (20,)), ((), (4,))])
def test_embedding_encoder_shapes(no_launches, shape, flat):
    ids = torch.zeros(shape, dtype=torch.int64)
    assert EmbeddingEncoder(10, num_bits=4).encode(ids).shape == flat
    assert EmbeddingEncoder(10, num_bits=4, flatten=False).encode(ids).shape == shape + (4,)


def test_network_refuses_an_encoder_without_thresholds():
    with pytest.raises(TypeError, match="thresholds.*EmbeddingEncoder.*layer API"):
        DWNNetwork(EmbeddingEncoder(10, num_bits=4), [], GroupSum(k=2, tau=1.0, use_randperm=False))


def test_dropout_module_seed_comes_from_the_cpu_generator(no_launches, monkeypatch):
    """Whatever the default device is."""
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    seeds = []
    monkeypatch.setattr(_native, "entry", lambda name: lambda *args: seeds.append(args[5]))
    x, drop = torch.ones(8), Dropout(0.5).train()
    for device in ("cpu", "meta"):
        torch.manual_seed(3)
        with torch.device(device):
            drop(x)
    torch.manual_seed(3)
    assert seeds == [int(torch.randint(0, 2 ** 62, (1,), dtype=torch.int64))] * 2
