"""Dropout whose mask is recomputed from (seed, offset, element index) instead of being stored.

Next to the bit flip of the layer options (difflut/layers/base_layer.py:189-262), which replaces x by 1 - x, this one
zeroes activations and rescales the others.  The mask depends neither on the element type nor on the launch.
"""

from typing import Optional

import torch
import torch.nn as nn

from .. import _native
from .warnings import warn_default_value

DEFAULT_DROPOUT_P: float = 0.5
_WORD = 1 << 63


def _check_p(p) -> float:
    if isinstance(p, bool) or not isinstance(p, (int, float)) or not 0.0 <= p <= 1.0:
        raise ValueError(f"dropout probability p must be a number in [0, 1], got {p}")
    return float(p)


def _apply_mask(x, p, seed, offset, counter):
    out = torch.empty_like(x)  # x is contiguous
    with _native.device_of(x):
        _native.entry("dl_dropout")(x.data_ptr(), out.data_ptr(), x.numel(), _native.DTYPE_CODES[x.dtype], p, seed, offset,
                                    None if counter is None else counter.data_ptr())
    return out


class _DropoutFn(torch.autograd.Function):
    """y = mask(x) / (1 - p); its own gradient, so it can be differentiated any number of times."""

    @staticmethod
    def forward(ctx, x, p, seed, offset, counter):
        ctx.rule = (p, seed, offset)
        if counter is not None:
            ctx.save_for_backward(counter)
        ctx.drawn = counter is not None
        return _apply_mask(x, p, seed, offset, counter)

    @staticmethod
    def backward(ctx, g):
        p, seed, offset = ctx.rule
        counter = ctx.saved_tensors[0] if ctx.drawn else None
        g = g.contiguous()
        if torch.is_grad_enabled():  # create_graph
            return _DropoutFn.apply(g, p, seed, offset, counter), None, None, None, None
        _native.refuse_tangents(g)
        return _apply_mask(g, p, seed, offset, counter), None, None, None, None


def dropout(x: torch.Tensor, p: float = DEFAULT_DROPOUT_P, seed: int = 0, offset: int = 0,
            counter: Optional[torch.Tensor] = None) -> torch.Tensor:
    """x / (1 - p) where kept, 0 where dropped, in x's type (float32, bfloat16 or float16).

    Element i (row-major) is dropped when word i % 4 of Philox4x32-10 with counter (i // 4, offset) and key `seed` is
    below p * 2^32 (rounded).  The same (p, seed, offset) drops the same elements: use another `offset` per call.
    `counter` (one int64 on x's device) is added to `offset` when the kernel runs, which lets a captured graph draw
    another mask per replay; it must keep its value until the backward pass has run.  Differentiable any number of times, in
    reverse mode."""
    p = _check_p(p)
    for name, value in (("seed", seed), ("offset", offset)):
        if isinstance(value, bool) or not isinstance(value, int) or not 0 <= value < _WORD:
            raise ValueError(f"{name} must be an integer in [0, 2^63), got {value}")
    _native.dtype_code(x, "dropout input")
    _native.require_cuda("dropout", x, counter)
    if counter is not None and (counter.dtype != torch.int64 or counter.numel() != 1):
        raise TypeError(f"counter must hold one int64, got {counter.numel()} x {counter.dtype}")
    x = x.contiguous()
    if _native.followed(x):
        return _DropoutFn.apply(x, p, seed, offset, counter)
    return _apply_mask(x, p, seed, offset, counter)


class Dropout(nn.Module):
    """Dropout as a module: a new mask per training call, the identity in eval mode.

    Eager calls take a fresh seed from torch's CPU generator (reproducible under torch.manual_seed), as the layers'
    bit flip does.  While a CUDA graph is being captured the mask comes from a counter on the device instead, which
    every replay advances; it is created by an eager training call on that device, so run one before the capture (any
    warm-up step does).  In a block that a captured backward pass recomputes (checkpointing) the recomputation would draw
    another mask than the forward pass: it raises RuntimeError, use `dropout` with a seed or counter of your own there."""

    def __init__(self, p: Optional[float] = None) -> None:
        super().__init__()
        if p is None:
            p = DEFAULT_DROPOUT_P
            warn_default_value("p (Dropout)", p, stacklevel=2)
        self.p = _check_p(p)
        self._counters = {}  # device -> (seed, counter): drawn from by captured graphs only

    def __getstate__(self):
        state = self.__dict__.copy()
        state["_counters"] = {}  # a copy draws masks of its own
        return state

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if not self.training or self.p == 0.0:
            return x
        _native.require_cuda("Dropout", x)
        with _native.device_of(x):
            capturing = torch.cuda.is_current_stream_capturing()
            held = self._counters.get(x.device)
            if not capturing:
                seed = self._draw_seed()  # one draw per call, so that a recomputed call finds its own again
                if held is None:
                    self._counters[x.device] = (seed ^ 1 << 61, torch.zeros(1, device=x.device, dtype=torch.int64))
                return dropout(x, self.p, seed)
            if torch._C._current_graph_task_id() != -1:  # called by autograd, in a backward pass
                raise RuntimeError("Dropout: a block recomputed while its backward pass is captured into a CUDA graph would draw "
                                   "another mask than its forward pass; use dropout() with a seed or counter of your own")
            if held is None:
                raise RuntimeError("Dropout: run one training call on this device before capturing a CUDA graph")
            seed, counter = held
            drawn = torch.empty(1, device=x.device, dtype=torch.int64)
            _native.call("dl_counter_draw", counter, drawn)
        return dropout(x, self.p, seed, 0, drawn)

    @staticmethod
    def _draw_seed() -> int:
        return int(torch.randint(0, 2 ** 62, (1,), dtype=torch.int64, device="cpu").item())

    def extra_repr(self) -> str:
        return f"p={self.p}"
