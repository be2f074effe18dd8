"""Group norm with an activation over channels-last data.

LUT nodes read their inputs as bits (`value >= 0.5`) or as probabilities; a norm followed by a sigmoid puts any layer's
values there, half of them on either side of 0.5.  Channels last is how the package's own layers write: rows (B, F), and
the memory behind ConvolutionalLayer's (B, C, H, W) output (difflut/layers/convolutional.py:199-240).
"""

import functools
from typing import Optional

import torch
import torch.nn as nn

from .. import _native

DEFAULT_GROUPNORM_EPS: float = 1e-5
ACTIVATIONS = {"none": 0, "relu": 1, "silu": 2, "sigmoid": 3}


def _check_activation(activation) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, got {activation!r}")
    return ACTIVATIONS[activation]


@functools.lru_cache(maxsize=1024)
def _scratch_bytes(N, S, C, G, code):
    """Workspace of (the forward, the backward pass)."""
    lib = _native.lib()
    sizes = (int(lib.dl_group_norm_scratch_bytes(N, S, C, G, code)),
             int(lib.dl_group_norm_bwd_scratch_bytes(N, S, C, G, code)))
    if min(sizes) < 0:
        raise RuntimeError(f"group_norm of {N} x {S} x {C} values in {G} groups is not supported")
    return sizes


def _address(t):
    return None if t is None else t.data_ptr()


def _forward(x, weight, bias, dims, eps, act, keep):
    """(result, mean and rstd behind the workspace, their address), the latter two for the backward pass only."""
    N, S, C, G, param_code = dims
    code = _native.DTYPE_CODES[x.dtype]
    y = torch.empty_like(x)
    size = _scratch_bytes(N, S, C, G, code)[0]
    held = x.new_empty(size // 4 + (2 * N * G if keep else 0), dtype=torch.float32) if keep or size else None
    scratch = _address(held)
    mean = scratch + size if keep else None
    with _native.device_of(x):
        _native.entry("dl_group_norm")(x.data_ptr(), _address(weight), _address(bias), y.data_ptr(), mean,
                                       mean + 4 * N * G if keep else None, scratch, N, S, C, G, code, param_code, act, eps)
    return y, held, size


class _GroupNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, dims, eps, act):
        y, held, mean_at = _forward(x, weight, bias, dims, eps, act, True)
        ctx.save_for_backward(x, weight, bias, held)
        ctx.spec = (dims, act, mean_at)
        return y

    @staticmethod
    @_native.once_differentiable_backward
    def backward(ctx, g):
        x, weight, bias, held = ctx.saved_tensors
        (N, S, C, G, param_code), act, mean_at = ctx.spec
        code = _native.DTYPE_CODES[x.dtype]
        g = g.contiguous()
        gx = torch.empty_like(x)
        gw = torch.empty_like(weight) if weight is not None and ctx.needs_input_grad[1] else None
        gb = torch.empty_like(bias) if bias is not None and ctx.needs_input_grad[2] else None
        scratch = x.new_empty(_scratch_bytes(N, S, C, G, code)[1], dtype=torch.uint8)
        mean = held.data_ptr() + mean_at
        with _native.device_of(x):
            _native.entry("dl_group_norm_bwd")(x.data_ptr(), g.data_ptr(), _address(weight), _address(bias), mean,
                                               mean + 4 * N * G, gx.data_ptr(), _address(gw), _address(gb),
                                               scratch.data_ptr(), N, S, C, G, code, param_code, act)
        return gx, gw, gb, None, None, None


def group_norm(x: torch.Tensor, num_groups: int, weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None, eps: float = DEFAULT_GROUPNORM_EPS,
               activation: str = "none") -> torch.Tensor:
    """`act(norm(x) * weight + bias)` for x (N, ..., C): every sample's group of C / num_groups channels is normalised
    over all positions in between, by its mean and biased variance.

    x is float32, bfloat16 or float16; weight and bias (C) are float32 or of x's type.  Statistics and sums are fp32, the
    result is rounded once (sigmoids below 2^-126 are 0).  activation: "none", "relu", "silu" or "sigmoid".  Differentiable
    once, in reverse mode."""
    act = _check_activation(activation)
    _native.dtype_code(x, "group_norm input")
    if x.dim() < 2:
        raise ValueError(f"group_norm expects (N, ..., C) input, got shape {tuple(x.shape)}")
    N, C = x.shape[0], x.shape[-1]
    S = 1
    for size in x.shape[1:-1]:
        S *= size
    if isinstance(num_groups, bool) or not isinstance(num_groups, int) or num_groups <= 0:
        raise ValueError(f"num_groups must be a positive integer, got {num_groups}")
    if C == 0 or C % num_groups != 0:
        raise ValueError(f"{C} channels do not form {num_groups} groups of equal size")
    if not eps >= 0.0:
        raise ValueError(f"eps must not be negative, got {eps}")
    param_dtype = None
    for name, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != (C,):
            raise ValueError(f"{name} must have shape ({C},), got {tuple(p.shape)}")
        if p.dtype not in (torch.float32, x.dtype):
            raise TypeError(f"{name} must be float32 or of the input's type {x.dtype}, got {p.dtype}")
        if param_dtype not in (None, p.dtype):
            raise TypeError(f"weight and bias must be of one type, got {param_dtype} and {p.dtype}")
        param_dtype = p.dtype
    _native.require_cuda("group_norm", x, weight, bias)
    if S == 0:
        raise ValueError(f"group_norm needs at least one position per sample, got shape {tuple(x.shape)}")
    x = x.contiguous()
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    dims = (N, S, C, num_groups, 0 if param_dtype is None else _native.DTYPE_CODES[param_dtype])
    if _native.followed(x, weight, bias):
        return _GroupNormFn.apply(x, weight, bias, dims, float(eps), act)
    return _forward(x, weight, bias, dims, float(eps), act, False)[0]


class GroupNorm(nn.Module):
    """Group norm with an activation as a module: (N, ..., C), or with `channel_dim=1` (N, C, ...).

    With `channel_dim=1` the memory still is channels last: the output of a ConvolutionalLayer and tensors in torch's
    channels_last format are taken as they are, any other layout is copied first."""

    def __init__(self, num_groups: int, num_channels: int, eps: float = DEFAULT_GROUPNORM_EPS, affine: bool = True,
                 activation: str = "none", channel_dim: int = -1) -> None:
        super().__init__()
        if num_groups <= 0 or num_channels <= 0 or num_channels % num_groups != 0:
            raise ValueError(f"{num_channels} channels do not form {num_groups} groups of equal size")
        if not eps >= 0.0:
            raise ValueError(f"eps must not be negative, got {eps}")
        _check_activation(activation)
        if channel_dim not in (-1, 1):
            raise ValueError(f"channel_dim must be -1 or 1, got {channel_dim}")
        self.num_groups, self.num_channels, self.eps = num_groups, num_channels, float(eps)
        self.activation, self.channel_dim = activation, channel_dim
        self.weight = nn.Parameter(torch.ones(num_channels)) if affine else None
        self.bias = nn.Parameter(torch.zeros(num_channels)) if affine else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dim() < 2 or x.shape[self.channel_dim] != self.num_channels:
            raise ValueError(f"GroupNorm expects {self.num_channels} channels in dimension {self.channel_dim}, got shape "
                             f"{tuple(x.shape)}")
        if self.channel_dim == 1:
            x = x.movedim(1, -1)
        y = group_norm(x, self.num_groups, self.weight, self.bias, self.eps, self.activation)
        return y.movedim(-1, 1) if self.channel_dim == 1 else y

    def extra_repr(self) -> str:
        return (f"{self.num_groups}, {self.num_channels}, eps={self.eps}, affine={self.weight is not None}, "
                f"activation={self.activation!r}, channel_dim={self.channel_dim}")
