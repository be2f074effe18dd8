"""Embedding encoder: token ids -> `num_bits` learned features per token.

The thermometer encoders turn real features into bits; for token ids or other categorical features the features
themselves are learned.  LUT nodes read them the way they read any layer input (`value >= 0.5` for DWN-type nodes,
a probability for Probabilistic nodes) and their input gradient trains the table.  No counterpart in the reference
(its encoders take real features; the interface is difflut/encoder/base_encoder.py:18-137).
"""

import functools
from typing import Optional

import torch
import torch.nn as nn

from .. import _native
from ..registry import register_encoder
from .base_encoder import BaseEncoder

DEFAULT_EMBEDDING_NUM_BITS: int = 8


@functools.lru_cache(maxsize=1024)
def _sizes(tokens, V, D, code):
    """Bytes of (the sorted tokens, the backward pass's workspace)."""
    lib = _native.lib()
    order = int(lib.dl_embedding_order_bytes(tokens, V, D, code))
    if order == 0:
        raise RuntimeError(f"the gradient of {tokens} tokens into a {V} x {D} table is not supported")
    return order, int(lib.dl_embedding_bwd_scratch_bytes(tokens, V, D, code))


def _forward(ids, weight, scale, padding, sort):
    """(looked-up rows, the sorted tokens that the backward pass wants or None)."""
    V, D = weight.shape
    code, tokens = _native.DTYPE_CODES[weight.dtype], ids.numel()
    out = weight.new_empty(ids.shape + (D,))
    order = weight.new_empty(_sizes(tokens, V, D, code)[0], dtype=torch.uint8) if sort else None
    with _native.device_of(weight):
        _native.entry("dl_embedding")(ids.data_ptr(), 64 if ids.dtype == torch.int64 else 32, weight.data_ptr(),
                                      out.data_ptr(), tokens, V, D, code, scale, padding,
                                      order.data_ptr() if sort else None)
    return out, order


class _EmbeddingFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding):
        out, order = _forward(ids, weight, scale, padding, True)
        ctx.save_for_backward(order)
        ctx.spec = (ids.numel(), weight.shape, weight.dtype, scale)
        return out

    @staticmethod
    @_native.once_differentiable_backward
    def backward(ctx, g):
        (order,), (tokens, (V, D), dtype, scale) = ctx.saved_tensors, ctx.spec
        code = _native.DTYPE_CODES[dtype]
        g = g.contiguous()
        gw = g.new_empty((V, D))
        scratch = order.new_empty(_sizes(tokens, V, D, code)[1])
        with _native.device_of(g):
            _native.entry("dl_embedding_bwd")(order.data_ptr(), g.data_ptr(), gw.data_ptr(), tokens, V, D, code, scale,
                                              scratch.data_ptr())
        return None, gw, None, None


def embedding_lookup(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
                     padding_idx: Optional[int] = None) -> torch.Tensor:
    """`scale * weight[ids]`, shape `ids.shape + (D,)`, in weight's type (float32, bfloat16 or float16).

    The gradient of `weight` sums the rows of equal ids in the order of their positions, in fp32, rounded once: the
    same bits on every run.  `padding_idx` takes no gradient.  An id outside [0, V) gives a NaN row and takes no
    gradient (torch raises a device assertion; nothing is read outside the table here).  Differentiable once, in reverse
    mode."""
    if not isinstance(ids, torch.Tensor) or ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"ids must be an int32 or int64 tensor, got {getattr(ids, 'dtype', type(ids))}")
    if weight.dim() != 2 or weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError(f"weight must be a non-empty (num_embeddings, features) matrix, got shape {tuple(weight.shape)}")
    _native.dtype_code(weight, "weight")
    _native.require_cuda("embedding_lookup", ids, weight)
    V = weight.shape[0]
    padding = -1
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"padding_idx must be within [-{V}, {V}), got {padding_idx}")
        padding = int(padding_idx) % V
    ids, weight = ids.contiguous(), weight.contiguous()
    if _native.followed(weight):
        return _EmbeddingFn.apply(ids, weight, float(scale), padding)
    return _forward(ids, weight, float(scale), padding, False)[0]


@register_encoder("embedding")
class EmbeddingEncoder(BaseEncoder):
    """Token ids (B, T) -> (B, T * num_bits) if `flatten` else (B, T, num_bits); a 1-D input is one sample.

    `weight` (num_embeddings, num_bits) starts uniform such that the scaled features lie in [0, 1), half of them
    above the 0.5 that DWN-type nodes threshold at.  There is nothing to fit: `fit` only returns the encoder."""

    def __init__(self, num_embeddings: int, num_bits: int = DEFAULT_EMBEDDING_NUM_BITS, scale: float = 1.0,
                 padding_idx: Optional[int] = None, flatten: bool = True,
                 dtype: torch.dtype = torch.float32) -> None:
        super().__init__(num_bits=num_bits, flatten=flatten)
        if not isinstance(num_embeddings, int) or num_embeddings <= 0:
            raise ValueError(f"num_embeddings must be a positive integer, got {num_embeddings}")
        if not isinstance(scale, (int, float)) or not scale > 0:
            raise ValueError(f"scale must be a positive number, got {scale}")
        if padding_idx is not None and not -num_embeddings <= padding_idx < num_embeddings:
            raise ValueError(f"padding_idx must be within [-{num_embeddings}, {num_embeddings}), got {padding_idx}")
        if dtype not in _native.DTYPE_CODES:
            raise TypeError(f"dtype must be float32, bfloat16 or float16, got {dtype}")
        self.num_embeddings, self.scale, self.padding_idx = num_embeddings, float(scale), padding_idx
        self.weight = nn.Parameter((torch.rand(num_embeddings, self.num_bits) / self.scale).to(dtype))
        if padding_idx is not None:
            with torch.no_grad():
                self.weight[padding_idx] = 0.0
        self._is_fitted = True

    def fit(self, x=None) -> "EmbeddingEncoder":
        return self

    def encode(self, x) -> torch.Tensor:
        ids = self._to_tensor(x)
        out = embedding_lookup(ids, self.weight, self.scale, self.padding_idx)
        if not self.flatten:
            return out
        return out.reshape(-1) if ids.dim() <= 1 else out.flatten(1)

    def to(self, *args, **kwargs) -> "EmbeddingEncoder":
        return nn.Module.to(self, *args, **kwargs)  # the table is a parameter, not a plain attribute

    def __repr__(self) -> str:
        return (f"EmbeddingEncoder(num_embeddings={self.num_embeddings}, num_bits={self.num_bits}, "
                f"scale={self.scale}, padding_idx={self.padding_idx}, flatten={self.flatten})")
