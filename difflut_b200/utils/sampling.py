"""Sampling a class per row of logits (GroupSum's output, or any other logits) from given random numbers."""

from typing import Union

import torch

from .. import _native

# integer types with values that int32 does not have
_WIDE = (torch.int64, torch.uint64, torch.uint32)


def _setting(name, value, rows, dtype, low, high, low_open=False):
    """(per-row tensor or None, scalar) of one setting, checked; per-row values are not read on the host."""
    if isinstance(value, torch.Tensor):
        if value.shape != (rows,):
            raise ValueError(f"{name} must be a number or have shape ({rows},), got {tuple(value.shape)}")
        if not dtype.is_floating_point:
            if value.is_floating_point() or value.is_complex():
                raise ValueError(f"{name} must hold integers, got {value.dtype}")
            # 64 bits that cannot hold the value make it negative: it keeps all classes, as a count that large does
            value = value.to(torch.int64).clamp(0, torch.iinfo(dtype).max) if value.dtype in _WIDE else value
        return value.to(dtype).contiguous(), None
    number = isinstance(value, (int, float) if dtype.is_floating_point else int) and not isinstance(value, bool)
    if not number or not (low < value if low_open else low <= value) or not value <= high:
        raise ValueError(f"{name} must be {'above' if low_open else 'at least'} {low} and at most {high}, got {value}")
    return None, value


@torch.no_grad()
def sample_logits(logits: torch.Tensor, u: torch.Tensor, temperature: Union[float, torch.Tensor] = 1.0,
                  top_k: Union[int, torch.Tensor] = 0, top_p: Union[float, torch.Tensor] = 1.0,
                  min_p: Union[float, torch.Tensor] = 0.0) -> torch.Tensor:
    """One class id (int64) per row of logits (R, V), by the random number u (R) in [0, 1) of that row.

    Weights are exp((logit - max) / temperature), temperature 0 takes the largest logit.  Kept are the `top_k` largest
    logits (0: all), of these in descending order those with less than `top_p` of their total weight before them (1:
    all), of these the ones that weigh at least `min_p` times the largest (0: all).  The id is the first one in
    ascending order whose running sum of kept weights exceeds u times their total.  Equal logits rank by index, lowest
    first.  NaN and -inf are never taken; a row without any other logit gives -1.  Weights are whole numbers of 2^-50 of the
    largest (above 4096 classes of 2^(log2 V - 62)): a class that weighs less than half of that is never drawn.

    Every setting is a number or a tensor (R) of its own for each row (float32; int32 for top_k; other float or integer
    types are converted, and counts that int32 does not hold keep all).  u is float32 or float64.  logits (float32,
    bfloat16 or float16) may be a view with any distance between its rows.  The result does not depend on the order of
    additions: the same id on every run."""
    code = _native.dtype_code(logits, "logits")
    if logits.dim() != 2 or logits.shape[1] == 0:
        raise ValueError(f"logits must have shape (rows, classes) with at least one class, got {tuple(logits.shape)}")
    R, V = logits.shape
    if not isinstance(u, torch.Tensor) or u.dtype not in (torch.float32, torch.float64):
        raise TypeError(f"u must be a float32 or float64 tensor, got {getattr(u, 'dtype', type(u))}")
    if u.shape != (R,):
        raise ValueError(f"u must have shape ({R},), got {tuple(u.shape)}")
    inf = float("inf")
    t, t_all = _setting("temperature", temperature, R, torch.float32, 0.0, inf)
    k, k_all = _setting("top_k", top_k, R, torch.int32, 0, 2 ** 62)
    p, p_all = _setting("top_p", top_p, R, torch.float32, 0.0, 1.0, low_open=True)
    m, m_all = _setting("min_p", min_p, R, torch.float32, 0.0, 1.0)
    _native.require_cuda("sample_logits", logits, u, t, k, p, m)
    if logits.stride(1) != 1 and V > 1:
        logits = logits.contiguous()
    u = u.contiguous()
    out = logits.new_empty(R, dtype=torch.int64)
    with _native.device_of(logits):
        _native.entry("dl_sample_rows")(
            logits.data_ptr(), logits.stride(0), u.data_ptr(), u.dtype == torch.float64,
            None if t is None else t.data_ptr(), 1.0 if t_all is None else t_all,
            None if k is None else k.data_ptr(), 0 if k_all is None else k_all,
            None if p is None else p.data_ptr(), 1.0 if p_all is None else p_all,
            None if m is None else m.data_ptr(), 0.0 if m_all is None else m_all, out.data_ptr(), R, V, code)
    return out
