"""Plain 64-bit forms of the token-path operators (embedding, dropout, group norm, sampling) for the tests."""

import math

import numpy as np
import torch

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def half_step(dtype) -> float:
    """Largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def smallest(dtype) -> float:
    """Half the spacing of the subnormal numbers: the absolute error of a rounding near zero."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


def check(got: torch.Tensor, ref: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    """|got - ref| <= bound element by element (all in float64)."""
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)} instead of {tuple(ref.shape)}"
    err = (got.detach().double().cpu() - ref.detach().double().cpu()).abs()
    bound = torch.as_tensor(bound, dtype=torch.float64).cpu()
    bad = ~(err <= bound)
    if bool(bad.any()):
        i = int(torch.where(bad, torch.nan_to_num(err, nan=math.inf), torch.zeros_like(err)).reshape(-1).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} elements off, element {i}: got "
                             f"{got.reshape(-1)[i].item()} ref {ref.reshape(-1)[i].item()} "
                             f"bound {bound.expand_as(err).reshape(-1)[i].item()}")


# ---------------------------------------------------------------------------------------------- dropout
def philox(counter, key):
    """Philox4x32-10: counter (n, 4) and key (k0, k1) -> (n, 4) uint32 words, by 64-bit integer products."""
    c = [np.asarray(counter)[:, j].astype(np.uint64) for j in range(4)]
    k0, k1 = int(key[0]), int(key[1])
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), p1 & low, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), p0 & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c, axis=1).astype(np.uint32)


def dropped(numel, p, seed, offset):
    """Boolean mask (numel,) of the elements that dropout zeroes."""
    q = np.arange((numel + 3) // 4, dtype=np.uint64)
    counter = np.stack([q & np.uint64(0xFFFFFFFF), q >> np.uint64(32), np.full_like(q, offset & 0xFFFFFFFF),
                        np.full_like(q, offset >> 32)], axis=1)
    words = philox(counter, (seed & 0xFFFFFFFF, seed >> 32)).reshape(-1)[:numel].astype(np.uint64)
    return torch.from_numpy(words < np.uint64(int(p * 2.0 ** 32 + 0.5)))


# ---------------------------------------------------------------------------------------------- embedding
def embedding_grad(ids, g, V, scale, padding=None):
    """(gradient, sum of absolute terms, terms) of the table, float64, by one addition per token."""
    ids, g = ids.reshape(-1).cpu(), g.detach().double().cpu().reshape(ids.numel(), -1)
    ok = (ids >= 0) & (ids < V)
    if padding is not None:
        ok &= ids != padding
    total = torch.zeros(V, g.shape[1], dtype=torch.float64)
    size, count = torch.zeros_like(total), torch.zeros(V, 1, dtype=torch.float64)
    for t in torch.nonzero(ok).reshape(-1).tolist():
        total[ids[t]] += g[t]
        size[ids[t]] += g[t].abs()
        count[ids[t]] += 1
    return total * scale, size * abs(scale), count


# ---------------------------------------------------------------------------------------------- group norm
def norm_reference(x, G, weight, bias, eps, act, g=None, depth=400):
    """Float64 results of x (N, S, C) and the bounds of their errors, as pairs.

    With u = 2^-24 and `depth` the longest chain of additions of a sum: the mean is off by depth * u * mean|x|, the
    variance by depth * u relative (its squares are centred), hence xh by `e_xh`, z by `e_z` and so on through the
    formulas; exponential and quotient of the sigmoid are a few u, the slopes change by at most half as much as z."""
    u = 2.0 ** -24
    N, S, C = x.shape
    x = x.detach().double().cpu()
    w = torch.ones(C, dtype=torch.float64) if weight is None else weight.detach().double().cpu()
    b = torch.zeros(C, dtype=torch.float64) if bias is None else bias.detach().double().cpu()

    def groups(t):
        return t.reshape(N, S, G, C // G)

    def mean(t):  # over a sample's group, spread over its elements
        return groups(t).mean(dim=(1, 3), keepdim=True).expand(N, S, G, C // G).reshape(N, S, C)

    mu = mean(x)
    rstd = torch.rsqrt(mean((x - mu) ** 2) + eps)
    xh = (x - mu) * rstd
    z = xh * w + b
    e_xh = depth * u * mean(x.abs()) * rstd + 2 * u * mu.abs() * rstd + xh.abs() * (depth / 2 + 4) * u
    e_z = e_xh * w.abs() + 2 * u * ((xh * w).abs() + b.abs())
    s = torch.sigmoid(z)
    y, slope = {"none": (z, torch.ones_like(z)), "relu": (z.clamp_min(0), (z > 0).double()),
                "silu": (z * s, s * (1 + z * (1 - s))), "sigmoid": (s, s * (1 - s))}[act]
    e_y = 1.1 * e_z + (10 + z.abs()) * u * (y.abs() + s)
    out = {"z": z, "y": (y, e_y)}
    if g is None:
        return out
    g = g.detach().double().cpu()
    dz = g * slope
    e_dz = g.abs() * ((0 if act in ("none", "relu") else 0.5) * e_z + (10 + z.abs()) * u)
    wdz = dz * w
    s1, s2 = mean(wdz), mean(wdz * xh)
    e_s1 = mean(e_dz * w.abs()) + (depth + 4) * u * mean(wdz.abs())
    e_s2 = mean(e_dz * (w * xh).abs() + wdz.abs() * e_xh) + (depth + 4) * u * mean((wdz * xh).abs())
    gx = rstd * (wdz - s1 - xh * s2)
    size = rstd * (wdz.abs() + s1.abs() + (xh * s2).abs())
    e_gx = rstd * (w.abs() * e_dz + e_s1 + xh.abs() * e_s2 + e_xh * s2.abs()) + size * (8 + depth / 2) * u
    gw, gb = (dz * xh).sum(dim=(0, 1)), dz.sum(dim=(0, 1))
    e_gw = (e_dz * xh.abs() + dz.abs() * e_xh + depth * u * (dz * xh).abs()).sum(dim=(0, 1))
    e_gb = (e_dz + depth * u * dz.abs()).sum(dim=(0, 1))
    out.update(gx=(gx, e_gx), gw=(gw, e_gw), gb=(gb, e_gb))
    return out


# ---------------------------------------------------------------------------------------------- sampling
def kept_weights(x, T=1.0, k=0, p=1.0, min_p=0.0):
    """(ids in ascending order, their weights) that survive temperature, top-k, top-p and min-p, in float64."""
    x = np.asarray(x, dtype=np.float64)
    ids = np.flatnonzero(x > -np.inf)
    if len(ids) == 0:
        return ids, np.zeros(0)
    ids = ids[np.lexsort((ids, -x[ids]))]
    if T <= 0:
        return ids[:1], np.ones(1)
    if k > 0:
        ids = ids[:k]
    top = x[ids[0]]
    w = (x[ids] == np.inf).astype(np.float64) if top == np.inf else np.exp((x[ids] - top) / T)
    if p < 1.0:
        ahead = np.concatenate(([0.0], np.cumsum(w)[:-1]))
        inside = ahead < max(p * w.sum(), 1e-300)
        ids, w = ids[inside], w[inside]
    ids, w = ids[w >= min_p], w[w >= min_p]
    order = np.argsort(ids)
    return ids[order], w[order]


def sample_row(x, u, T=1.0, k=0, p=1.0, min_p=0.0) -> int:
    ids, w = kept_weights(x, T, k, p, min_p)
    if len(ids) == 0:
        return -1
    upto = np.cumsum(w)
    return int(ids[min(int(np.searchsorted(upto, u * upto[-1], side="right")), int(np.flatnonzero(w)[-1]))])
