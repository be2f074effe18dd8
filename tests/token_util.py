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
