"""What a token model of LUT layers does around its layers, as measured cases.

Four operators: the embedding encoder (token ids to features, with its gradient by sorted tokens), group norm with an
activation over channels-last data (it brings values into the range that LUT nodes threshold), dropout from a
counter-based generator, and sampling of a class from GroupSum logits with given random numbers.  `run` computes
a case either in its plain form (elementary torch operations) or, with `own` set, by the calls a user makes.
"""

import math

import numpy as np
import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}


# ------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one step of generation for 32 streams: a row of the table each
        {"name": "embed_step", "op": "embed", "train": False, "T": 32, "V": 32000, "D": 1024, "dtype": "bf16",
         "padding": False},
        # a small vocabulary of ragged width, trained in fp32, with a padding id
        {"name": "embed_train_odd", "op": "embed", "train": True, "T": 5003, "V": 10007, "D": 515, "dtype": "fp32",
         "padding": True},
        # a training batch of 32 sequences of 2048 tokens
        {"name": "embed_train", "op": "embed", "train": True, "T": 65536, "V": 65536, "D": 1024, "dtype": "bf16",
         "padding": False},
        # raw features of one small batch of 28 x 28 images
        {"name": "dropout_small", "op": "dropout", "numel": 128 * 784, "p": 0.1, "dtype": "fp32"},
        # activations between two layers: batch 8192, 8000 nodes
        {"name": "dropout_train", "op": "dropout", "numel": 8192 * 8000, "p": 0.25, "dtype": "bf16"},
        # a convolutional LUT layer's output: 128 images, 24 x 24 positions, 32 trees
        {"name": "norm_conv", "op": "norm", "train": True, "N": 128, "S": 576, "C": 32, "G": 8, "act": "sigmoid",
         "dtype": "fp32"},
        # feature rows in front of a LUT layer (no spatial positions)
        {"name": "norm_rows", "op": "norm", "train": True, "N": 8192, "S": 1, "C": 1024, "G": 32, "act": "sigmoid",
         "dtype": "bf16"},
        # feature maps of 64 x 64
        {"name": "norm_maps", "op": "norm", "train": True, "N": 16, "S": 4096, "C": 512, "G": 32, "act": "silu",
         "dtype": "bf16"},
        # inference on a ragged map whose groups hold 10 channels
        {"name": "norm_odd_infer", "op": "norm", "train": False, "N": 7, "S": 1517, "C": 120, "G": 12, "act": "relu",
         "dtype": "fp16"},
        # one step of generation for eight streams with settings of their own
        {"name": "sample_step", "op": "sample", "R": 8, "V": 32000, "dtype": "bf16", "per_row": True,
         "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0},
        # classes of a byte-level GroupSum head for a whole batch
        {"name": "sample_classes", "op": "sample", "R": 8192, "V": 256, "dtype": "fp32", "per_row": False,
         "temperature": 1.0, "top_k": 40, "top_p": 1.0, "min_p": 0.0},
        # a wide batch with a large vocabulary, nucleus and min-p
        {"name": "sample_wide", "op": "sample", "R": 256, "V": 65536, "dtype": "fp32", "per_row": False,
         "temperature": 0.9, "top_k": 0, "top_p": 0.9, "min_p": 0.01},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over the logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["embed", "dropout", "norm", "sample"])
    dtype = rng.choice(["fp32", "bf16", "fp16"])
    if op == "embed":
        T, V, D = _spread(rng, 1, 65536), _spread(rng, 100, 65536), _spread(rng, 8, 1024)
        if rng.random() < 0.5:
            D = max(8, D // 8 * 8)
        while max(T, V) * D * _SIZE[dtype] > 65536 * 1024 * 2:
            T, V = max(1, T // 2), max(100, V // 2)
        return {"op": op, "train": rng.random() < 0.6, "T": T, "V": V, "D": D, "dtype": dtype,
                "padding": rng.random() < 0.3}
    if op == "dropout":
        numel = _spread(rng, 100, 8192 * 4000)
        return {"op": op, "numel": numel, "p": rng.choice([0.0, 0.05, 0.1, 0.25, 0.5, 0.9]), "dtype": dtype}
    if op == "norm":
        train = rng.random() < 0.7
        G = rng.choice([1, 2, 4, 8, 12, 16, 32])
        per = rng.choice([1, 2, 3, 4, 6, 8, 10, 16, 20, 32]) if G > 1 else rng.choice([5, 16, 64, 100, 256])
        S = 1 if rng.random() < 0.25 else _spread(rng, 2, 10000)
        while S * per < 16:  # fewer values than that have no statistics worth the name
            per *= 2
        C = G * per
        N = _spread(rng, 1, max(2, min(8192, (1 << 24) // (S * C))))
        return {"op": op, "train": train, "N": N, "S": S, "C": C, "G": G,
                "act": rng.choice(["none", "silu", "sigmoid"] if train else ["none", "relu", "silu", "sigmoid"]),
                "dtype": dtype}
    V = _spread(rng, 2, 131072)
    R = _spread(rng, 1, max(2, min(8192, (1 << 23) // V)))
    return {"op": op, "R": R, "V": V, "dtype": dtype, "per_row": rng.random() < 0.5,
            "temperature": rng.choice([0.5, 0.7, 1.0, 1.3]), "top_k": rng.choice([0, 1, 5, 40, 50, 200]),
            "top_p": rng.choice([1.0, 0.95, 0.9, 0.5]), "min_p": rng.choice([0.0, 0.0, 0.02, 0.1])}


# ------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(int(seed))
    dt = _TYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    s = dict(case)
    if case["op"] == "embed":
        T, V, D = case["T"], case["V"], case["D"]
        # ids in order of frequency, the frequency falling as 1 / rank
        r = torch.rand(T, generator=g, device=dev, dtype=torch.float64)
        s["ids"] = (torch.exp(r * math.log(V + 1.0)) - 1.0).long().clamp_(0, V - 1)
        s["weight"] = (normal(V, D) * 0.5).to(dt)
        s["scale"] = math.sqrt(D)
        s["padding_idx"] = 0 if case["padding"] else None
        if case["train"]:
            s["weight"].requires_grad_(True)
            s["grad"] = normal(T, D).to(dt)
    elif case["op"] == "dropout":
        s["x"] = normal(case["numel"]).to(dt).requires_grad_(True)
        s["grad"] = normal(case["numel"]).to(dt)
        s["seed"], s["offset"] = (int(seed) * 0x9E3779B97F4A7C15 + 12345) % (1 << 62), 7 + int(seed) % 1000
    elif case["op"] == "norm":
        N, S, C = case["N"], case["S"], case["C"]
        s["x"] = (normal(N, S, C) * 1.5 + normal(C)).to(dt)
        s["weight"] = 1.0 + 0.2 * normal(C)
        s["bias"] = 0.1 * normal(C)
        s["eps"] = 1e-5
        if case["train"]:
            for name in ("x", "weight", "bias"):
                s[name].requires_grad_(True)
            s["grad"] = normal(N, S, C).to(dt)
    else:
        R, V = case["R"], case["V"]
        x = normal(R, V) * 2.5
        # a few candidates stand out, some classes are masked, in a larger batch one row entirely
        x += 6.0 * (torch.rand(R, V, generator=g, device=dev) < min(0.5, 4.0 / V))
        x = torch.where(torch.rand(R, V, generator=g, device=dev) < 0.05, -math.inf, x)
        if R >= 8:
            x[R // 2] = -math.inf
        s["logits"] = x.to(dt)
        s["u"] = torch.rand(R, generator=g, device=dev)
        if case["per_row"]:
            mix = torch.arange(R, device=dev)
            s["temperature"] = torch.where(mix % 5 == 3, 0.0, case["temperature"]).float()
            s["top_k"] = torch.where(mix % 4 == 1, 0, case["top_k"]).int()
            s["top_p"] = torch.where(mix % 3 == 2, 1.0, case["top_p"]).float()
            s["min_p"] = torch.full((R,), case["min_p"], device=dev)
    return s


# ------------------------------------------------------------------------------------------------- passes
def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    if s["op"] == "embed":
        from difflut_b200.encoder import embedding_lookup

        out = embedding_lookup(s["ids"], s["weight"], scale=s["scale"], padding_idx=s["padding_idx"])
        if not s["train"]:
            return out
        return out.detach(), torch.autograd.grad(out, s["weight"], s["grad"])[0]
    if s["op"] == "dropout":
        from difflut_b200.utils import dropout

        y = dropout(s["x"], s["p"], seed=s["seed"], offset=s["offset"])
        return y.detach(), torch.autograd.grad(y, s["x"], s["grad"])[0]
    if s["op"] == "norm":
        from difflut_b200.utils import group_norm

        y = group_norm(s["x"], s["G"], s["weight"], s["bias"], eps=s["eps"], activation=s["act"])
        if not s["train"]:
            return y
        return (y.detach(),) + torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["grad"])
    from difflut_b200.utils import sample_logits

    return sample_logits(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                         min_p=s["min_p"])


@torch.no_grad()
def _run_plain(s):
    return {"embed": _plain_embed, "dropout": _plain_dropout, "norm": _plain_norm, "sample": _plain_sample}[s["op"]](s)


def _plain_embed(s):
    ids, weight = s["ids"], s["weight"]
    out = (weight[ids].float() * s["scale"]).to(weight.dtype)
    if not s["train"]:
        return out
    acc = torch.zeros(weight.shape, device=weight.device, dtype=torch.float32)
    acc.index_add_(0, ids, s["grad"].float())
    if s["padding_idx"] is not None:
        acc[s["padding_idx"]] = 0.0
    return out, (acc * s["scale"]).to(weight.dtype)


def _wide_product(a, m):
    """High and low 32 bits of a * m for 32-bit values held in int64 (the product itself would not fit)."""
    low = a * (m & 0xFFFF)
    high = a * (m >> 16)
    low = low + ((high & 0xFFFF) << 16)
    return (high >> 16) + (low >> 32), low & 0xFFFFFFFF


def _plain_words(numel, seed, offset, device):
    """Philox4x32-10 (Salmon et al. 2011), one block for four elements."""
    q = torch.arange((numel + 3) // 4, device=device, dtype=torch.int64)
    c0, c1 = q & 0xFFFFFFFF, q >> 32
    c2, c3 = torch.full_like(q, offset & 0xFFFFFFFF), torch.full_like(q, offset >> 32)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        h0, l0 = _wide_product(c0, 0xD2511F53)
        h1, l1 = _wide_product(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = h1 ^ c1 ^ k0, l1, h0 ^ c3 ^ k1, l0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return torch.stack((c0, c1, c2, c3), dim=1).reshape(-1)[:numel]


def _plain_dropout(s):
    x, p = s["x"], s["p"]
    keep = _plain_words(x.numel(), s["seed"], s["offset"], x.device) >= int(p * 4294967296.0 + 0.5)
    zero = torch.zeros((), device=x.device)
    return tuple(torch.where(keep, t.float() * (1.0 / (1.0 - p)), zero).to(x.dtype) for t in (x, s["grad"]))


def _plain_norm(s):
    x, weight, bias, act = s["x"], s["weight"], s["bias"], s["act"]
    N, S, C, G = s["N"], s["S"], s["C"], s["G"]
    m = S * (C // G)
    xg = x.float().view(N, S, G, C // G)
    mean = xg.sum(dim=(1, 3), keepdim=True) / m
    rstd = torch.rsqrt(((xg - mean) * (xg - mean)).sum(dim=(1, 3), keepdim=True) / m + s["eps"])
    xh = ((xg - mean) * rstd).view(N, S, C)
    z = xh * weight + bias
    sig = 1.0 / (1.0 + torch.exp(-z))
    y = {"none": z, "relu": z.clamp_min(0.0), "silu": z * sig, "sigmoid": sig}[act]
    if not s["train"]:
        return y.to(x.dtype)
    slope = {"none": torch.ones_like(z), "relu": (z > 0).float(), "silu": sig * (1.0 + z * (1.0 - sig)),
             "sigmoid": sig * (1.0 - sig)}[act]
    dz = s["grad"].float() * slope
    dweight, dbias = (dz * xh).sum(dim=(0, 1)), dz.sum(dim=(0, 1))
    dxh = (dz * weight).view(N, S, G, C // G)
    xh = xh.view(N, S, G, C // G)
    s1 = dxh.sum(dim=(1, 3), keepdim=True) / m
    s2 = (dxh * xh).sum(dim=(1, 3), keepdim=True) / m
    dx = ((dxh - s1 - xh * s2) * rstd).view(N, S, C)
    return y.to(x.dtype), dx.to(x.dtype), dweight, dbias


def _column(value, rows, device):
    if isinstance(value, torch.Tensor):
        return value.double().view(rows, 1)
    return torch.full((rows, 1), float(value), device=device, dtype=torch.float64)


def _plain_sample(s):
    x = s["logits"].double()
    R, V = x.shape
    T, k, p, min_p = (_column(s[n], R, x.device) for n in ("temperature", "top_k", "top_p", "min_p"))
    greedy = T == 0
    k = torch.where(greedy, 1.0, torch.where(k <= 0, float(V), k))
    T = torch.where(greedy, 1.0, T)
    valid = x > -math.inf
    x = torch.where(valid, x, -math.inf)
    # descending, equal values by index
    ordered, order = torch.sort(x, dim=1, descending=True, stable=True)
    top = ordered[:, :1]
    w = torch.exp((ordered - top) / T)
    w = torch.where(top == math.inf, (ordered == math.inf).double(), w)
    keep = (torch.arange(V, device=x.device) < k) & (ordered > -math.inf)
    w = torch.where(keep, w, 0.0)
    upto = torch.cumsum(w, dim=1)
    keep &= (upto - w < p * upto[:, -1:]) | (p >= 1.0)
    keep &= w >= min_p
    w = torch.where(keep, w, 0.0)
    kept = torch.zeros_like(w).scatter_(1, order, w)
    upto = torch.cumsum(kept, dim=1)
    hit = (upto > s["u"].double().view(R, 1) * upto[:, -1:]) & (kept > 0)
    ids = torch.arange(V, device=x.device)
    token = torch.where(hit, ids, V).amin(dim=1)
    last = torch.where(kept > 0, ids, -1).amax(dim=1)
    return torch.where(token < V, token, last)


# ------------------------------------------------------------------------------------------------- cost
def _distinct(T, V):
    """Expected number of distinct ids among T."""
    v = np.arange(V, dtype=np.float64)
    p = np.log((v + 2.0) / (v + 1.0)) / math.log(V + 1.0)
    return float((1.0 - np.exp(T * np.log1p(-np.minimum(p, 1.0 - 1e-12)))).sum())


def work(case):
    size = _SIZE[case["dtype"]]
    if case["op"] == "embed":
        T, V, D = case["T"], case["V"], case["D"]
        moved = 8 * T + (_distinct(T, V) + T) * D * size
        flops = T * D
        if case["train"]:
            moved += (T + V) * D * size
            flops += (T + V) * D
    elif case["op"] == "dropout":
        moved, flops = 4 * case["numel"] * size, 2 * case["numel"]
    elif case["op"] == "norm":
        n = case["N"] * case["S"] * case["C"]
        moved = (4 if case["train"] else 2) * n * size + (16 if case["train"] else 8) * case["C"]
        flops = (30 if case["train"] else 10) * n
    else:
        n = case["R"] * case["V"]
        moved, flops = n * size + 12 * case["R"], 8 * n
    return {"bytes": float(moved), "flops": float(flops)}


# ------------------------------------------------------------------------------------------------- definition
def exact(case, seed):
    s = prepare(case, seed)
    return {"embed": _exact_embed, "dropout": _exact_dropout, "norm": _exact_norm, "sample": _exact_sample}[s["op"]](s)


def _host(t):
    return t.detach().double().cpu().numpy()


def _exact_embed(s):
    ids, table = s["ids"].cpu().numpy(), _host(s["weight"])
    out = torch.from_numpy(np.take(table, ids, axis=0) * s["scale"])
    if not s["train"]:
        return out
    rows = _host(s["grad"])
    order = np.argsort(ids, kind="stable")
    starts = np.flatnonzero(np.r_[True, np.diff(ids[order]) != 0])
    sums = np.zeros_like(table)
    for a, b in zip(starts, np.r_[starts[1:], len(ids)]):
        sums[ids[order[a]]] = rows[order[a:b]].sum(axis=0)
    if s["padding_idx"] is not None:
        sums[s["padding_idx"]] = 0.0
    return out, torch.from_numpy(sums * s["scale"])


def _exact_dropout(s):
    n = s["x"].numel()
    mask32, thirty_two = np.uint64(0xFFFFFFFF), np.uint64(32)
    q = np.arange((n + 3) // 4, dtype=np.uint64)
    a, b = q & mask32, q >> thirty_two
    c = np.full_like(q, s["offset"] % (1 << 32))
    d = np.full_like(q, s["offset"] // (1 << 32))
    key = [s["seed"] % (1 << 32), s["seed"] // (1 << 32)]
    for _ in range(10):
        first, second = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, c = (second >> thirty_two) ^ b ^ np.uint64(key[0]), (first >> thirty_two) ^ d ^ np.uint64(key[1])
        b, d = second & mask32, first & mask32
        key = [(key[0] + 0x9E3779B9) % (1 << 32), (key[1] + 0xBB67AE85) % (1 << 32)]
    words = np.empty((len(q), 4), dtype=np.uint32)
    for j, col in enumerate((a, b, c, d)):
        words[:, j] = col
    dropped = torch.from_numpy(words.reshape(-1)[:n] < math.floor(s["p"] * 2.0 ** 32 + 0.5))
    return tuple((t.detach().cpu().double() / (1.0 - s["p"])).masked_fill_(dropped, 0.0) for t in (s["x"], s["grad"]))


def _exact_norm(s):
    N, S, C, G = s["N"], s["S"], s["C"], s["G"]
    x, weight, bias = (s[n].detach().double().requires_grad_(s["train"]) for n in ("x", "weight", "bias"))
    with torch.enable_grad():
        by_group = x.transpose(1, 2).reshape(N * G, -1)
        var, mean = torch.var_mean(by_group, dim=1, correction=0, keepdim=True)
        z = ((by_group - mean) / torch.sqrt(var + s["eps"])).view(N, C, S).transpose(1, 2) * weight + bias
        y = {"none": lambda t: t, "relu": torch.relu, "silu": lambda t: t * torch.sigmoid(t),
             "sigmoid": torch.sigmoid}[s["act"]](z)
        if not s["train"]:
            return y
        return (y.detach(),) + torch.autograd.grad(y, (x, weight, bias), s["grad"].double())


def _exact_sample(s):
    x, u = _host(s["logits"]), _host(s["u"])
    R, V = x.shape
    settings = [np.broadcast_to(_host(v) if isinstance(v, torch.Tensor) else np.float64(v), (R,))
                for v in (s["temperature"], s["top_k"], s["top_p"], s["min_p"])]
    out = np.full(R, -1, dtype=np.int64)
    for r in range(R):
        T, k, p, min_p = (float(v[r]) for v in settings)
        ids = np.flatnonzero(x[r] > -math.inf)
        if len(ids) == 0:
            continue
        ids = ids[np.argsort(-x[r, ids], kind="stable")]
        if T == 0.0 or x[r, ids[0]] == math.inf and not (x[r, ids[1:]] == math.inf).any():
            out[r] = ids[0]
            continue
        if k > 0:
            ids = ids[:int(k)]
        with np.errstate(invalid="ignore"):
            w = np.exp((x[r, ids] - x[r, ids[0]]) / T)
        if x[r, ids[0]] == math.inf:
            w = (x[r, ids] == math.inf).astype(np.float64)
        if p < 1.0:
            ahead = np.r_[0.0, np.cumsum(w)[:-1]]
            inside = ahead < p * w.sum()
            ids, w = ids[inside], w[inside]
        ids, w = ids[w >= min_p], w[w >= min_p]
        by_index = np.argsort(ids)
        upto = np.cumsum(w[by_index])
        at = int(np.searchsorted(upto, u[r] * upto[-1], side="right"))
        out[r] = ids[by_index[min(at, len(ids) - 1)]]
    return torch.from_numpy(out)
