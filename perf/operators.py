"""What is measured of the network-training operators: the dense layer with its epilogue (`gshell_amd.nn.linear`), the table lookup with its sorted
gradient (`gshell_amd.nn.embedding`) and the global gradient norm with clipping (`gshell_amd.optim.clip_grads`, `grad_norm`)."""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
ACTS = ["none", "relu", "softplus", "silu", "gelu"]
# the largest listed case of each operator bounds what draw() may ask for
LINEAR_MOST_FLOPS = 6.0 * 16384 * 4096 * 4096
EMBED_MOST_BYTES = 600e6
CLIP_MOST_ELEMENTS = 600_000_000


def listed():
    return [
        # one token through a square projection: bound by the weight's bytes and by latency
        {"name": "linear one row bf16", "op": "linear", "type": "bf16", "M": 1, "N": 4096, "K": 4096, "act": "none", "beta": 1.0, "bias": True, "residual": True, "train": False},
        # a small serving batch through an expanding layer
        {"name": "linear 24 rows fp16", "op": "linear", "type": "fp16", "M": 24, "N": 8192, "K": 2048, "act": "silu", "beta": 1.0, "bias": True, "residual": False, "train": False},
        # a training step of a wide layer: the product itself is what bounds it
        {"name": "linear train bf16 wide", "op": "linear", "type": "bf16", "M": 16384, "N": 4096, "K": 4096, "act": "gelu", "beta": 1.0, "bias": True, "residual": True, "train": True},
        # a hidden layer of the signed-distance network (256 wide, softplus with beta 100) over the rows of a grid, forward and backward
        {"name": "linear train fp32 hidden", "op": "linear", "type": "fp32", "M": 131072, "N": 256, "K": 256, "act": "softplus", "beta": 100.0, "bias": True, "residual": False, "train": True},
        # that network's layer behind the skip connection (256 + 39 inputs) at the 50 000 points of the eikonal term
        {"name": "linear fp32 skip layer", "op": "linear", "type": "fp32", "M": 50000, "N": 256, "K": 295, "act": "softplus", "beta": 100.0, "bias": True, "residual": False, "train": False},
        # ragged in every direction, rows that start at odd addresses
        {"name": "linear train fp16 ragged", "op": "linear", "type": "fp16", "M": 1537, "N": 1000, "K": 777, "act": "silu", "beta": 1.0, "bias": True, "residual": True, "train": True},
        # the lookup before a decoding step of eight sequences
        {"name": "embedding 8 rows bf16", "op": "embedding", "type": "bf16", "T": 8, "V": 32000, "D": 4096, "scale": 1.0, "padding": -1, "skew": True, "train": False},
        # a training batch over a large table: few rows are used often, most seldom
        {"name": "embedding train bf16", "op": "embedding", "type": "bf16", "T": 65536, "V": 50000, "D": 1024, "scale": 32.0, "padding": 0, "skew": True, "train": True},
        # a learned code for each of 72 camera poses, looked up for the pixels of a 512 x 512 view batch: long runs of the same row
        {"name": "embedding train fp32 views", "op": "embedding", "type": "fp32", "T": 262144, "V": 72, "D": 32, "scale": 1.0, "padding": -1, "skew": False, "train": True},
        # the gradients of the signed-distance network alone: 16 small tensors, latency
        {"name": "clip fp32 network", "op": "clip", "type": "fp32", "tensors": 16, "elements": 500_737, "norm_only": False, "max_norm": 1.0},
        # the reconstruction's geometry and material gradients: the texture table, deformations, mSDF values, two networks
        {"name": "clip fp32 reconstruction", "op": "clip", "type": "fp32", "tensors": 30, "elements": 22_000_003, "norm_only": False, "max_norm": 1.0},
        # a large network's gradients in one bucket of many tensors
        {"name": "clip bf16 large", "op": "clip", "type": "bf16", "tensors": 300, "elements": 600_000_000, "norm_only": False, "max_norm": 1.0},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "embedding", "clip"])
    kind = rng.choice(["bf16", "fp16", "fp32"])
    if op == "linear":
        # relu without its gradient: one pre-activation that rounds to the other side of zero changes an entry of the gradient as a whole,
        # which says nothing of how exactly either side computes
        train = rng.random() < 0.5
        while True:
            case = {"op": op, "type": kind, "M": _log(rng, 1, 131072), "N": _log(rng, 16, 8192), "K": _log(rng, 16, 8192), "act": rng.choice([a for a in ACTS if a != "relu" or not train]),
                    "beta": rng.choice([1.0, 100.0]), "bias": rng.random() < 0.8, "residual": rng.random() < 0.4, "train": train}
            if rng.random() < 0.5:          # layers are mostly widths of a multiple of 64
                case["N"], case["K"] = max(64, case["N"] // 64 * 64), max(64, case["K"] // 64 * 64)
            # a product in 32 bits costs what one in 16 bits of about eight times the size does
            if work(case)["flops"] * (4 if kind == "fp32" else 1) <= LINEAR_MOST_FLOPS and work(case)["bytes"] <= 4e9:
                return case
    if op == "embedding":
        train = rng.random() < 0.7
        while True:
            V = _log(rng, 2, 131072)
            case = {"op": op, "type": kind, "T": _log(rng, 1, 262144), "V": V, "D": _log(rng, 8, 4096), "scale": rng.choice([1.0, 0.5, 32.0]),
                    "padding": rng.choice([-1, 0, V - 1]), "skew": rng.random() < 0.5, "train": train}
            if rng.random() < 0.5:
                case["D"] = max(8, case["D"] // 8 * 8)
            if work(case)["bytes"] <= EMBED_MOST_BYTES:
                return case
    n = _log(rng, 1, 400)
    return {"op": op, "type": kind, "tensors": n, "elements": _log(rng, max(1000, 4 * n), CLIP_MOST_ELEMENTS // (2 if kind == "fp32" else 1)), "norm_only": rng.random() < 0.3,
            "max_norm": rng.choice([0.5, 1.0, 1e6])}


def _sizes(case):
    """Element counts of a clip case's tensors: from a few elements to a large share of all, odd ones among them."""
    n, total = case["tensors"], case["elements"]
    share = np.exp(np.random.RandomState(n).uniform(0.0, 6.0, n))
    sizes = np.maximum(1, np.floor(share / share.sum() * (total - n)).astype(np.int64))
    sizes[int(np.argmax(sizes))] += total - int(sizes.sum())
    return [int(s) for s in sizes]


def _randn(shape, gen, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32) * scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = DTYPES[case["type"]]
    state = dict(case)
    if case["op"] == "linear":
        M, N, K, train = case["M"], case["N"], case["K"], case["train"]
        # a steep softplus (beta 100) belongs to a network whose pre-activations are a few tenths
        scale = 0.2 if case["act"] == "softplus" and case["beta"] > 10 else 1.0
        state["x"] = _randn((M, K), gen, dtype, scale).requires_grad_(train)
        state["weight"] = _randn((N, K), gen, dtype, 1.0 / math.sqrt(K)).requires_grad_(train)
        state["b"] = _randn((N,), gen, dtype, 0.1 * scale).requires_grad_(train) if case["bias"] else None
        state["r"] = _randn((M, N), gen, dtype, scale).requires_grad_(train) if case["residual"] else None
        state["g"] = _randn((M, N), gen, dtype) if train else None
    elif case["op"] == "embedding":
        T, V, D = case["T"], case["V"], case["D"]
        u = torch.rand(T, generator=gen, device="cuda", dtype=torch.float64)
        # skewed: row v is used about 1 / v as often as the first
        ids = torch.exp(u * math.log(V + 1.0)) - 1.0 if case["skew"] else u * V
        state["ids"] = ids.long().clamp(0, V - 1)
        state["weight"] = _randn((V, D), gen, dtype, 1.0 / math.sqrt(D)).requires_grad_(case["train"])
        state["g"] = _randn((T, D), gen, dtype) if case["train"] else None
    else:
        sizes = _sizes(case)
        state["bucket"] = _randn((sum(sizes),), gen, dtype, 1e-2)
        state["grads"] = list(state["bucket"].split(sizes))
        if not case["norm_only"]:
            state["clipped"] = torch.zeros_like(state["bucket"])
            state["out"] = list(state["clipped"].split(sizes))
    return state


def _act_plain(z, act, beta):
    """The activation and its derivative in 32 bits."""
    if act == "relu":
        return z.clamp(min=0), (z > 0).float()
    if act == "softplus":
        t = torch.exp(-(beta * z).abs())
        return z.clamp(min=0) + torch.log1p(t) / beta, torch.where(z >= 0, torch.ones_like(t), t) / (1 + t)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    if act == "gelu":
        phi = 0.5 * torch.special.erfc(-z * math.sqrt(0.5))
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return z, None


def _linear_plain(s):
    dtype = s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    z = x @ w.t()
    if s["b"] is not None:
        z = z + s["b"].float()
    y, d = _act_plain(z, s["act"], s["beta"])
    if s["r"] is not None:
        y = y + s["r"].float()
    if not s["train"]:
        return y.to(dtype)
    gz = s["g"].float()
    if d is not None:
        gz = gz * d
    grads = [gz @ w, gz.t() @ x]
    if s["b"] is not None:
        grads.append(gz.sum(0))
    return [y.to(dtype)] + [v.to(dtype) for v in grads] + ([s["g"]] if s["r"] is not None else [])


def _linear_own(s):
    from gshell_amd import nn
    act = None if s["act"] == "none" else s["act"]
    if not s["train"]:
        return nn.linear(s["x"], s["weight"], s["b"], s["r"], activation=act, beta=s["beta"])
    y = nn.linear(s["x"], s["weight"], s["b"], s["r"], activation=act, beta=s["beta"])
    leaves = [v for v in (s["x"], s["weight"], s["b"], s["r"]) if v is not None]
    return [y] + list(torch.autograd.grad(y, leaves, s["g"]))


def _embedding_plain(s):
    w, ids = s["weight"], s["ids"]
    y = (w[ids].float() * s["scale"]).to(w.dtype)
    if not s["train"]:
        return y
    d = torch.zeros(w.shape, dtype=torch.float32, device=w.device)
    d.index_add_(0, ids, s["g"].float() * s["scale"])
    if s["padding"] >= 0:
        d[s["padding"]] = 0
    return [y, d.to(w.dtype)]


def _embedding_own(s):
    from gshell_amd import nn
    pad = s["padding"] if s["padding"] >= 0 else None
    y = nn.embedding(s["ids"], s["weight"], scale=s["scale"], padding_idx=pad)
    return [y, torch.autograd.grad(y, s["weight"], s["g"])[0]] if s["train"] else y


def _clip_plain(s):
    norm = torch.stack(torch._foreach_norm(s["grads"], 2, dtype=torch.float32)).square().sum().sqrt()
    if s["norm_only"]:
        return norm
    coef = (s["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    torch._foreach_copy_(s["out"], torch._foreach_mul([g.float() for g in s["grads"]], coef))
    return [norm, s["clipped"]]


def _clip_own(s):
    from gshell_amd import optim
    if s["norm_only"]:
        return optim.grad_norm(s["grads"])
    return [optim.clip_grads(s["grads"], s["max_norm"], out=s["out"]), s["clipped"]]


def run(state):
    op = state["op"]
    if own:
        return _linear_own(state) if op == "linear" else _embedding_own(state) if op == "embedding" else _clip_own(state)
    with torch.no_grad():
        return _linear_plain(state) if op == "linear" else _embedding_plain(state) if op == "embedding" else _clip_plain(state)


def work(case):
    es = 4 if case["type"] == "fp32" else 2
    if case["op"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        once = M * K + N * K + M * N * (2 if case["residual"] else 1) + (N if case["bias"] else 0)
        if not case["train"]:
            return {"bytes": once * es, "flops": 2.0 * M * N * K}
        return {"bytes": (once + M * N + M * K + N * K + (N if case["bias"] else 0)) * es, "flops": 6.0 * M * N * K}
    if case["op"] == "embedding":
        T, V, D = case["T"], case["V"], case["D"]
        fwd = T * 8 + (min(T, V) + T) * D * es
        return {"bytes": fwd + (T + V) * D * es if case["train"] else fwd, "flops": float(T * D) * (2 if case["train"] else 1)}
    n = case["elements"]
    return {"bytes": n * es * (1 if case["norm_only"] else 2), "flops": float(n) * (2 if case["norm_only"] else 3)}


def exact(case, seed):
    """The same outputs from the definitions in 64 bits, with gradients by differentiation."""
    s = prepare(case, seed)
    if case["op"] == "linear":
        leaf = {k: s[k].detach().double().requires_grad_(case["train"]) for k in ("x", "weight", "b", "r") if s[k] is not None}
        z = torch.matmul(leaf["x"], leaf["weight"].t())
        if "b" in leaf:
            z = z + leaf["b"]
        if case["act"] == "relu":
            z = torch.relu(z)
        elif case["act"] == "softplus":
            z = torch.logaddexp(torch.zeros_like(z), z * case["beta"]) / case["beta"]
        elif case["act"] == "silu":
            z = z * torch.sigmoid(z)
        elif case["act"] == "gelu":
            z = 0.5 * z * (1 + torch.erf(z / math.sqrt(2)))
        y = z + leaf["r"] if "r" in leaf else z
        if not case["train"]:
            return y
        return [y.detach()] + list(torch.autograd.grad(y, list(leaf.values()), s["g"].double()))
    if case["op"] == "embedding":
        w = s["weight"].detach().double()
        y = torch.index_select(w, 0, s["ids"]) * case["scale"]
        if not case["train"]:
            return y
        # the gradient as a product with the one-hot matrix, by rows sorted and differences of their running sums
        order = torch.argsort(s["ids"], stable=True)
        counts = torch.bincount(s["ids"], minlength=case["V"])
        ends = torch.cumsum(counts, 0)
        run_sum = torch.cat([torch.zeros(1, case["D"], dtype=torch.float64, device="cuda"), torch.cumsum(s["g"].double()[order], 0)])
        d = (run_sum[ends] - run_sum[ends - counts]) * case["scale"]
        if case["padding"] >= 0:
            d[case["padding"]] = 0
        return [y, d]
    flat = s["bucket"].double()
    norm = torch.linalg.vector_norm(flat)
    if case["norm_only"]:
        return norm
    return [norm, flat * min(1.0, case["max_norm"] / (float(norm) + 1e-6))]
