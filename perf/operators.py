"""The layer operators as they are timed: cases, inputs, plain form, kernels' calls, cost and 64-bit definition.

What is timed is the work between the matrix products of a transformer layer: layer normalisation and its gradient, the
product of single tokens with 4-bit weights, and the reordering of tokens by expert and back with its gradient.

Three operators:

``layer_norm``  y = (x - mean) * rstd * w + b per row; its gradient gives dx per row and dw, db summed over the rows.
``w4``          y = x W^T for a few tokens, W[m][n] = (q - z) * s with 4-bit q and one s (and z) per group of n.
``experts``     tokens sorted by the expert they are sent to (offsets, positions, order), copied to their places
                (``dispatch``), summed back with the router's weights (``combine``), and the gradient of that sum.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_EPS = 1e-5


def listed():
    return [
        # the norm ahead of the first projection when one sequence is decoded: latency is all there is
        {"name": "norm of one token", "op": "layer_norm", "rows": 1, "cols": 8192, "type": "f16", "wtype": "f16"},
        # the same norm over a batch of training sequences, parameters kept in FP32
        {"name": "norm of a batch", "op": "layer_norm", "rows": 16384, "cols": 4096, "type": "bf16", "wtype": "f32"},
        # backward over a ragged batch of a narrow FP32 model: rows that start on any 4-byte address
        {"name": "norm gradient, odd", "op": "layer_norm_grad", "rows": 4099, "cols": 1001, "type": "f32", "wtype": "f32"},
        # backward of a training batch in bfloat16
        {"name": "norm gradient of a batch", "op": "layer_norm_grad", "rows": 16384, "cols": 6144, "type": "bf16", "wtype": "f32"},
        # one token through a square projection: small enough that latency and the start of the stream count
        {"name": "4-bit, one token", "op": "w4", "batch": 1, "M": 4096, "N": 4096, "group": 128, "zeros": False, "type": "bf16"},
        # one token through the largest projection, fine groups with zero points: a stream of weights
        {"name": "4-bit, one token, wide", "op": "w4", "batch": 1, "M": 16384, "N": 16384, "group": 64, "zeros": True, "type": "f16"},
        # the FP32 path of the library's other products, on a narrow matrix
        {"name": "4-bit, one token, fp32", "op": "w4", "batch": 1, "M": 1000, "N": 4096, "group": 32, "zeros": False, "type": "f32"},
        # thirteen sequences decoded together, sizes that no tile divides and a last group that is cut short
        {"name": "4-bit, thirteen tokens", "op": "w4", "batch": 13, "M": 6143, "N": 8200, "group": 128, "zeros": False, "type": "bf16"},
        # a decode step's tokens handed to many experts
        {"name": "dispatch, decode", "op": "dispatch", "tokens": 32, "topk": 8, "experts": 128, "cols": 4096, "padded": 0.0, "type": "bf16"},
        # a training batch handed to a few experts, the end of it padding
        {"name": "dispatch of a batch", "op": "dispatch", "tokens": 16384, "topk": 2, "experts": 8, "cols": 4096, "padded": 0.06, "type": "bf16"},
        # the experts' answers summed back: FP32, odd sizes
        {"name": "combine, odd", "op": "combine", "tokens": 8191, "topk": 4, "experts": 64, "cols": 1001, "padded": 0.0, "type": "f32"},
        # the gradient of that sum over a training batch: rows for the experts and a dot product per choice
        {"name": "combine gradient", "op": "combine_grad", "tokens": 8192, "topk": 2, "experts": 64, "cols": 6144, "padded": 0.06, "type": "bf16"},
    ]


def _between(rng, lo, hi):
    """A whole number in lo ... hi, even in its logarithm; half of them odd or at least not round."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5:
        n = n // 64 * 64 if n >= 128 else n
    return max(lo, min(hi, n))


def draw(rng):
    kind = rng.choice(["layer_norm", "layer_norm_grad", "w4", "dispatch", "combine", "combine_grad"])
    type_ = rng.choice(["f32", "f16", "bf16"])
    if kind in ("layer_norm", "layer_norm_grad"):
        cols = _between(rng, 64, 16384)
        return {"op": kind, "rows": _between(rng, 1, max(1, min(16384, 16384 * 4096 // cols))), "cols": cols, "type": type_,
                "wtype": rng.choice(["f32", type_])}
    if kind == "w4":
        return {"op": kind, "batch": _between(rng, 1, 16), "M": _between(rng, 512, 16384), "N": _between(rng, 512, 16384),
                "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5, "type": type_}
    topk = rng.randint(1, 8)
    cols = _between(rng, 256, 8192)
    return {"op": kind, "tokens": _between(rng, 1, max(1, min(16384, 8192 * 4096 // (topk * cols)))), "topk": topk,
            "experts": max(topk, _between(rng, 4, 256)), "cols": cols, "padded": rng.choice([0.0, 0.1]), "type": type_}


# ---- inputs ---------------------------------------------------------------

def _activations(g, rows, cols, dtype):
    """Rows as a residual stream holds them: a common offset, and a few columns far larger than the rest."""
    scale = torch.ones(cols, device="cuda")
    scale[torch.randperm(cols, generator=g, device="cuda")[: max(1, cols // 512)]] = 20.0
    return (torch.randn(rows, cols, generator=g, device="cuda") * scale + 0.25).to(dtype)


def _inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed * 7919 + 13)
    dtype, s = _TYPES[case["type"]], {}
    if case["op"] in ("layer_norm", "layer_norm_grad"):
        rows, cols, wtype = case["rows"], case["cols"], _TYPES[case["wtype"]]
        s["x"] = _activations(g, rows, cols, dtype)
        s["w"] = (1.0 + 0.1 * torch.randn(cols, generator=g, device="cuda")).to(wtype)
        s["b"] = (0.1 * torch.randn(cols, generator=g, device="cuda")).to(wtype)
        if case["op"] == "layer_norm_grad":
            s["dy"] = (0.02 * torch.randn(rows, cols, generator=g, device="cuda")).to(dtype)
            var, mean = torch.var_mean(s["x"].float(), dim=1, unbiased=False)
            s["mean"], s["rstd"] = mean.contiguous(), torch.rsqrt(var + _EPS)
        return s
    if case["op"] == "w4":
        M, N, group = case["M"], case["N"], case["group"]
        groups = -(-N // group)
        W = torch.zeros(M, groups * group, device="cuda")
        W[:, :N] = torch.randn(M, N, generator=g, device="cuda") / math.sqrt(N)
        W = W.view(M, groups, group)
        if case["zeros"]:
            lo, hi = W.amin(2).clamp(max=0), W.amax(2).clamp(min=0)
            scale = ((hi - lo) / 15).to(dtype)
            z = (-lo / scale.float()).round().clamp(0, 15)
        else:
            scale = (W.abs().amax(2) / 7).to(dtype)
            z = torch.full_like(scale, 8, dtype=torch.float32)
        q = ((W / scale.float()[..., None]).round() + z[..., None]).clamp(0, 15).to(torch.uint8).view(M, groups * group)
        del W
        # two values a byte, the even column in the low half; rows start every multiple of 16 bytes
        bytes_ = torch.zeros(M, -(-((N + 1) // 2) // 16) * 16, dtype=torch.uint8, device="cuda")
        q[:, N:] = 0
        q = q[:, : N + (N & 1)]
        bytes_[:, : (N + 1) // 2] = q[:, 0::2] | (q[:, 1::2] << 4)
        s["q"], s["scales"], s["zeros"] = bytes_, scale, z.to(torch.uint8) if case["zeros"] else None
        s["x"] = _activations(g, case["batch"], N, dtype)
        return s
    tokens, topk, experts, cols = case["tokens"], case["topk"], case["experts"], case["cols"]
    # a router's choices: some experts are wanted more than others, a token's experts differ, padding goes nowhere
    liking = torch.randn(experts, generator=g, device="cuda")
    logits = torch.randn(tokens, experts, generator=g, device="cuda") + 0.7 * liking
    top = torch.topk(logits, topk, dim=1)
    ids = top.indices.to(torch.int32)
    real = tokens - int(tokens * case["padded"])
    ids[real:] = -1
    s["ids"] = ids.contiguous()
    if case["op"] == "dispatch":
        s["x"] = _activations(g, tokens, cols, dtype)
        return s
    s["weights"] = torch.softmax(top.values, dim=1).contiguous()
    s["pos"] = _sorted(ids, experts)[1]
    s["xs"] = _activations(g, tokens * topk, cols, dtype)
    if case["op"] == "combine_grad":
        s["dy"] = (0.02 * torch.randn(tokens, cols, generator=g, device="cuda")).to(dtype)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    dtype = _TYPES[case["type"]]
    if not own:
        return s
    # what a program that makes these calls holds besides: output buffers and workspaces, allocated once
    from hpcdeepneuralnetworks_amd import blas

    s["blas"] = blas
    op = case["op"]
    if op == "layer_norm":
        s["y"] = torch.empty_like(s["x"])
        s["mean"], s["rstd"] = (torch.empty(case["rows"], device="cuda") for _ in range(2))
    elif op == "layer_norm_grad":
        s["dx"] = torch.empty_like(s["x"])
        s["dw"], s["db"] = torch.empty_like(s["w"]), torch.empty_like(s["w"])
        s["ws"] = torch.empty(max(blas.layer_norm_grad_workspace_bytes(case["rows"], case["cols"]), 16), dtype=torch.uint8, device="cuda")
    elif op == "w4":
        s["y"] = torch.empty(case["batch"], case["M"], dtype=dtype, device="cuda")
    else:
        tokens, topk, experts, cols = case["tokens"], case["topk"], case["experts"], case["cols"]
        if op == "dispatch":
            s["offsets"] = torch.empty(experts + 1, dtype=torch.int32, device="cuda")
            s["pos"] = torch.empty(tokens, topk, dtype=torch.int32, device="cuda")
            s["order"] = torch.full((tokens * topk,), -1, dtype=torch.int32, device="cuda")
            s["out"] = torch.zeros(tokens * topk, cols, dtype=dtype, device="cuda")
            s["ws"] = torch.empty(max(blas.expert_sort_workspace_bytes(tokens, topk, experts), 16), dtype=torch.uint8, device="cuda")
        elif op == "combine":
            s["y"] = torch.empty(tokens, cols, dtype=dtype, device="cuda")
        else:
            s["dxs"] = torch.zeros(tokens * topk, cols, dtype=dtype, device="cuda")
            s["dweights"] = torch.empty(tokens, topk, device="cuda")
    return s


# ---- one pass -------------------------------------------------------------

def _sorted(ids, experts):
    """Offsets of the experts, the place of every choice (-1: none) and the choice at every place (-1: none)."""
    flat = ids.reshape(-1).long()
    sent = (flat >= 0) & (flat < experts)
    key = torch.where(sent, flat, experts)
    order = torch.sort(key, stable=True).indices
    place = torch.empty_like(order)
    place[order] = torch.arange(order.numel(), device=ids.device)
    counts = (key[None, :] == torch.arange(experts, device=ids.device)[:, None]).sum(1)
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=ids.device)
    offsets[1:] = counts.cumsum(0)
    pos = torch.where(sent, place, -1).to(torch.int32).view(ids.shape)
    order = torch.where(sent[order], order, -1).to(torch.int32)
    return offsets, pos, order


def _plain(s):
    case = s["case"]
    op, dtype = case["op"], _TYPES[case["type"]]
    if op == "layer_norm":
        x = s["x"].float()
        mean = x.mean(1, keepdim=True)
        x = x - mean
        rstd = torch.rsqrt((x * x).mean(1, keepdim=True) + _EPS)
        y = x * rstd * s["w"].float() + s["b"].float()
        return {"y": y.to(dtype), "mean": mean[:, 0], "rstd": rstd[:, 0]}
    if op == "layer_norm_grad":
        rstd = s["rstd"][:, None]
        xhat = (s["x"].float() - s["mean"][:, None]) * rstd
        dy = s["dy"].float()
        g = dy * s["w"].float()
        dx = rstd * (g - g.mean(1, keepdim=True) - xhat * (g * xhat).mean(1, keepdim=True))
        wtype = s["w"].dtype
        return {"dx": dx.to(dtype), "dw": (dy * xhat).sum(0).to(wtype), "db": dy.sum(0).to(wtype)}
    if op == "w4":
        M, N, group = case["M"], case["N"], case["group"]
        q = s["q"][:, : (N + 1) // 2]
        W = torch.stack((q & 15, q >> 4), dim=2).view(M, -1)[:, :N].float()
        zero = 8.0 if s["zeros"] is None else s["zeros"].float().repeat_interleave(group, dim=1)[:, :N]
        W = (W - zero) * s["scales"].float().repeat_interleave(group, dim=1)[:, :N]
        return {"y": (s["x"].float() @ W.t()).to(dtype)}
    tokens, topk, cols = case["tokens"], case["topk"], case["cols"]
    if op == "dispatch":
        offsets, pos, order = _sorted(s["ids"], case["experts"])
        rows = s["x"][order.clamp(min=0).long() // topk]
        return {"offsets": offsets, "pos": pos, "order": order, "out": torch.where(order[:, None] >= 0, rows, torch.zeros_like(rows))}
    pos, sent = s["pos"].clamp(min=0).long(), s["pos"] >= 0
    picked = torch.where(sent[..., None], s["xs"][pos].float(), 0.0)
    if op == "combine":
        return {"y": (picked * s["weights"][..., None]).sum(1).to(dtype)}
    dy = s["dy"].float()
    dweights = (picked * dy[:, None, :]).sum(2)
    dxs = torch.zeros(tokens * topk + 1, cols, dtype=dtype, device=dy.device)
    dxs[torch.where(sent, pos, tokens * topk)] = (dy[:, None, :] * s["weights"][..., None]).to(dtype)
    return {"dxs": dxs[:-1], "dweights": dweights}


def run(s):
    if not own:
        return _plain(s)
    case, blas = s["case"], s["blas"]
    op = case["op"]
    if op == "layer_norm":
        blas.layer_norm(case["rows"], case["cols"], s["x"], s["w"], s["b"], _EPS, s["y"], s["mean"], s["rstd"])
        return {"y": s["y"], "mean": s["mean"], "rstd": s["rstd"]}
    if op == "layer_norm_grad":
        blas.layer_norm_grad(case["rows"], case["cols"], s["dy"], s["x"], s["w"], s["mean"], s["rstd"], s["dx"], s["dw"], s["db"], s["ws"])
        return {"dx": s["dx"], "dw": s["dw"], "db": s["db"]}
    if op == "w4":
        blas.w4_gemv(case["batch"], case["M"], case["N"], case["group"], 1.0, s["q"], s["scales"], s["zeros"], s["x"], 0.0, s["y"])
        return {"y": s["y"]}
    tokens, topk, cols = case["tokens"], case["topk"], case["cols"]
    if op == "dispatch":
        blas.expert_sort(tokens, topk, case["experts"], s["ids"], s["offsets"], s["pos"], s["order"], s["ws"])
        blas.expert_gather(tokens, topk, tokens * topk, cols, s["x"], s["pos"], s["out"])
        return {"offsets": s["offsets"], "pos": s["pos"], "order": s["order"], "out": s["out"]}
    if op == "combine":
        blas.expert_combine(tokens, topk, tokens * topk, cols, s["xs"], s["pos"], s["weights"], s["y"])
        return {"y": s["y"]}
    blas.expert_combine_grad(tokens, topk, tokens * topk, cols, s["dy"], s["xs"], s["pos"], s["weights"], s["dxs"], s["dweights"])
    return {"dxs": s["dxs"], "dweights": s["dweights"]}


# ---- cost and definition --------------------------------------------------

def work(case):
    op, e = case["op"], _BYTES[case["type"]]
    if op in ("layer_norm", "layer_norm_grad"):
        n, c, ew = case["rows"] * case["cols"], case["cols"], _BYTES[case["wtype"]]
        if op == "layer_norm":
            return {"bytes": 2 * n * e + 2 * c * ew + 8 * case["rows"], "flops": 8 * n}
        return {"bytes": 3 * n * e + 3 * c * ew + 8 * case["rows"], "flops": 16 * n}
    if op == "w4":
        M, N, groups = case["M"], case["N"], -(-case["N"] // case["group"])
        return {"bytes": M * ((N + 1) // 2) + M * groups * (e + (1 if case["zeros"] else 0)) + case["batch"] * (M + N) * e,
                "flops": 2 * case["batch"] * M * N}
    tokens, topk, cols = case["tokens"], case["topk"], case["cols"]
    real = tokens - int(tokens * case["padded"])
    if op == "dispatch":
        # the choices read, positions, order and offsets written; every token's row read once and written topk times
        return {"bytes": 12 * tokens * topk + 4 * (case["experts"] + 1) + real * (1 + topk) * cols * e, "flops": real * topk}
    if op == "combine":
        return {"bytes": 8 * tokens * topk + (real * topk + tokens) * cols * e, "flops": 2 * real * topk * cols}
    return {"bytes": 12 * tokens * topk + real * (1 + 2 * topk) * cols * e, "flops": 3 * real * topk * cols}


def exact(case, seed):
    s = _inputs(case, seed)
    op = case["op"]
    if op == "layer_norm":
        x = s["x"].double()
        n = case["cols"]
        mean = x.sum(1) / n
        var = ((x - mean[:, None]) ** 2).sum(1) / n
        rstd = 1.0 / torch.sqrt(var + _EPS)
        y = torch.addcmul(s["b"].double(), (x - mean[:, None]) / torch.sqrt(var + _EPS)[:, None], s["w"].double())
        return {"y": y, "mean": mean, "rstd": rstd}
    if op == "layer_norm_grad":
        n, r = case["cols"], s["rstd"].double()[:, None]
        x, dy = (s["x"].double() - s["mean"].double()[:, None]) * r, s["dy"].double()
        dw, db = torch.zeros(2, n, dtype=torch.float64, device=x.device)
        torch.sum(dy * x, 0, out=dw)
        torch.sum(dy, 0, out=db)
        dy *= s["w"].double()
        a, c = dy.sum(1, keepdim=True) / n, (dy * x).sum(1, keepdim=True) / n
        return {"dx": r * (dy - a - x * c), "dw": dw, "db": db}
    if op == "w4":
        M, N, group = case["M"], case["N"], case["group"]
        x, y = s["x"].double(), torch.zeros(case["batch"], M, dtype=torch.float64, device="cuda")
        for g in range(-(-N // group)):
            n0, n1 = g * group, min(N, (g + 1) * group)
            n = torch.arange(n0, n1, device="cuda")
            byte = s["q"][:, n // 2].int()
            q = torch.where(n % 2 == 0, byte % 16, byte // 16).double()
            z = s["zeros"][:, g].double()[:, None] if case["zeros"] else 8
            y += torch.mm(x[:, n0:n1], (q - z).t().contiguous()) * s["scales"][:, g].double()
        return {"y": y}
    tokens, topk, experts = case["tokens"], case["topk"], case["experts"]
    if op == "dispatch":
        order, offsets = [], [0]
        flat = s["ids"].cpu().reshape(-1).tolist()
        where = [[] for _ in range(experts)]
        for slot, i in enumerate(flat):
            if 0 <= i < experts:
                where[i].append(slot)
        for slots in where:
            order += slots
            offsets.append(len(order))
        pos = torch.full((tokens * topk,), -1, dtype=torch.int32)
        pos[torch.tensor(order, dtype=torch.int64)] = torch.arange(len(order), dtype=torch.int32)
        out = torch.zeros(tokens * topk, case["cols"], dtype=torch.float64, device="cuda")
        out[: len(order)] = s["x"].double()[torch.tensor([o // topk for o in order], dtype=torch.int64, device="cuda")]
        order += [-1] * (tokens * topk - len(order))
        return {"offsets": torch.tensor(offsets, dtype=torch.int32), "pos": pos.view(tokens, topk),
                "order": torch.tensor(order, dtype=torch.int32), "out": out}
    xs, w = s["xs"], s["weights"].double()
    if op == "combine":
        y = torch.zeros(tokens, case["cols"], dtype=torch.float64, device="cuda")
        for j in range(topk):
            t = torch.nonzero(s["pos"][:, j] >= 0)[:, 0]
            y[t] += xs[s["pos"][t, j].long()].double() * w[t, j][:, None]
        return {"y": y}
    dxs = torch.zeros(tokens * topk, case["cols"], dtype=torch.float64, device="cuda")
    dweights = torch.zeros(tokens, topk, dtype=torch.float64, device="cuda")
    dy = s["dy"].double()
    for j in range(topk):
        t = torch.nonzero(s["pos"][:, j] >= 0)[:, 0]
        p = s["pos"][t, j].long()
        dxs[p] = dy[t] * w[t, j][:, None]
        dweights[t, j] = (dy[t] * xs[p].double()).sum(1)
    return {"dxs": dxs, "dweights": dweights}
