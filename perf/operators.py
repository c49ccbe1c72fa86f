"""The operators of the fp8 dense path and of mixture-of-experts layers, as cases that can be measured.

Five operators, each in its plain form (elementary torch operations in 32 bits, or in 64 where a border decides) and as the call a
user makes of the framework:

  quant    values -> 8-bit floating point (e4m3) with a scale for each 128 values along K
  gemm     matrix product of two such operands, with bias, residual and activation
  route    router logits -> the experts of each token and their weights
  experts  the experts' two-layer networks on bfloat16 weights, summed over each token's experts
  experts8 the same on 8-bit weights, the hidden layer rounded to 8 bits in between
"""
import math

import numpy as np
import torch

own = False

BLOCK = 128
FP8_MAX = 448.0
TINY = 2.0 ** -126
ACTS = {"none": 0, "relu": 1, "relu6": 2, "gelu": 5}
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------ cases


def listed():
    return [
        # one image's pooled features on their way into the classifier: latency alone
        {"name": "quant_single", "op": "quant", "m": 1, "k": 768, "x": "bf16"},
        # the patch embeddings of a captured batch of 64 images (196 tokens each) before a projection
        {"name": "quant_batch", "op": "quant", "m": 12544, "k": 768, "x": "bf16"},
        # the classifier of one image: 1000 classes
        {"name": "gemm_single", "op": "gemm", "m": 1, "k": 768, "n": 1000, "out": "bf16", "act": "none", "residual": False},
        # the first dense layer behind a 7x7x512 feature map, 64 images: a hundred megabytes of weights for 64 rows
        {"name": "gemm_weights", "op": "gemm", "m": 64, "k": 25088, "n": 4096, "out": "bf16", "act": "relu", "residual": False},
        # attention's output projection at 64 images, added to the residual stream
        {"name": "gemm_project", "op": "gemm", "m": 12544, "k": 768, "n": 768, "out": "bf16", "act": "none", "residual": True},
        # the large end: a wide hidden layer over many rows, its height no multiple of a tile
        {"name": "gemm_large", "op": "gemm", "m": 16200, "k": 4096, "n": 8192, "out": "bf16", "act": "gelu", "residual": False},
        # one image's token count against 64 experts, plain softmax routing
        {"name": "route_small", "op": "route", "t": 196, "e": 64, "k": 2, "x": "bf16", "score": "softmax", "bias": False, "groups": 1, "kept": 1,
         "best": 1, "renorm": True, "scale": 1.0, "padding": 0},
        # 64 images against 256 experts in 8 groups, sigmoid scores with the balancing bias; 9 of the images only fill the batch
        {"name": "route_batch", "op": "route", "t": 12544, "e": 256, "k": 8, "x": "f32", "score": "sigmoid", "bias": True, "groups": 8, "kept": 4,
         "best": 2, "renorm": True, "scale": 2.5, "padding": 1764},
        # one token: what a pooled head of experts costs for a single image
        {"name": "experts_single", "op": "experts", "t": 1, "e": 16, "k": 2, "d": 768, "h": 1536, "act": "gelu", "padding": 0},
        # a layer of experts in a vision transformer at 64 images, 14 of them filling the batch
        {"name": "experts_batch", "op": "experts", "t": 12544, "e": 32, "k": 2, "d": 768, "h": 1536, "act": "gelu", "padding": 2744},
        # a few tokens over many small experts of odd widths: the weights of most experts are read for a row or two
        {"name": "experts8_few", "op": "experts8", "t": 33, "e": 64, "k": 4, "d": 1000, "h": 700, "act": "relu", "padding": 0},
        # many tokens over many experts
        {"name": "experts8_large", "op": "experts8", "t": 8192, "e": 64, "k": 8, "d": 2048, "h": 1024, "act": "gelu", "padding": 0},
    ]


def _log(rng, low, high, step=1):
    v = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    return max(low, min(high, v // step * step or step))


def draw(rng):
    op = rng.choice(["quant", "gemm", "gemm", "route", "experts", "experts8"])
    if op == "quant":
        return {"op": op, "m": _log(rng, 1, 16384), "k": _log(rng, 1, 8192), "x": rng.choice(["bf16", "f32"])}
    if op == "gemm":
        while True:
            c = {"op": op, "m": _log(rng, 1, 16384), "k": _log(rng, 64, 25088), "n": _log(rng, 10, 8192), "out": rng.choice(["bf16", "f32"]),
                 "act": rng.choice(sorted(ACTS)), "residual": rng.random() < 0.4}
            if c["m"] * c["k"] * c["n"] <= 16200 * 4096 * 8192 and (c["m"] + c["n"]) * c["k"] <= 1.2e8:
                return c
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        e = groups * _log(rng, 4, 512 // groups)
        kept = rng.randint(max(1, groups // 2), groups)
        return {"op": op, "t": _log(rng, 1, 16384), "e": e, "k": rng.randint(1, min(8, kept * (e // groups))), "x": rng.choice(["bf16", "f32"]),
                "score": rng.choice(["softmax", "sigmoid"]), "bias": rng.random() < 0.5, "groups": groups, "kept": kept, "best": rng.choice([1, 2]),
                "renorm": rng.random() < 0.7, "scale": rng.choice([1.0, 2.5]), "padding": 0}
    step = 8 if op == "experts" else 1
    while True:
        e = _log(rng, 2, 64)
        c = {"op": op, "t": _log(rng, 1, 12544), "e": e, "k": rng.randint(1, min(8, e)), "d": _log(rng, 64, 2048, step), "h": _log(rng, 64, 2048, step),
             "act": rng.choice(["relu", "gelu"]), "padding": 0}
        c["padding"] = rng.choice([0, 0, c["t"] // 5])
        if c["t"] * c["k"] * c["d"] * c["h"] <= 8192 * 8 * 2048 * 1024:
            return c


def _up(n, to):
    return -(-n // to) * to


def work(c):
    if c["op"] == "quant":
        n = c["m"] * c["k"]
        return {"bytes": n * TYPES[c["x"]].itemsize + c["m"] * _up(c["k"], BLOCK) * (1 + 4 / BLOCK), "flops": 2 * n}
    if c["op"] == "gemm":
        m, n, k = c["m"], c["n"], c["k"]
        out = TYPES[c["out"]].itemsize
        scales = 4 * _up(k, BLOCK) // BLOCK * (m + _up(n, BLOCK) // BLOCK)
        return {"bytes": (m + n) * k + scales + 4 * n + m * n * (out + (2 if c["residual"] else 0)), "flops": 2 * m * n * k}
    if c["op"] == "route":
        n = c["t"] * c["e"]
        return {"bytes": n * TYPES[c["x"]].itemsize + c["t"] * c["k"] * 8 + (4 * c["e"] if c["bias"] else 0), "flops": 8 * n}
    rows = (c["t"] - c["padding"]) * c["k"]
    hit = c["e"] * (1 - (1 - c["k"] / c["e"]) ** (c["t"] - c["padding"]))  # experts that some token goes to, on the average
    size = 2 if c["op"] == "experts" else 1 + 4 / BLOCK ** 2
    return {"bytes": hit * (2 * c["d"] * c["h"] * size + 4 * (c["d"] + c["h"])) + 4 * c["t"] * c["d"] + 8 * c["t"] * c["k"],
            "flops": 4 * rows * c["d"] * c["h"]}


# ----------------------------------------------------------------- inputs


def _activations(gen, m, k, kind):
    """Values as they come out of a normalisation: near unit size, some channels much larger than the rest."""
    x = torch.randn(m, k, device="cuda", generator=gen)
    wide = 1 + 9 * (torch.rand(k, device="cuda", generator=gen) < 0.02).float()
    return (x * wide).to(TYPES[kind])


def _blocks(x):
    """[..., K] in 32 bits -> [..., K/128, 128], the last block filled with zeros."""
    k = x.shape[-1]
    x = torch.nn.functional.pad(x, (0, _up(k, BLOCK) - k))
    return x.reshape(*x.shape[:-1], -1, BLOCK)


def _round8(x):
    """What the operator `quant` computes, plainly: (e4m3 values [M, K up to whole blocks], scales [blocks, M])."""
    b = _blocks(x.float())
    s = (b.abs().amax(-1).double() / FP8_MAX).clamp_min(TINY).float()  # in 64 bits first: a division by a plain number is a product in 32
    return (b / s[..., None]).to(torch.float8_e4m3fn).reshape(*b.shape[:-2], -1), s.movedim(-1, -2).contiguous()


def _weights8(gen, shape):
    """A weight [..., N, K] as the fp8 layers hold it: e4m3, K filled up to whole blocks, a scale for each 128 x 128 values."""
    n, k = shape[-2:]
    w = torch.randn(shape, device="cuda", generator=gen) * k ** -0.5
    w = torch.nn.functional.pad(w, (0, _up(k, BLOCK) - k, 0, _up(n, BLOCK) - n))
    w = w.reshape(*shape[:-2], w.shape[-2] // BLOCK, BLOCK, w.shape[-1] // BLOCK, BLOCK)
    s = (w.abs().amax((-3, -1)) / FP8_MAX).clamp_min(TINY)
    q = (w / s[..., :, None, :, None]).to(torch.float8_e4m3fn).reshape(*shape[:-2], _up(n, BLOCK), -1)
    return q[..., :n, :].contiguous(), s


def _chosen(gen, t, e, k, padding):
    """Experts and weights as a router gives them, some experts more popular than others; no expert (-1) for the rows that fill the batch."""
    logits = torch.randn(t, e, device="cuda", generator=gen) + 0.5 * torch.randn(e, device="cuda", generator=gen)
    w, ids = logits.softmax(-1).topk(k, -1)
    w, ids = w / w.sum(-1, keepdim=True), ids.to(torch.int32)
    if padding:
        ids[t - padding:] = -1
        w[t - padding:] = 0
    return ids.contiguous(), w.contiguous()


def prepare(c, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    if c["op"] == "quant":
        return {"c": c, "x": _activations(gen, c["m"], c["k"], c["x"])}
    if c["op"] == "gemm":
        a, sa = _round8(_activations(gen, c["m"], c["k"], "f32"))
        b, sb = _weights8(gen, (c["n"], c["k"]))
        bias = torch.randn(c["n"], device="cuda", generator=gen) * 0.1
        res = torch.randn(c["m"], c["n"], device="cuda", generator=gen).to(torch.bfloat16) if c["residual"] else None
        return {"c": c, "a": a, "sa": sa, "b": b, "sb": sb, "bias": bias, "res": res}
    if c["op"] == "route":
        x = torch.randn(c["t"], c["e"], device="cuda", generator=gen) * 1.5 + 0.5 * torch.randn(c["e"], device="cuda", generator=gen)
        if c["padding"]:
            x[c["t"] - c["padding"]:] = -math.inf
        bias = torch.randn(c["e"], device="cuda", generator=gen) * 0.1 if c["bias"] else None
        return {"c": c, "x": x.to(TYPES[c["x"]]), "bias": bias}
    t, e, d, h = c["t"], c["e"], c["d"], c["h"]
    s = {"c": c, "x": _activations(gen, t, d, "bf16")}
    s["ids"], s["w"] = _chosen(gen, t, e, c["k"], c["padding"])
    s["b1"] = torch.randn(e, h, device="cuda", generator=gen) * 0.1
    s["b2"] = torch.randn(e, d, device="cuda", generator=gen) * 0.1
    if c["op"] == "experts":
        # [expert][outputs][inputs], the inputs filled up to a multiple of 64 as in every dense layer of the framework
        for name, n, k in (("w1", h, d), ("w2", d, h)):
            w = torch.zeros(e, n, _up(k, 64), dtype=torch.bfloat16, device="cuda")
            w[..., :k] = torch.randn(e, n, k, device="cuda", generator=gen) * k ** -0.5
            s[name] = w
    else:
        s["w1"], s["s1"] = _weights8(gen, (e, h, d))
        s["w2"], s["s2"] = _weights8(gen, (e, d, h))
    return s


# ------------------------------------------------------------- the operators


def run(s):
    return (_own if own else _plain)[s["c"]["op"]](s)


def _act(y, act):
    if act == "relu":
        return y.clamp_min(0)
    if act == "relu6":
        return y.clamp(0, 6)
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
    return y


def _plain_quant(s):
    return list(_round8(s["x"]))


def _values(q, s):
    """e4m3 rows and their scales [blocks, M] as 32-bit values."""
    b = q.float().reshape(*q.shape[:-1], -1, BLOCK)
    return (b * s.movedim(-2, -1)[..., None]).reshape(q.shape)


def _weight_values(q, s):
    n = q.shape[-2]
    return q.float() * s.repeat_interleave(BLOCK, -2)[..., :n, :].repeat_interleave(BLOCK, -1)


def _plain_gemm(s):
    c = s["c"]
    y = _values(s["a"], s["sa"]) @ _weight_values(s["b"], s["sb"]).t() + s["bias"]
    if s["res"] is not None:
        y = y + s["res"].float()
    return _act(y, c["act"]).to(TYPES[c["out"]])


def _plain_route(s):
    # in 64 bits throughout: which expert is chosen hangs on the last digit where two scores are close
    c, x = s["c"], s["x"].double()
    open_ = ~x.isnan() & (x > -math.inf)
    if c["score"] == "softmax":
        top = x.masked_fill(~open_, -math.inf).amax(-1, keepdim=True)
        p = torch.where(x == top, torch.zeros_like(x), x - top).exp().masked_fill(~open_, 0)
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    else:
        p = torch.sigmoid(x).masked_fill(~open_, 0)
    key = (p if s["bias"] is None else p + s["bias"].double()).masked_fill(~open_, -math.inf)
    if c["groups"] > 1:
        g = key.reshape(c["t"], c["groups"], -1)
        best = g.sort(dim=-1, descending=True)[0][..., :c["best"]]
        total = best.masked_fill(best == -math.inf, 0).sum(-1).masked_fill(best[..., 0] == -math.inf, -math.inf)
        at = total.sort(dim=-1, descending=True, stable=True)[1][:, :c["kept"]]
        kept = torch.zeros_like(total, dtype=torch.bool).scatter_(1, at, True)
        key = g.masked_fill(~kept[..., None], -math.inf).reshape(c["t"], c["e"])
    v, ids = key.sort(dim=-1, descending=True, stable=True)
    v, ids = v[:, :c["k"]], ids[:, :c["k"]]
    none = v == -math.inf
    w = p.gather(1, ids).masked_fill(none, 0)
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
    return {"ids": ids.masked_fill(none, -1).to(torch.int32), "weights": (w * c["scale"]).float()}


def _rows_by_expert(ids, e):
    """Blocks of rows, each of one expert: (expert of each block, the assignment at each place or -1). Sizes that follow from the shapes alone."""
    n = ids.numel()
    size = 1 if n <= 4 * e else 64
    flat = ids.reshape(-1).long()
    key = torch.where(flat < 0, e, flat)
    order = key.sort(stable=True)[1]
    count = torch.zeros(e + 1, dtype=torch.long, device=ids.device).scatter_add_(0, key, torch.ones_like(key))
    blocks = (count + size - 1) // size
    blocks[e] = 0
    first = blocks.cumsum(0) - blocks
    begin = count.cumsum(0) - count
    of = key[order]
    place = first[of] * size + torch.arange(n, device=ids.device) - begin[of]
    total = n // size + min(n, e)
    rows = torch.full((total * size + 1,), -1, dtype=torch.long, device=ids.device)
    rows[torch.where(of == e, total * size, place)] = order
    expert = torch.searchsorted(blocks.cumsum(0), torch.arange(total, device=ids.device), right=True).clamp_max(e - 1)
    return expert, rows[:-1].reshape(total, size)


def _sum_of_experts(s, rows, y):
    """Each token's weighted sum over its experts' rows."""
    c = s["c"]
    out = torch.zeros(c["t"] * c["k"] + 1, c["d"], device=y.device)
    at = rows.reshape(-1)
    out[torch.where(at < 0, c["t"] * c["k"], at)] = y.reshape(-1, c["d"])
    return (out[:-1].reshape(c["t"], c["k"], -1) * s["w"][..., None]).sum(1).to(torch.bfloat16)


def _plain_experts(s):
    c = s["c"]
    expert, rows = _rows_by_expert(s["ids"], c["e"])
    x = s["x"].float()[rows.clamp_min(0) // c["k"]]
    h = torch.bmm(x, s["w1"][expert, :, :c["d"]].float().transpose(1, 2)) + s["b1"][expert][:, None]
    y = torch.bmm(_act(h, c["act"]), s["w2"][expert, :, :c["h"]].float().transpose(1, 2)) + s["b2"][expert][:, None]
    return _sum_of_experts(s, rows, y)


def _plain_experts8(s):
    c = s["c"]
    expert, rows = _rows_by_expert(s["ids"], c["e"])
    x = _values(*_round8(s["x"]))[rows.clamp_min(0) // c["k"]]
    h = torch.bmm(x, _weight_values(s["w1"], s["s1"])[expert].transpose(1, 2)) + s["b1"][expert][:, None]
    y = torch.bmm(_values(*_round8(_act(h, c["act"]))), _weight_values(s["w2"], s["s2"])[expert].transpose(1, 2)) + s["b2"][expert][:, None]
    return _sum_of_experts(s, rows, y)


_plain = {"quant": _plain_quant, "gemm": _plain_gemm, "route": _plain_route, "experts": _plain_experts, "experts8": _plain_experts8}


def _ext():
    from tensorflow_web_deploy_amd.ops.native import ext
    return ext()


def _own_quant(s):
    m, k = s["x"].shape
    q = torch.empty(m, _up(k, BLOCK), dtype=torch.float8_e4m3fn, device="cuda")
    sc = torch.empty(_up(k, BLOCK) // BLOCK, m, device="cuda")
    _ext().quant_fp8(s["x"], q, sc, 1)
    return [q, sc]


def _own_gemm(s):
    c = s["c"]
    y = torch.empty(c["m"], c["n"], dtype=TYPES[c["out"]], device="cuda")
    _ext().gemm_fp8(s["a"], s["sa"], s["b"], s["sb"], y, s["bias"], s["res"], ACTS[c["act"]])
    return y


def _own_route(s):
    c = s["c"]
    ids = torch.empty(c["t"], c["k"], dtype=torch.int32, device="cuda")
    w = torch.empty(c["t"], c["k"], device="cuda")
    _ext().moe_route(s["x"], s["bias"], ids, w, 0 if c["score"] == "softmax" else 1, c["groups"], c["kept"], c["best"], c["renorm"], c["scale"])
    return {"ids": ids, "weights": w}


def _own_experts(s):
    c = s["c"]
    y = torch.empty(c["t"], c["d"], dtype=torch.bfloat16, device="cuda")
    _ext().moe_mlp_bf16(s["x"], s["ids"], s["w"], s["w1"], s["b1"], s["w2"], s["b2"], y, None, ACTS[c["act"]])
    return y


def _own_experts8(s):
    c = s["c"]
    y = torch.empty(c["t"], c["d"], dtype=torch.bfloat16, device="cuda")
    _ext().moe_mlp_fp8(s["x"], s["ids"], s["w"], s["w1"], s["s1"], s["b1"], s["w2"], s["s2"], s["b2"], y, None, ACTS[c["act"]])
    return y


_own = {"quant": _own_quant, "gemm": _own_gemm, "route": _own_route, "experts": _own_experts, "experts8": _own_experts8}


# ------------------------------------------------------- by definition, in 64 bits


def _exact8(v):
    """Rows in 64 bits -> the values that their e4m3 form stands for, and that form: each block of 128 is divided by its scale (a 32-bit number) to a
    32-bit quotient, which is rounded to the nearest of the 8-bit values, the even one of two. Values of bfloat16 meet ties often, so each of the two
    roundings belongs to the definition."""
    m, k = v.shape
    full = torch.zeros(m, _up(k, BLOCK), dtype=torch.float64, device=v.device)
    full[:, :k] = v
    back, eighth, scales = torch.empty_like(full), torch.empty_like(full), []
    for j in range(0, full.shape[1], BLOCK):
        part = full[:, j:j + BLOCK]
        sc = torch.clamp((part.abs().max(1).values / FP8_MAX).float(), min=TINY).double()
        q = (part / sc[:, None]).float().double()
        # the step between 8-bit values is an eighth of the power of two below, and 2^-9 under 2^-6
        step = torch.exp2(torch.floor(torch.log2(q.abs().clamp_min(2.0 ** -6))) - 3)
        q = torch.round(q / step) * step
        eighth[:, j:j + BLOCK], back[:, j:j + BLOCK] = q, q * sc[:, None]
        scales.append(sc)
    return back, eighth, torch.stack(scales)


def _exact_act(y, act):
    return {"none": lambda v: v, "relu": torch.relu, "relu6": lambda v: torch.minimum(torch.relu(v), torch.full_like(v, 6)),
            "gelu": lambda v: v * 0.5 * torch.erfc(-v / math.sqrt(2))}[act](y)


def _exact_weight(q, s):
    q = q.double()
    for i in range(s.shape[0]):
        for j in range(s.shape[1]):
            q[i * BLOCK:(i + 1) * BLOCK, j * BLOCK:(j + 1) * BLOCK] *= s[i, j].double()
    return q


def exact(c, seed):
    s = prepare(c, seed)
    if c["op"] == "quant":
        _, q, sc = _exact8(s["x"].double())
        return [q, sc]
    if c["op"] == "gemm":
        a = s["a"].double()
        for j in range(s["sa"].shape[0]):
            a[:, j * BLOCK:(j + 1) * BLOCK] *= s["sa"][j].double()[:, None]
        w = _exact_weight(s["b"], s["sb"])
        y = torch.empty(c["m"], c["n"], dtype=torch.float64, device="cuda")
        for i in range(0, c["m"], 4096):
            z = a[i:i + 4096] @ w.t() + s["bias"].double()
            if s["res"] is not None:
                z += s["res"][i:i + 4096].double()
            y[i:i + 4096] = _exact_act(z, c["act"])
        return y
    if c["op"] == "route":
        return {"ids": None, "weights": _exact_route(c, s)}
    x = s["x"].double() if c["op"] == "experts" else _exact8(s["x"].double())[0]
    y = torch.zeros(c["t"], c["d"], dtype=torch.float64, device="cuda")
    for i in range(c["e"]):
        t, j = torch.nonzero(s["ids"] == i, as_tuple=True)
        if not len(t):
            continue
        if c["op"] == "experts":
            h = _exact_act(x[t] @ s["w1"][i, :, :c["d"]].double().t() + s["b1"][i].double(), c["act"])
            z = h @ s["w2"][i, :, :c["h"]].double().t()
        else:
            h = _exact_act(x[t] @ _exact_weight(s["w1"][i], s["s1"][i]).t() + s["b1"][i].double(), c["act"])
            z = _exact8(h)[0] @ _exact_weight(s["w2"][i], s["s2"][i]).t()
        y.index_add_(0, t, (z + s["b2"][i].double()) * s["w"][t, j].double()[:, None])
    return y


def _exact_route(c, s):
    x = s["x"].double().cpu().numpy()
    bias = np.zeros(c["e"]) if s["bias"] is None else s["bias"].double().cpu().numpy()
    shut = np.isnan(x) | np.isneginf(x)
    live = np.where(shut, -np.inf, x)
    with np.errstate(all="ignore"):
        if c["score"] == "softmax":
            top = live.max(1, keepdims=True)
            p = np.exp(live - np.where(np.isneginf(top), 0, top))
            p = np.where(shut, 0, p) / np.maximum(p.sum(1, keepdims=True), 1e-300)
        else:
            p = np.where(shut, 0, 1 / (1 + np.exp(-live)))
    key = np.where(shut, -np.inf, p + bias)
    if c["groups"] > 1:
        g = key.reshape(c["t"], c["groups"], -1)
        best = -np.sort(-g, axis=2)[:, :, :c["best"]]
        total = np.where(np.isneginf(best[:, :, 0]), -np.inf, np.where(np.isneginf(best), 0, best).sum(2))
        rank = np.argsort(np.argsort(-total, axis=1, kind="stable"), axis=1, kind="stable")
        key = np.where(rank[:, :, None] < c["kept"], g, -np.inf).reshape(c["t"], c["e"])
    at = np.argsort(-key, axis=1, kind="stable")[:, :c["k"]]
    w = np.where(np.isneginf(np.take_along_axis(key, at, 1)), 0, np.take_along_axis(p, at, 1))
    if c["renorm"]:
        w = w / np.maximum(w.sum(1, keepdims=True), 1e-300)
    return w * c["scale"]
