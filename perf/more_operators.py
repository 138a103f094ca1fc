"""The dense linear layer and the routing from logits as timed cases.

Two families, each one pass of a public entry point as a program calls it:

- ``linear``: activations times 16-bit weights with bias, activation and
  residual in the epilogue (``dense_linear``); with ``train`` its gradients too;
- ``route``: experts chosen from a router's logits, by groups where asked, and
  their weights (``moe_route_logits``); with ``train`` the weights' gradient too.

``own`` chooses between the plain form (elementary torch operations in 32
bits) and the framework's calls.  ``exact`` gives the same outputs in 64 bits.
"""

from __future__ import annotations

import math
import os
import sys

import torch

own = False

_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "vllm-cmp170hx_amd")

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def _calls():
    """The framework's operators (imported only where they are called)."""
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from vllm_mi355x.kernels import dense, moe
    return dense, moe


# ---- cases ---------------------------------------------------------------------


def _linear(name, k, n, rows, dtype, *, out=None, activation="none", bias=False, residual=False,
            clamp=0.0, gap=0, train=False):
    """n: columns of the output (a gated activation has twice as many weight
    rows); gap: elements between the rows of a larger buffer that x is a part of."""
    return {"name": name, "family": "linear", "k": k, "n": n, "rows": rows, "dtype": dtype,
            "out": out or dtype, "activation": activation, "bias": bias, "residual": residual,
            "clamp": clamp, "gap": gap, "train": train}


def _route(name, rows, experts, topk, dtype, *, scoring="sigmoid", bias=False, groups=1,
           topk_groups=1, renormalize=True, scale=1.0, padded=0.0, train=False):
    return {"name": name, "family": "route", "rows": rows, "experts": experts, "topk": topk,
            "dtype": dtype, "scoring": scoring, "bias": bias, "groups": groups,
            "topk_groups": topk_groups, "renormalize": renormalize, "scale": scale,
            "padded": padded, "train": train}


def listed():
    return [
        # One token's logits in a decode step: a small matrix, 32-bit outputs.
        _linear("linear_router_1", 7168, 257, 1, "bf16", out="fp32"),
        # One token through a shared expert's gate and up projections.
        _linear("linear_decode_1", 4096, 14336, 1, "bf16", activation="swiglu"),
        # A decode batch through a matrix whose sizes are no tile's multiple.
        _linear("linear_batch_20", 2592, 5003, 20, "fp16", activation="gelu", bias=True,
                residual=True),
        # A short prompt through a shared expert's down projection, added to the
        # routed experts' sum.
        _linear("linear_rows_400", 14336, 4096, 400, "bf16", residual=True),
        # A whole prefill chunk through the largest matrix.
        _linear("linear_prefill_2048", 8192, 28672, 2048, "bf16", activation="silu", bias=True),
        # A router's training step: 32-bit logits of a whole batch, with the
        # gradients of the activations and the router's weights.
        _linear("linear_router_train_4096", 4096, 288, 4096, "bf16", out="fp32", train=True),
        # A training step of a small feed-forward layer on a ragged batch.
        _linear("linear_train_1000", 2048, 768, 1000, "fp16", activation="gelu_tanh", bias=True,
                residual=True, train=True),
        # A training step of a shared expert's gate and up projections.
        _linear("linear_train_4096", 4096, 14336, 4096, "bf16", activation="swiglu", train=True),
        # One token's experts in a decode step: the smallest call.
        _route("route_decode_1", 1, 256, 8, "fp32", bias=True, groups=8, topk_groups=4, scale=2.5),
        # A prefill chunk's experts by softmax from 16-bit logits (which tie).
        _route("route_prefill_2048", 2048, 128, 8, "bf16", scoring="softmax"),
        # A micro batch of a router's training step.
        _route("route_train_200", 200, 128, 8, "fp32", scoring="softmax", renormalize=False,
               train=True),
        # A whole training batch, some of it padding, by groups with a bias for
        # balance.
        _route("route_train_65536", 65536, 256, 8, "fp32", bias=True, groups=8, topk_groups=4,
               scale=2.5, padded=0.1, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _log_size(rng, lo, hi):
    """Log-uniform in [lo, hi]: a multiple of 64, of 8, or any size."""
    unit = rng.choice([64, 64, 8, 1])
    return unit * _log_int(rng, -(-lo // unit), hi // unit)


_ACTIVATIONS = ["none", "none", "relu", "gelu", "gelu_tanh", "silu", "swiglu", "swiglu"]
# What one drawn case may cost: the largest listed ones.
_MAX_PRODUCT = 2048 * 8192 * 28672
_MAX_WEIGHTS = 8192 * 28672
_MAX_LOGITS = 65536 * 256


def draw(rng):
    while True:
        train = rng.choice([False, False, True])
        if rng.choice([True, True, False]):
            dtype, activation = rng.choice(["bf16", "fp16"]), rng.choice(_ACTIVATIONS)
            case = _linear("", _log_size(rng, 64, 16384), _log_size(rng, 16, 28672),
                           _log_int(rng, 1, 8192), dtype,
                           out=rng.choice([dtype, dtype, "fp32"]), activation=activation,
                           bias=rng.choice([False, True]), residual=rng.choice([False, True]),
                           clamp=7.0 if activation == "swiglu" and rng.random() < 0.5 else 0.0,
                           gap=rng.choice([0, 0, 64, 3]), train=train)
            weights = case["k"] * case["n"] * (2 if activation == "swiglu" else 1)
            fits = (weights <= _MAX_WEIGHTS
                    and weights * case["rows"] * (3 if train else 1) <= _MAX_PRODUCT)
        else:
            groups = rng.choice([1, 1, 2, 4, 8])
            experts = groups * _log_int(rng, max(2, 8 // groups), 512 // groups)
            topk_groups = rng.randint(1, groups)
            choosable = topk_groups * (experts // groups)
            case = _route("", _log_int(rng, 1, 65536), experts, rng.randint(1, min(10, choosable)),
                          rng.choice(["bf16", "fp16", "fp32"]),
                          scoring=rng.choice(["softmax", "sigmoid"]),
                          bias=rng.choice([False, True]), groups=groups, topk_groups=topk_groups,
                          renormalize=rng.choice([True, True, False]),
                          scale=rng.choice([1.0, 2.5]), padded=rng.choice([0.0, 0.1, 0.5]),
                          train=train)
            fits = case["rows"] * experts <= _MAX_LOGITS
        if fits:
            del case["name"]
            return case


# ---- inputs --------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def _activations(g, rows, k, dtype):
    """Normal values with the few large channels that activations have."""
    x = _normal(g, rows, k)
    x *= 1.0 + 7.0 * (torch.rand(k, device="cuda", generator=g) < 0.005)
    return x.to(_DTYPES[dtype])


def _weights(g, n, k, dtype):
    """Normal weights, rows of unlike size among them, that keep a unit input
    near unit size."""
    w = torch.empty(n, k, dtype=_DTYPES[dtype], device="cuda")
    step = max(1, (1 << 25) // k)
    for r0 in range(0, n, step):
        r1 = min(n, r0 + step)
        w[r0:r1] = _normal(g, r1 - r0, k) * (torch.exp(0.5 * _normal(g, r1 - r0, 1)) / math.sqrt(k))
    return w


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case, "leaves": []}
    if case["family"] == "linear":
        k, n, rows, dtype = case["k"], case["n"], case["rows"], case["dtype"]
        lines = 2 * n if case["activation"] == "swiglu" else n
        s["x"] = _activations(g, rows, k + case["gap"], dtype)[:, :k]
        s["w"] = _weights(g, lines, k, dtype)
        s["bias"] = (0.1 * _normal(g, lines)).to(_DTYPES[dtype]) if case["bias"] else None
        s["residual"] = _normal(g, rows, n).to(_DTYPES[case["out"]]) if case["residual"] else None
        if case["train"]:
            s["leaves"] = [name for name in ("x", "w", "bias", "residual") if s[name] is not None]
            # the gradient of a mean over the rows, under a loss scale
            s["upstream"] = _normal(g, rows, n).to(_DTYPES[case["out"]])
    else:
        t, e = case["rows"], case["experts"]
        # A router's logits: some experts liked by all rows
        logits = _normal(g, t, e)
        logits += 0.5 * _normal(g, e)
        s["logits"] = logits.to(_DTYPES[case["dtype"]])
        s["bias"] = 0.05 * _normal(g, e) if case["bias"] else None
        s["is_padding"] = None
        if case["padded"]:
            s["is_padding"] = torch.rand(t, device="cuda", generator=g) < case["padded"]
        if case["train"]:
            s["leaves"] = ["logits"]
            s["upstream"] = _normal(g, t, case["topk"])
    for name in s["leaves"]:
        s[name] = s[name].detach().requires_grad_()
    return s


# ---- the plain forms, 32 bits ----------------------------------------------------


def _sigmoid(v):
    e = torch.exp(-v.abs())
    return torch.where(v >= 0, 1 / (1 + e), e / (1 + e))


_TANH_A, _TANH_B = math.sqrt(2 / math.pi), 0.044715


def _activated(activation, z):
    """(act(z), its slope) of elementwise activations."""
    if activation == "none":
        return z, torch.ones_like(z)
    if activation == "relu":
        return z * (z > 0), (z > 0).float()
    if activation == "silu":
        s = _sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    if activation == "gelu":
        half = 0.5 * (1 + torch.erf(z / math.sqrt(2)))
        return z * half, half + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    u = _TANH_A * (z + _TANH_B * z * z * z)
    half = _sigmoid(2 * u)  # (1 + tanh u) / 2
    return z * half, half + z * half * (1 - half) * 2 * _TANH_A * (1 + 3 * _TANH_B * z * z)


def _plain_linear(s):
    case = s["case"]
    out, dtype = _DTYPES[case["out"]], _DTYPES[case["dtype"]]
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    gated = case["activation"] == "swiglu"
    if gated:
        limit = case["clamp"] or math.inf
        g, u = z[:, :case["n"]], z[:, case["n"]:]
        in_g, in_u = g <= limit, u.abs() <= limit
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        h, slope = _activated("silu", g)
        y = h * u
    else:
        y, slope = _activated(case["activation"], z)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    y = y.to(out)
    if not case["train"]:
        return y
    dy = s["upstream"].float()
    dz = torch.cat([dy * u * slope * in_g, dy * h * in_u], 1) if gated else dy * slope
    r = {"y": y, "x": (dz @ w).to(dtype), "w": (dz.t() @ x).to(dtype)}
    if s["bias"] is not None:
        r["bias"] = dz.sum(0).to(dtype)
    if s["residual"] is not None:
        r["residual"] = s["upstream"].clone()
    return r


def _first(keys, count):
    """The places of the `count` largest of each row, largest first, ties to the
    lower place."""
    return keys.sort(dim=1, descending=True, stable=True).indices[:, :count]


def _plain_route(s):
    case = s["case"]
    l = s["logits"].float()
    t, e, groups = case["rows"], case["experts"], case["groups"]
    if case["scoring"] == "softmax":
        z = torch.exp(l - l.amax(1, keepdim=True))
        score = z / z.sum(1, keepdim=True)
    else:
        score = _sigmoid(l)
    if s["bias"] is None:
        keys = l  # in the scores' order
    else:  # 64 bits: keys lie close to each other
        d = l.double()
        if case["scoring"] == "softmax":
            d = torch.exp(d - d.amax(1, keepdim=True))
            d = d / d.sum(1, keepdim=True)
        else:
            d = 1 / (1 + torch.exp(-d))
        keys = d + s["bias"].double()
    if groups > 1:
        by_group = keys.view(t, groups, e // groups)
        top = by_group.sort(dim=2, descending=True).values[:, :, :1 if s["bias"] is None else 2]
        kept = torch.zeros(t, groups, dtype=torch.bool, device=l.device)
        kept.scatter_(1, _first(top.sum(2), case["topk_groups"]), True)
        keys = torch.where(kept[:, :, None], by_group, -math.inf).view(t, e)
    ids = _first(keys, case["topk"])
    chosen = score.gather(1, ids)
    total = chosen.sum(1, keepdim=True)
    part = chosen / total if case["renormalize"] else chosen
    weights = part * case["scale"]
    kept = torch.ones(t, 1, dtype=torch.bool, device=l.device)
    if s["is_padding"] is not None:
        kept = ~s["is_padding"][:, None]
    out = {"weights": weights * kept, "ids": torch.where(kept, ids, -1).to(torch.int32)}
    if case["train"]:
        g = s["upstream"] * case["scale"] * kept
        if case["renormalize"]:
            g = g - (g * part).sum(1, keepdim=True)
            at = part * g if case["scoring"] == "softmax" else part * (1 - chosen) * g
            grad = torch.zeros_like(l).scatter_(1, ids, at)
        elif case["scoring"] == "softmax":
            grad = -score * (g * chosen).sum(1, keepdim=True)
            grad.scatter_add_(1, ids, chosen * g)
        else:
            grad = torch.zeros_like(l).scatter_(1, ids, chosen * (1 - chosen) * g)
        out["logits"] = grad.to(s["logits"].dtype)
    return out


def run(state):
    s = state
    case = s["case"]
    if not own:
        with torch.no_grad():
            return _plain_linear(s) if case["family"] == "linear" else _plain_route(s)
    dense, moe = _calls()
    leaves = [s[name] for name in s["leaves"]]
    if case["family"] == "linear":
        y = dense.dense_linear(
            s["x"], s["w"], s["bias"],
            activation=None if case["activation"] == "none" else case["activation"],
            residual=s["residual"], out_dtype=_DTYPES[case["out"]],
            clamp_limit=case["clamp"] or None)
        if not case["train"]:
            return y
        grads = torch.autograd.grad(y, leaves, s["upstream"])
        return {"y": y, **dict(zip(s["leaves"], grads))}
    weights, ids = moe.moe_route_logits(
        s["logits"], case["topk"], bias=s["bias"], num_groups=case["groups"],
        topk_groups=case["topk_groups"], renormalize=case["renormalize"],
        routed_scaling_factor=case["scale"], is_padding=s["is_padding"], scoring=case["scoring"])
    if not case["train"]:
        return {"weights": weights, "ids": ids}
    grad, = torch.autograd.grad(weights, leaves, s["upstream"])
    return {"weights": weights, "ids": ids, "logits": grad}


# ---- what a pass cannot do without -------------------------------------------------


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    a = size[case["dtype"]]
    if case["family"] == "linear":
        m, k, n, o = case["rows"], case["k"], case["n"], size[case["out"]]
        lines = 2 * n if case["activation"] == "swiglu" else n
        moved = m * k * a + lines * k * a + m * n * o
        moved += lines * a * case["bias"] + m * n * o * case["residual"]
        flops = 2 * m * k * lines
        if case["train"]:  # the upstream gradient in, the inputs' gradients out
            moved += m * n * o + m * k * a + lines * k * a
            moved += lines * a * case["bias"] + m * n * o * case["residual"]
            flops *= 3
        return {"bytes": moved, "flops": flops}
    t, e, slots = case["rows"], case["experts"], case["rows"] * case["topk"]
    moved = t * e * a + slots * 8 + t * bool(case["padded"]) + 4 * e * case["bias"]
    flops = 8 * t * e
    if case["train"]:
        moved += slots * 4 + t * e * a
        flops += 8 * slots
    return {"bytes": moved, "flops": flops}


# ---- 64 bits -------------------------------------------------------------------------


def _exact_linear(case, s):
    """By blocks of rows; the slopes from torch's own derivatives."""
    n, gated = case["n"], case["activation"] == "swiglu"
    w = s["w"].detach().double()
    b = 0 if s["bias"] is None else s["bias"].detach().double()[None]
    f = torch.nn.functional
    ys, dxs, dw, db = [], [], 0, 0
    step = max(1, (1 << 26) // w.shape[0])
    for r0 in range(0, case["rows"], step):
        x = s["x"].detach()[r0:r0 + step].double()
        with torch.enable_grad():
            z = (torch.matmul(x, w.t()) + b).requires_grad_(case["train"])
            if gated:
                g, u = z.split(n, 1)
                if case["clamp"]:
                    g, u = g.clamp(max=case["clamp"]), u.clamp(-case["clamp"], case["clamp"])
                y = f.silu(g) * u
            elif case["activation"] == "none":
                y = z * 1
            elif case["activation"] == "gelu_tanh":
                y = f.gelu(z, approximate="tanh")
            else:
                y = getattr(f, case["activation"])(z)
            if case["train"]:
                dz, = torch.autograd.grad(y, z, s["upstream"][r0:r0 + step].double())
                dxs.append(torch.matmul(dz, w))
                dw = dw + torch.matmul(dz.t(), x)
                db = db + dz.sum(0)
        y = y.detach()
        if s["residual"] is not None:
            y = y + s["residual"].detach()[r0:r0 + step].double()
        ys.append(y)
    y = torch.cat(ys)
    if not case["train"]:
        return y
    r = {"y": y, "x": torch.cat(dxs), "w": dw}
    if s["bias"] is not None:
        r["bias"] = db
    if s["residual"] is not None:
        r["residual"] = s["upstream"].double()
    return r


def _exact_route(case, s):
    l = s["logits"].detach().double()
    t, e, groups = case["rows"], case["experts"], case["groups"]
    score = torch.softmax(l, 1) if case["scoring"] == "softmax" else torch.special.expit(l)
    key = l if s["bias"] is None else score + s["bias"].double()
    rows = torch.arange(t, device=l.device)
    if groups > 1:
        left = key.clone()
        parts = left.view(t, groups, -1)
        rank = parts.amax(2)
        if s["bias"] is not None:
            again = parts.clone()
            again.scatter_(2, parts.argmax(2, keepdim=True), -math.inf)
            rank = rank + again.amax(2)
        open_group = torch.zeros_like(rank, dtype=torch.bool)
        for _ in range(case["topk_groups"]):
            best = (rank == rank.amax(1, keepdim=True)).int().argmax(1)  # the first of the largest
            open_group[rows, best] = True
            rank[rows, best] = -math.inf
        key = torch.where(open_group.repeat_interleave(e // groups, 1), key, -math.inf)
    else:
        key = key.clone()
    ids = torch.empty(t, case["topk"], dtype=torch.int64, device=l.device)
    for j in range(case["topk"]):
        best = (key == key.amax(1, keepdim=True)).int().argmax(1)
        ids[:, j] = best
        key[rows, best] = -math.inf

    def weigh(logits):
        if case["scoring"] == "softmax":
            p = torch.softmax(logits, 1).gather(1, ids)
        else:
            p = torch.special.expit(logits).gather(1, ids)
        return case["scale"] * (p / p.sum(1, keepdim=True) if case["renormalize"] else p)

    kept = torch.ones(t, dtype=torch.bool, device=l.device)
    if s["is_padding"] is not None:
        kept = ~s["is_padding"]
    with torch.enable_grad():
        leaf = l.clone().requires_grad_()
        weights = weigh(leaf) * kept[:, None]
        out = {"weights": weights.detach(),
               "ids": torch.where(kept[:, None], ids, -1).to(torch.int32)}
        if case["train"]:
            out["logits"], = torch.autograd.grad(weights, leaf, s["upstream"].double())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_linear(case, s) if case["family"] == "linear" else _exact_route(case, s)
