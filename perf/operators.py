"""The MXFP4 and router-balance operators as timed cases.

Four families, each one pass of a public entry point as a program calls it:

- ``quantize``: a tensor to MXFP4 (blocks of 32 along the last axis, E2M1
  codes under one E8M0 scale) and back, as a program that quantizes weights
  and looks at what they became does;
- ``linear``: activations times MXFP4 weights, the activations quantized on
  the way (``mxfp4_linear``);
- ``moe``: the routed experts with MXFP4 weights (``fused_mxfp4_moe``);
- ``balance``: a router's load-balance loss, its per-expert counts and its
  gradient (``moe_balance_loss``).

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
_BLOCK = 32


def _calls():
    """The framework's operators (imported only where they are called)."""
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    from vllm_mi355x.kernels import moe, mxfp4
    return mxfp4, moe


# ---- cases ---------------------------------------------------------------------


def _quantize(name, rows, k, dtype, *, gap=0):
    """gap: elements between the rows of a larger buffer that x is a part of."""
    return {"name": name, "family": "quantize", "rows": rows, "k": k, "dtype": dtype, "gap": gap}


def _linear(name, k, n, rows, dtype, *, out=None):
    return {"name": name, "family": "linear", "k": k, "n": n, "rows": rows, "dtype": dtype,
            "out": out or dtype}


def _moe(name, experts, hidden, inter, topk, rows, dtype, *, shared_by=1, clamp=0.0, zipf=0.0):
    """experts: those held here; shared_by: over how many such parts the layer's
    experts are spread (slots of the others' experts take no work here)."""
    return {"name": name, "family": "moe", "experts": experts, "hidden": hidden, "inter": inter,
            "topk": topk, "rows": rows, "dtype": dtype, "shared_by": shared_by, "clamp": clamp,
            "zipf": zipf}


def _balance(name, rows, experts, topk, dtype, *, scoring="softmax", padded=0.0):
    return {"name": name, "family": "balance", "rows": rows, "experts": experts, "topk": topk,
            "dtype": dtype, "scoring": scoring, "padded": padded}


def listed():
    return [
        # A decode step's activations, quantized before a product that is
        # called with codes: the smallest call.
        _quantize("quantize_decode_4", 4, 4096, "bf16"),
        # A weight matrix on its way into a quantized checkpoint, a column
        # slice of a fused matrix in 32 bits.
        _quantize("quantize_weight_fp32", 14336, 4096, "fp32", gap=1024),
        # One user's decode step through an up projection.
        _linear("linear_decode_1", 4096, 14336, 1, "bf16"),
        # A decode batch through a matrix whose sizes are no tile's multiple.
        _linear("linear_batch_20", 2592, 5003, 20, "fp16"),
        # A short prompt through a down projection, the sums kept in 32 bits
        # for what follows.
        _linear("linear_rows_400", 14336, 4096, 400, "bf16", out="fp32"),
        # A whole prefill chunk through the largest matrix.
        _linear("linear_prefill_2048", 8192, 28672, 2048, "bf16"),
        # One user's decode step through a fine-grained MoE layer.
        _moe("moe_decode_1", 128, 2048, 768, 8, 1, "bf16"),
        # A decode batch, the experts unevenly liked.
        _moe("moe_batch_64", 128, 2048, 768, 8, 64, "fp16", zipf=1.1),
        # A short prompt where a quarter of the layer's experts is held here,
        # sizes that end inside a tile, a clamped activation.
        _moe("moe_part_300", 16, 2592, 1184, 4, 300, "bf16", shared_by=4, clamp=7.0),
        # A prefill chunk of the fine-grained layer.
        _moe("moe_prefill_2048", 128, 2048, 768, 8, 2048, "bf16"),
        # A micro batch of a router's training step.
        _balance("balance_rows_200", 200, 128, 8, "fp32"),
        # A whole training batch, some of it padding, sigmoid scores.
        _balance("balance_rows_65536", 65536, 256, 8, "fp32", scoring="sigmoid", padded=0.1),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _log_blocks(rng, lo, hi):
    """A multiple of 32, log-uniform in [lo, hi]."""
    return _BLOCK * _log_int(rng, -(-lo // _BLOCK), hi // _BLOCK)


# What one drawn case may cost: the largest listed ones.
_MAX_ELEMENTS = 14336 * 4096
_MAX_LINEAR = 2048 * 8192 * 28672
_MAX_EXPERT_ELEMENTS = 128 * 3 * 2048 * 768
_MAX_MOE = 2048 * 8 * 3 * 2048 * 768
_MAX_LOGITS = 65536 * 256


def draw(rng):
    while True:
        family = rng.choice(["quantize", "linear", "linear", "moe", "moe", "balance"])
        dtype = rng.choice(["bf16", "fp16"])
        if family == "quantize":
            case = _quantize("", _log_int(rng, 1, 32768), _log_blocks(rng, 32, 16384),
                             rng.choice(["bf16", "fp16", "fp32"]), gap=rng.choice([0, 0, 8, 1024]))
            fits = case["rows"] * case["k"] <= _MAX_ELEMENTS
        elif family == "linear":
            case = _linear("", _log_blocks(rng, 256, 16384), _log_int(rng, 16, 28672),
                           _log_int(rng, 1, 4096), dtype, out=rng.choice([dtype, dtype, "fp32"]))
            fits = case["rows"] * case["k"] * case["n"] <= _MAX_LINEAR
        elif family == "moe":
            experts = _log_int(rng, 4, 256)
            case = _moe("", experts, _log_blocks(rng, 512, 7168), _log_blocks(rng, 128, 2048),
                        rng.randint(1, min(8, experts)), _log_int(rng, 1, 4096), dtype,
                        shared_by=rng.choice([1, 1, 2, 4]), clamp=rng.choice([0.0, 0.0, 7.0]),
                        zipf=rng.choice([0.0, 0.0, 1.1]))
            size = 3 * case["hidden"] * case["inter"]
            fits = (experts * size <= _MAX_EXPERT_ELEMENTS
                    and case["rows"] * case["topk"] * size <= _MAX_MOE)
        else:
            experts = _log_int(rng, 4, 512)
            case = _balance("", _log_int(rng, 1, 65536), experts, rng.randint(1, min(10, experts)),
                            rng.choice(["bf16", "fp16", "fp32"]),
                            scoring=rng.choice(["softmax", "sigmoid"]),
                            padded=rng.choice([0.0, 0.1, 0.5]))
            fits = case["rows"] * experts <= _MAX_LOGITS
        if fits:
            del case["name"]
            return case


# ---- inputs --------------------------------------------------------------------


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _packed_weights(g, *shape):
    """MXFP4 codes (two a byte, the even element in the low nibble) and scale
    bytes of normal weights at 0.02, rows of unlike size among them."""
    codes = torch.empty(*shape[:-1], shape[-1] // 2, dtype=torch.uint8, device="cuda")
    scales = torch.empty(*shape[:-1], shape[-1] // _BLOCK, dtype=torch.uint8, device="cuda")
    rows = math.prod(shape[:-1])
    flat, flat_s = codes.view(rows, -1), scales.view(rows, -1)
    step = max(1, (1 << 25) // shape[-1])
    for r0 in range(0, rows, step):
        r1 = min(rows, r0 + step)
        w = torch.randn(r1 - r0, shape[-1], device="cuda", generator=g)
        w *= 0.02 * torch.exp(0.5 * torch.randn(r1 - r0, 1, device="cuda", generator=g))
        code, e = _plain_codes(w)
        code = code.to(torch.uint8).reshape(r1 - r0, -1, 2)
        flat[r0:r1] = code[..., 0] | (code[..., 1] << 4)
        flat_s[r0:r1] = (e + 127).to(torch.uint8)
    return codes, scales


def _activations(g, rows, k, dtype):
    """Normal values with the few large channels that activations have."""
    x = torch.randn(rows, k, device="cuda", generator=g)
    x *= 1.0 + 7.0 * (torch.rand(k, device="cuda", generator=g) < 0.005)
    return x.to(_DTYPES[dtype])


def _routing(g, rows, experts, topk, zipf):
    """Top-k of normal logits (over a Zipf liking where asked), softmax weights
    renormalized over the chosen."""
    logits = torch.randn(rows, experts, device="cuda", generator=g)
    if zipf:
        order = torch.rand(experts, device="cuda", generator=g).argsort().float()
        logits -= zipf * torch.log(order + 1.0)
    top, ids = logits.topk(topk, dim=1)
    top = torch.exp(top - top[:, :1])
    return (top / top.sum(1, keepdim=True)).contiguous(), ids.to(torch.int32).contiguous()


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    if case["family"] == "quantize":
        x = _activations(g, case["rows"], case["k"] + case["gap"], case["dtype"])
        s["x"] = x[:, :case["k"]]
    elif case["family"] == "linear":
        s["x"] = _activations(g, case["rows"], case["k"], case["dtype"])
        s["w"], s["w_scale"] = _packed_weights(g, case["n"], case["k"])
    elif case["family"] == "moe":
        e, h, i = case["experts"], case["hidden"], case["inter"]
        s["x"] = _activations(g, case["rows"], h, case["dtype"])
        s["w1"], s["w1_scale"] = _packed_weights(g, e, 2 * i, h)
        s["w2"], s["w2_scale"] = _packed_weights(g, e, h, i)
        every = e * case["shared_by"]
        s["topk_weights"], s["topk_ids"] = _routing(g, case["rows"], every, case["topk"],
                                                    case["zipf"])
        s["expert_map"] = None
        if every > e:  # this part's experts, spread over the layer's
            held = torch.rand(every, device="cuda", generator=g).argsort()[:e].sort().values
            s["expert_map"] = torch.full((every,), -1, dtype=torch.int32, device="cuda")
            s["expert_map"][held] = torch.arange(e, dtype=torch.int32, device="cuda")
        s["workspace"] = {}
    else:
        t, e = case["rows"], case["experts"]
        # A router's logits: some experts liked by all rows
        logits = torch.randn(t, e, device="cuda", generator=g)
        logits += 0.5 * torch.randn(e, device="cuda", generator=g)
        logits = logits.to(_DTYPES[case["dtype"]])
        s["ids"] = logits.float().topk(case["topk"], dim=1).indices.to(torch.int32).contiguous()
        s["is_padding"] = None
        if case["padded"]:
            s["is_padding"] = torch.rand(t, device="cuda", generator=g) < case["padded"]
            s["ids"][s["is_padding"]] = -1
        s["logits"] = logits.requires_grad_()
        # the loss's coefficient times a loss scale, as the step's gradient is given
        s["upstream"] = torch.full((), float(t), device="cuda")
    return s


# ---- the plain forms, 32 bits ----------------------------------------------------


def _plain_codes(x):
    """(codes 0..15 of x's shape, scale exponents per block), x in 32 bits: the
    scale 2^e with e two below the exponent of the block's largest magnitude,
    the magnitudes rounded to 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to even codes)."""
    b = x.reshape(*x.shape[:-1], -1, _BLOCK)
    e = (torch.frexp(b.abs().amax(-1))[1] - 3).clamp(-126, 125)
    v = b * torch.exp2(-e.to(x.dtype))[..., None]
    a = v.abs()
    low, mid = torch.round(2 * a), torch.round(a) + 2
    code = torch.where(a < 2, low, torch.where(a < 4, mid, (torch.round(a / 2) + 4).clamp(max=7)))
    code = code + 8 * ((v < 0) & (code > 0))
    return code.reshape(x.shape), e


def _plain_values(x):
    """x as its MXFP4 codes stand for it, in 32 bits."""
    code, e = _plain_codes(x)
    v = _grid(x.device)[code.long()].reshape(*e.shape, _BLOCK)
    return (v * torch.exp2(e.to(torch.float32))[..., None]).reshape(x.shape)


def _grid(device, dtype=torch.float32):
    half = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=dtype, device=device)
    return torch.cat([half, -half])


def _unpacked(codes, scales, dtype=torch.float32):
    """The values of packed codes and scale bytes."""
    both = torch.stack([codes & 15, codes >> 4], -1)
    v = _grid(codes.device, dtype)[both.long()].reshape(*scales.shape, _BLOCK)
    v = v * torch.exp2(scales.to(dtype) - 127)[..., None]
    return v.reshape(*codes.shape[:-1], codes.shape[-1] * 2)


def _plain_moe(s):
    case, x = s["case"], _plain_values(s["x"].float())
    ids = s["topk_ids"].long()
    if s["expert_map"] is not None:
        ids = s["expert_map"].long()[ids]
    order = ids.reshape(-1).argsort(stable=True)
    counts = (ids.reshape(-1, 1) == torch.arange(case["experts"], device=x.device)).sum(0).tolist()
    at = ids.numel() - sum(counts)  # the slots of experts held elsewhere come first
    out = torch.zeros(x.shape, dtype=torch.float32, device=x.device)
    limit = case["clamp"] or math.inf
    for e, count in enumerate(counts):
        if not count:
            continue
        slots = order[at:at + count]
        at += count
        rows = slots // case["topk"]
        gu = x[rows] @ _unpacked(s["w1"][e], s["w1_scale"][e]).t()
        g, u = gu[:, :case["inter"]].clamp(max=limit), gu[:, case["inter"]:].clamp(-limit, limit)
        h = _plain_values(g / (1 + torch.exp(-g)) * u)
        y = h @ _unpacked(s["w2"][e], s["w2_scale"][e]).t()
        out.index_add_(0, rows, y * s["topk_weights"].reshape(-1)[slots, None])
    return out.to(s["x"].dtype)


def _plain_balance(s):
    case = s["case"]
    with torch.no_grad():
        l = s["logits"].float()
        e = case["experts"]
        counted = torch.ones_like(l[:, :1]) if s["is_padding"] is None else (~s["is_padding"])[:, None].float()
        rows = counted.sum().clamp(min=1)
        at = torch.where(s["ids"] < 0, e, s["ids"]).long().reshape(-1)
        counts = torch.zeros(e + 1, dtype=torch.int64, device=l.device).index_add_(
            0, at, torch.ones_like(at))[:e]
        f = counts.float() * e / (rows * case["topk"])
        if case["scoring"] == "softmax":
            z = torch.exp(l - l.amax(1, keepdim=True))
            p = z / z.sum(1, keepdim=True)
            slope = p
        else:
            z = 1 / (1 + torch.exp(-l))
            total = z.sum(1, keepdim=True)
            p = z / total
            slope = p * (1 - z)
        r = (p * f).sum(1, keepdim=True)
        loss = (r * counted).sum() / rows
        grad = slope * (f - r) * (counted / rows) * s["upstream"]
    return {"loss": loss, "counts": counts, "grad": grad.to(s["logits"].dtype)}


def run(state):
    s = state
    case = s["case"]
    family = case["family"]
    if family == "quantize":
        if own:
            mxfp4, _ = _calls()
            codes, scales = mxfp4.mxfp4_quantize(s["x"])
            return mxfp4.mxfp4_dequantize(codes, scales, s["x"].dtype)
        return _plain_values(s["x"].float()).to(s["x"].dtype)
    if family == "linear":
        if own:
            mxfp4, _ = _calls()
            return mxfp4.mxfp4_linear(s["x"], s["w"], s["w_scale"], out_dtype=_DTYPES[case["out"]])
        y = _plain_values(s["x"].float()) @ _unpacked(s["w"], s["w_scale"]).t()
        return y.to(_DTYPES[case["out"]])
    if family == "moe":
        if own:
            mxfp4, _ = _calls()
            return mxfp4.fused_mxfp4_moe(
                s["x"], s["w1"], s["w2"], s["w1_scale"], s["w2_scale"], s["topk_weights"],
                s["topk_ids"], clamp_limit=case["clamp"] or None, expert_map=s["expert_map"],
                workspace=s["workspace"])
        return _plain_moe(s)
    if own:
        _, moe = _calls()
        loss, counts = moe.moe_balance_loss(s["logits"], s["ids"], scoring=case["scoring"],
                                            is_padding=s["is_padding"])
        grad, = torch.autograd.grad(loss, s["logits"], s["upstream"])
        return {"loss": loss, "counts": counts, "grad": grad}
    return _plain_balance(s)


# ---- what a pass cannot do without -------------------------------------------------


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    packed = 0.5 + 1 / _BLOCK
    if case["family"] == "quantize":
        n = case["rows"] * case["k"]
        return {"bytes": 2 * n * size[case["dtype"]], "flops": 4 * n}
    if case["family"] == "linear":
        m, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": m * k * size[case["dtype"]] + n * k * packed + m * n * size[case["out"]],
                "flops": 2 * m * k * n}
    if case["family"] == "moe":
        e, h, i, t = case["experts"], case["hidden"], case["inter"], case["rows"]
        every = e * case["shared_by"]
        slots = t * case["topk"] / case["shared_by"]
        # experts that at least one slot chooses, as many as even liking gives
        touched = e * (1 - (1 - case["topk"] / every) ** t)
        return {"bytes": touched * 3 * h * i * packed + 2 * t * h * 2 + t * case["topk"] * 8,
                "flops": 6 * slots * h * i}
    t, e = case["rows"], case["experts"]
    return {"bytes": 2 * t * e * size[case["dtype"]] + t * case["topk"] * 4 + 8 * e,
            "flops": 12 * t * e}


# ---- 64 bits -------------------------------------------------------------------------


def _exact_values(x):
    """x (64 bits) as MXFP4 holds it, by comparing with the midpoints between
    the grid's values: a tie belongs to the side whose code is even."""
    b = x.reshape(*x.shape[:-1], -1, _BLOCK)
    top = b.abs().amax(-1, keepdim=True)
    scale = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -120))))
    scale = torch.where(scale > top, scale / 2, torch.where(scale * 2 <= top, scale * 2, scale)) / 4
    a = b.abs() / scale
    over = torch.zeros_like(a)
    for middle, step, even_above in ((0.25, 0.5, False), (0.75, 0.5, True), (1.25, 0.5, False),
                                     (1.75, 0.5, True), (2.5, 1.0, False), (3.5, 1.0, True),
                                     (5.0, 2.0, False)):
        over += step * ((a >= middle) if even_above else (a > middle))
    return (torch.sign(b) * over * scale).reshape(x.shape)


def _exact_weights(codes, scales):
    sign = torch.tensor([1.0, -1.0], dtype=torch.float64, device=codes.device)
    parts = []
    for nibble in (codes & 15, codes >> 4):
        exponent, mantissa = ((nibble >> 1) & 3).double(), (nibble & 1).double()
        size = torch.where(exponent == 0, mantissa / 2, (1 + mantissa / 2) * 2 ** (exponent - 1))
        parts.append(sign[(nibble >> 3).long()] * size)
    v = torch.stack(parts, -1).reshape(*codes.shape[:-1], -1)
    return v * (2.0 ** (scales.double() - 127)).repeat_interleave(_BLOCK, -1)


def exact(case, seed):
    s = prepare(case, seed)
    family = case["family"]
    if family == "quantize":
        return _exact_values(s["x"].double())
    if family == "linear":
        x = _exact_values(s["x"].double())
        out = torch.empty(case["rows"], case["n"], dtype=torch.float64, device=x.device)
        for n0 in range(0, case["n"], 4096):
            out[:, n0:n0 + 4096] = x @ _exact_weights(s["w"][n0:n0 + 4096],
                                                      s["w_scale"][n0:n0 + 4096]).t()
        return out
    if family == "moe":
        x = _exact_values(s["x"].double())
        out = torch.zeros_like(x)
        for e in range(case["experts"]):
            own_id = e if s["expert_map"] is None else int((s["expert_map"] == e).nonzero())
            rows, slots = (s["topk_ids"] == own_id).nonzero(as_tuple=True)
            if not len(rows):
                continue
            w1 = _exact_weights(s["w1"][e], s["w1_scale"][e])
            g = x[rows] @ w1[:case["inter"]].t()
            u = x[rows] @ w1[case["inter"]:].t()
            if case["clamp"]:
                g = torch.minimum(g, torch.full_like(g, case["clamp"]))
                u = torch.maximum(torch.minimum(u, torch.full_like(u, case["clamp"])),
                                  torch.full_like(u, -case["clamp"]))
            h = _exact_values(g * torch.special.expit(g) * u)
            y = h @ _exact_weights(s["w2"][e], s["w2_scale"][e]).t()
            # a row holds an expert once at most: no index repeats
            out[rows] += y * s["topk_weights"][rows, slots].double()[:, None]
        return out
    with torch.no_grad():
        l = s["logits"].double()
        kept = torch.ones(case["rows"], dtype=torch.bool, device=l.device)
        if s["is_padding"] is not None:
            kept = ~s["is_padding"]
        n, e = int(kept.sum()), case["experts"]
        counts = torch.bincount(s["ids"][kept].reshape(-1).long(), minlength=e)
        grad = torch.zeros_like(l)
        if not n:
            return {"loss": l.sum() * 0, "counts": counts, "grad": grad}
        f = counts.double() * e / (n * case["topk"])
        a = l[kept]
        if case["scoring"] == "softmax":
            p = torch.special.softmax(a, 1)
            d = p
        else:
            q = torch.special.expit(a)
            p = q / q.sum(1, keepdim=True)
            d = p * torch.special.expit(-a)
        share = p @ f
        grad[kept] = d * (f[None, :] - share[:, None]) / n * float(s["upstream"])
        return {"loss": share.mean(), "counts": counts, "grad": grad}
