"""Routing from logits on the GPU against the FP64 oracle.

Ids are exact: keys that lie within FP32's errors are compared in 64 bits.

Tolerances: a sigmoid is off by 2^-21 of it (exponential 2^-22, a sum and a reciprocal), an
exponential of a difference by 2^-22 and by the difference's own rounding, 2^-25 of
it; sums of up to 1024 positive terms by 22 roundings of 2^-24; a quotient adds its
sides': 2^-19 of a weight, and 2^-24 of the largest difference in the row.  A gradient is w (g -
sum w g / c): 2^-18 of the magnitudes and the weights' errors, then half a step of its
type.  (A few terms of 2^-120 for what lies below FP32's normal numbers.)
"""

import numpy as np
import pytest
import torch

from oracle import route_logits_oracle as L

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def moe():
    from vllm_mi355x.kernels import moe as module
    return module


def on(device, a):
    return None if a is None else torch.from_numpy(np.ascontiguousarray(a)).to(device)


def check(moe, logits, topk, sigmoid, bias=None, groups=1, topk_groups=1, renormalize=True, scale=1.0, padding=None, up=None):
    """One call with its gradient; returns (weights, ids, gradient)."""
    device = logits.device
    l = logits.detach().double().cpu().numpy()
    ids, w = L.route(l, topk, sigmoid, bias, groups, topk_groups, renormalize, scale, padding)
    leaf = logits.detach().requires_grad_()
    gw, gi = moe.moe_route_logits(leaf, topk, on(device, bias), groups, topk_groups, renormalize, scale, on(device, padding),
                                  "sigmoid" if sigmoid else "softmax")
    assert gw.shape == gi.shape == (len(l), topk) and gw.dtype == torch.float32 and gi.dtype == torch.int32
    assert not gi.requires_grad
    assert np.array_equal(gi.cpu().numpy(), ids), np.flatnonzero((gi.cpu().numpy() != ids).any(1))[:9]
    got = gw.detach().double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        finite = np.where(np.isfinite(l), l, np.nan)
        spread = np.nan_to_num(np.nanmax(finite, 1, initial=-1e30) - np.nanmin(finite, 1, initial=1e30)) if l.shape[1] else 0
    spread = np.minimum(np.maximum(spread, 0), 1500)
    rel = 2.0 ** -19 + 2.0 ** -24 * spread[:, None]
    poisoned = np.isnan(w)
    assert np.array_equal(np.isnan(got), poisoned)
    assert (np.abs(got - w)[~poisoned] <= (rel * np.abs(w) + abs(scale) * 2.0 ** -120)[~poisoned]).all()
    if up is None:
        up = np.random.default_rng(len(l)).standard_normal((len(l), topk)).astype(np.float32)
    grad, = torch.autograd.grad(gw, leaf, on(device, up))
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    gg = grad.double().cpu().numpy()
    info = torch.finfo(logits.dtype)
    for t in range(len(l)):
        if poisoned[t].any():
            assert np.isnan(gg[t][ids[t][ids[t] >= 0]]).all()
            continue
        want = L.gradient(l[t], ids[t], w[t], up[t].astype(np.float64), sigmoid, renormalize, scale)
        held = ids[t] >= 0
        size = np.zeros(l.shape[1])
        mean = np.abs(w[t] * up[t]).sum()
        if held.any() and scale:
            s, _, _ = L.scores(l[t], sigmoid)
            if not sigmoid and not renormalize:
                size = s * mean
                size[ids[t][held]] += np.abs(w[t] * up[t])[held]
            else:
                size[ids[t][held]] = np.abs(w[t][held]) * (np.abs(up[t][held]) + (mean / abs(scale) if renormalize else 0))
                if sigmoid:
                    size[ids[t][held]] *= L.complements(l[t])[ids[t][held]]
        tol = size * (2.0 ** -18 + 2.0 ** -23 * spread[t]) + 2.0 ** -120
        tol = tol + info.eps / 2 * (np.abs(want) + tol) + info.smallest_normal * info.eps
        assert (np.abs(gg[t] - want) <= tol).all(), f"row {t}: {(np.abs(gg[t] - want) - tol).max():.3g}"
    return gw, gi, grad


SIZES = [(1, 1, 1, 1, 1), (1, 256, 8, 8, 4), (3, 5, 4, 1, 1), (64, 64, 6, 8, 3), (200, 128, 8, 4, 2), (7, 65, 3, 5, 2), (70, 160, 6, 8, 3),
         (300, 257, 8, 1, 1), (33, 512, 10, 16, 4), (5, 1000, 8, 40, 7), (2, 1024, 1, 64, 1), (500, 40, 2, 2, 1), (60, 256, 20, 4, 3),
         (31, 64, 64, 1, 1), (17, 1024, 64, 32, 3), (40, 96, 5, 3, 2), (11, 256, 8, 32, 5), (9, 48, 4, 12, 5), (1030, 256, 8, 8, 4)]


@pytest.mark.parametrize("rows,experts,topk,groups,topk_groups", SIZES)
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_matches_the_oracle(moe, device, rows, experts, topk, groups, topk_groups, dtype, scoring):
    print(f"route {rows}x{experts} k={topk} groups={groups}/{topk_groups} {dtype} {scoring}", flush=True)
    rng = np.random.default_rng(rows * 7 + experts)
    logits = torch.from_numpy(rng.standard_normal((rows, experts)) * 2).to(TYPES[dtype]).to(device)
    bias = (rng.standard_normal(experts) * 0.1).astype(np.float32)
    padding = rng.random(rows) < 0.2
    check(moe, logits, topk, scoring == "sigmoid", bias, groups, topk_groups, True, 2.5, padding)
    check(moe, logits, topk, scoring == "sigmoid", None, groups, topk_groups, False, -0.5)
    check(moe, logits, topk, scoring == "sigmoid", None, 1, 1, True, 1.0, padding)
    check(moe, logits, topk, scoring == "sigmoid", bias, 1, 1, False, 1.0)


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("sigmoid", [False, True])
def test_masks(moe, device, dtype, sigmoid):
    """Experts masked with -inf or the type's lowest value, rows where all are, far
    logits, NaN and infinities, in padding rows too."""
    rng = np.random.default_rng(6)
    logits = torch.from_numpy(rng.standard_normal((16, 24))).to(TYPES[dtype]).to(device)
    low, inf = torch.finfo(logits.dtype).min, float("inf")
    logits[0] = -inf
    logits[1] = low
    logits[2, ::2] = -inf
    logits[3, 2:] = low
    logits[4] = 60.0
    logits[5] = -60.0
    logits[6] = torch.linspace(-700, -720, 24, device=device)
    logits[7] = -inf
    logits[7, 5] = -300.0
    logits[8, 3] = inf
    logits[9, 4] = float("nan")
    logits[10, 3] = -inf
    logits[11] = 0.0
    logits[12] = torch.linspace(0, -1400, 24, device=device)
    logits[13] = float("nan")
    bias = (rng.standard_normal(24) * 0.1).astype(np.float32)
    bias[2], bias[7], bias[9] = -np.inf, np.nan, np.inf
    padding = np.zeros(16, bool)
    padding[14:] = True
    logits[14] = float("nan")
    for b in (None, bias, np.zeros(24, np.float32)):
        for groups, open_groups in ((1, 1), (6, 2), (4, 3)):
            for renormalize in (False, True):
                check(moe, logits, 5, sigmoid, b, groups, open_groups, renormalize, 1.5, padding)
    w, ids, grad = check(moe, logits, 5, sigmoid, bias, padding=np.ones(16, bool))
    assert not w.any() and (ids == -1).all() and not grad.any()


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("groups,topk_groups", [(1, 1), (8, 4), (5, 2), (16, 3)])
def test_keys_closer_than_fp32(moe, device, sigmoid, groups, topk_groups):
    """Biases that make every key nearly equal (2^-25 apart): only 64 bits tell them,
    and equal ones go to the lower expert."""
    rng = np.random.default_rng(groups)
    experts = 80
    for dtype in ("fp32", "bf16"):
        logits = torch.from_numpy(rng.standard_normal((40, experts))).to(TYPES[dtype]).to(device)
        l = logits.double().cpu().numpy()
        for t in (0, 17):
            s, _, _ = L.scores(l[t], sigmoid)
            bias = (0.7 - s).astype(np.float32)
            check(moe, logits[t:t + 1], 8, sigmoid, bias, groups, topk_groups)
            check(moe, logits, 8, sigmoid, bias, groups, topk_groups)
        same = torch.full((6, experts), 0.3, device=device, dtype=TYPES[dtype])
        _, ids, _ = check(moe, same, 4, sigmoid, np.zeros(experts, np.float32), groups, topk_groups)
        assert (ids == torch.arange(4, device=device)).all()


def test_large_biases(moe, device):
    """Biases far larger than scores, of both signs, some cancelling in a group."""
    rng = np.random.default_rng(9)
    logits = torch.from_numpy(rng.standard_normal((30, 64))).float().to(device)
    bias = (rng.standard_normal(64) * 10.0 ** rng.integers(-3, 7, 64)).astype(np.float32)
    bias[8:16] = [1e6, -1e6, 1e6, -1e6, 1e6, 1e6, 2e6, -2e6]
    for groups, open_groups in ((1, 1), (8, 3), (4, 2)):
        check(moe, logits, 8, True, bias, groups, open_groups)
        check(moe, logits, 8, False, bias, groups, open_groups, False)


def test_strides_types_and_nothing(moe, device):
    rng = np.random.default_rng(3)
    for dtype in TYPES:
        wide = torch.from_numpy(rng.standard_normal((40, 100))).to(TYPES[dtype]).to(device)
        for view in (wide[:, 5:65], wide[::2, :61], wide[:1, 3:64], wide[:, 4:5], wide.t()[:1].t()):
            check(moe, view, min(4, view.shape[1]), False, scale=0.5)
        w, ids, grad = check(moe, wide[:0], 3, True)
        assert w.shape == (0, 3) and grad.shape == (0, 100)
    w, ids = moe.moe_route_logits(wide, 4)
    assert not w.requires_grad
    leaf = wide.clone().requires_grad_()
    with torch.no_grad():
        assert not moe.moe_route_logits(leaf, 4)[0].requires_grad
    # upstream gradients as autograd gives them: broadcast ones, transposed ones
    w, _ = moe.moe_route_logits(leaf, 4, renormalize=False)
    a, = torch.autograd.grad(w.sum(), leaf, retain_graph=True)
    b, = torch.autograd.grad(w, leaf, torch.ones_like(w), retain_graph=True)
    assert torch.equal(a, b)
    up = torch.randn(4, 40, device=device)
    a, = torch.autograd.grad(w, leaf, up.t(), retain_graph=True)
    b, = torch.autograd.grad(w, leaf, up.t().contiguous(), retain_graph=True)
    assert torch.equal(a, b)
    check(moe, wide, 4, True, scale=0.0)


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gradient_by_differences(moe, device, scoring, renormalize):
    """Against central differences of the 64-bit weights of the same choice."""
    rng = np.random.default_rng(8)
    l = rng.standard_normal((4, 12)).astype(np.float32)
    leaf = on(device, l).requires_grad_()
    w, ids = moe.moe_route_logits(leaf, 3, None, 4, 2, renormalize, 2.5, scoring=scoring)
    up = rng.standard_normal((4, 3)).astype(np.float32)
    grad, = torch.autograd.grad(w, leaf, on(device, up))
    ids, sigmoid = ids.cpu().numpy(), scoring == "sigmoid"
    for t in range(4):
        for e in range(12):
            d = np.zeros(12)
            d[e] = 1e-5
            row = l[t].astype(np.float64)
            diff = (up[t] * (L.weigh(row + d, ids[t], sigmoid, renormalize, 2.5) - L.weigh(row - d, ids[t], sigmoid, renormalize, 2.5))).sum() / 2e-5
            # 1e-8: the differences' own error; the rest FP32
            assert abs(grad[t, e].item() - diff) <= 1e-8 + 2.0 ** -18 * 2.5 * np.abs(up[t]).sum()


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_one_slot_has_no_gradient(moe, device, scoring):
    """A single renormalized weight is the scale whatever the logits: its gradient is 0, not a
    rounding; rows with one expert left likewise."""
    g = torch.Generator(device=device).manual_seed(2)
    logits = torch.randn(300, 40, device=device, generator=g)
    up = torch.randn(300, 1, device=device, generator=g)
    leaf = logits.clone().requires_grad_()
    w, _ = moe.moe_route_logits(leaf, 1, routed_scaling_factor=2.3, scoring=scoring)
    grad, = torch.autograd.grad(w, leaf, up)
    assert (w == torch.tensor(2.3, device=device)).all() and not grad.any()
    logits[:, 3:] = -float("inf")
    logits[:, :2] = -float("inf")
    leaf = logits.requires_grad_()
    w, ids = moe.moe_route_logits(leaf, 4, routed_scaling_factor=2.3, scoring=scoring)
    assert (ids == torch.tensor([2, -1, -1, -1], device=device)).all()
    grad, = torch.autograd.grad(w, leaf, torch.randn(300, 4, device=device, generator=g))
    assert not grad.any()


def test_deterministic_and_backward_twice(moe, device):
    rng = np.random.default_rng(4)
    logits = torch.from_numpy(rng.standard_normal((3000, 128))).float().to(device).requires_grad_()
    bias = torch.zeros(128, device=device)
    w, ids = moe.moe_route_logits(logits, 8, bias, 8, 4)
    up = torch.randn(3000, 8, device=device)
    g1, = torch.autograd.grad(w, logits, up, retain_graph=True)
    g2, = torch.autograd.grad(w, logits, up, retain_graph=True)
    assert torch.equal(g1, g2)
    for _ in range(3):
        again, same = moe.moe_route_logits(logits, 8, bias, 8, 4)
        assert torch.equal(again, w) and torch.equal(ids, same)
    # a row's result is that row's alone
    part, pids = moe.moe_route_logits(logits[1000:1003], 8, bias, 8, 4)
    assert torch.equal(part, w[1000:1003]) and torch.equal(pids, ids[1000:1003])
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(w, logits, up, create_graph=True)
    with torch.no_grad():
        w.mul_(2)
    with pytest.raises(RuntimeError):  # autograd's own: the saved weights have changed
        torch.autograd.grad(w, logits, up)


def test_refusals(moe, device):
    l = torch.zeros(6, 8, device=device)
    pad = torch.zeros(6, dtype=torch.bool, device=device)
    bias = torch.zeros(8, device=device)
    r = moe.moe_route_logits
    for call in (lambda: r(l.double(), 2), lambda: r(l.cpu(), 2), lambda: r(l.t(), 2), lambda: r(l[0], 2), lambda: r(l, 0), lambda: r(l, 9),
                 lambda: r(torch.zeros(2, 100, device=device), 65), lambda: r(torch.zeros(2, 1025, device=device), 2),
                 lambda: r(l[:1].expand(6, 8), 2), lambda: r(l, 2, bias.half()), lambda: r(l, 2, bias[:7]), lambda: r(l, 2, bias.cpu()),
                 lambda: r(l, 2, bias[None]), lambda: r(l, 2, num_groups=3), lambda: r(l, 2, num_groups=0), lambda: r(l, 2, num_groups=4, topk_groups=5),
                 lambda: r(l, 2, num_groups=4, topk_groups=0), lambda: r(l, 3, num_groups=4, topk_groups=1), lambda: r(l, 2, is_padding=pad[:5]),
                 lambda: r(l, 2, is_padding=pad.float()), lambda: r(l, 2, is_padding=pad.cpu()), lambda: r(l, 2, routed_scaling_factor=float("inf")),
                 lambda: r(torch.zeros(2, 130, device=device), 2, num_groups=65, topk_groups=3), lambda: r(l[:, :0], 1)):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail("taken")
    with pytest.raises(ValueError):
        r(l, 2, scoring="tanh")


@pytest.mark.parametrize("rows", [1, 100, 6000])
def test_graph_and_streams(moe, device, rows):
    """Forward and backward captured, replayed with new inputs between eager work, and
    eager calls on two streams at once: equal bits."""
    rng = np.random.default_rng(rows)
    sets = [(torch.from_numpy(rng.standard_normal((rows, 96))).float().to(device), on(device, (rng.standard_normal(96) * .1).astype(np.float32)),
             on(device, rng.random(rows) < 0.2), torch.randn(rows, 4, device=device)) for _ in range(3)]

    def step(logits, bias, pad, up):
        leaf = logits.detach().requires_grad_()
        w, ids = moe.moe_route_logits(leaf, 4, bias, 8, 3, is_padding=pad)
        grad, = torch.autograd.grad(w, leaf, up)
        return w.detach(), ids, grad

    want = [step(*s) for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step(*sets[0])
    second = step(*sets[1])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    for got, w in ((first, want[0]), (second, want[1])):
        assert all(torch.equal(a, b) for a, b in zip(got, w))
    static = tuple(t.clone() for t in sets[0])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = step(*static)
    for i in (1, 2, 0, 1):
        for dst, src in zip(static, sets[i]):
            dst.copy_(src)
        graph.replay()
        again = step(*sets[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
        assert all(torch.equal(a, b) for a, b in zip(again, want[i]))


def test_offsets_past_32_bits(moe, device):
    """Rows 2^30 elements apart, and as many rows as make a gradient of over 2^32 elements."""
    g = torch.Generator(device=device).manual_seed(1)
    few = torch.randn(5, 64, device=device, generator=g).bfloat16()
    far = torch.empty(5, 1 << 30, dtype=torch.bfloat16, device=device)
    far[:, 8:72] = few
    w, ids = moe.moe_route_logits(far[:, 8:72], 6)
    want = moe.moe_route_logits(few, 6)
    assert torch.equal(w, want[0]) and torch.equal(ids, want[1])
    del far
    rows = (1 << 22) + 5
    many = torch.zeros(rows, 1024, dtype=torch.bfloat16, device=device)
    many[-5:, 100:164] = few
    leaf = many.requires_grad_()
    w, ids = moe.moe_route_logits(leaf, 6, scoring="softmax", renormalize=False)
    small = many[-5:].detach().requires_grad_()
    sw, sids = moe.moe_route_logits(small, 6, scoring="softmax", renormalize=False)
    up = torch.ones(rows, 6, device=device)
    up[-5:] = torch.randn(5, 6, device=device, generator=g)
    grad, = torch.autograd.grad(w, leaf, up)
    sgrad, = torch.autograd.grad(sw, small, up[-5:])
    assert torch.equal(w[-5:], sw) and torch.equal(ids[-5:], sids) and torch.equal(grad[-5:], sgrad)
    assert (ids[:-5] == torch.arange(6, device=device)).all()
