"""The router's load on the GPU against the FP64 oracle and central differences.

Tolerances: expf is good to 2 FP32 ulps, a row's sums of E positive terms to
(E / 64 + 8) roundings of 2^-24, the quotient and products to a few more: 2^-18
of a row's magnitudes for up to 1024 experts.  A gradient is p (f - r) g / n, so
its bound is that of p (|f| + |r|) g / n, then half a step of its type.
"""

import numpy as np
import pytest
import torch

from oracle import balance_oracle as B

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def moe():
    from vllm_mi355x.kernels import moe as module
    return module


def make(rng, rows, experts, topk, dtype, device, pad=0.2):
    logits = torch.from_numpy(rng.standard_normal((rows, experts)) * 3).to(TYPES[dtype]).to(device)
    ids = rng.integers(-1, experts + 1, (rows, topk)).astype(np.int32)
    padding = rng.random(rows) < pad
    return logits, ids, padding


def check(moe, logits, ids, padding, sigmoid, device, upstream=1.0):
    l = logits.detach().double().cpu().numpy()
    want, wc, wg = B.loss_and_grad(l, ids, sigmoid, padding)
    leaf = logits.detach().requires_grad_()
    loss, counts = moe.moe_balance_loss(leaf, torch.from_numpy(ids).to(device), "sigmoid" if sigmoid else "softmax",
                                        None if padding is None else torch.from_numpy(padding).to(device))
    assert loss.dtype == torch.float32 and loss.shape == () and counts.dtype == torch.int64
    assert np.array_equal(counts.cpu().numpy(), wc)
    assert abs(loss.item() - want) <= 2.0 ** -18 * abs(want) + 1e-30
    grad, = torch.autograd.grad(loss * upstream, leaf)
    assert grad.dtype == logits.dtype and grad.shape == logits.shape
    n = len(l) if padding is None else int((~padding).sum())
    tol = np.zeros_like(l)
    if n:
        f = wc * (l.shape[1] / (n * ids.shape[1]))
        kept = np.ones(len(l), bool) if padding is None else ~padding
        p, d = B.probabilities(l[kept], sigmoid)
        tol[kept] = 2.0 ** -18 * d * (np.abs(f) + np.abs(p @ f)[:, None]) / n * abs(upstream)
    info = torch.finfo(logits.dtype)
    tol = tol + info.eps / 2 * (np.abs(wg * upstream) + tol) + info.smallest_normal * info.eps
    off = np.abs(grad.double().cpu().numpy() - wg * upstream) - tol
    assert (off <= 0).all(), f"max excess {off.max():.3g}"
    return loss, grad


@pytest.mark.parametrize("rows,experts,topk", [(1, 1, 1), (1, 8, 2), (3, 5, 4), (64, 64, 6), (200, 128, 8), (7, 65, 3),
                                               (300, 257, 8), (33, 512, 10), (5, 1000, 8), (2, 1024, 1), (5000, 40, 2), (2500, 256, 8),
                                               (9000, 16, 4), (256, 128, 8), (257, 128, 8)])
@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("sigmoid", [False, True])
def test_matches_the_oracle(moe, device, rows, experts, topk, dtype, sigmoid):
    print(f"balance {rows}x{experts} k={topk} {dtype} sigmoid={sigmoid}", flush=True)
    rng = np.random.default_rng(rows + experts)
    logits, ids, padding = make(rng, rows, experts, topk, dtype, device)
    check(moe, logits, ids, padding, sigmoid, device, upstream=rows * 0.5)
    check(moe, logits, ids, None, sigmoid, device, upstream=-2.0)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_masked_logits(moe, device, dtype, sigmoid):
    """Experts masked with -inf or the type's lowest value, rows where all are,
    far positive and negative logits, and every row padding."""
    rng = np.random.default_rng(6)
    logits, ids, padding = make(rng, 12, 20, 3, dtype, device)
    low = torch.finfo(logits.dtype).min
    logits[0] = -float("inf")
    logits[1] = low
    logits[2, ::2] = -float("inf")
    logits[3, 1:] = low
    logits[4] = 60.0
    logits[5] = -60.0
    logits[6, 0] = -float("inf")
    padding[:7] = False
    check(moe, logits, ids, padding, sigmoid, device)
    loss, grad = check(moe, logits, ids, np.ones(12, bool), sigmoid, device)
    assert loss.item() == 0 and not grad.any()
    padded = logits.clone()
    padded[padding.nonzero()[0]] = float("nan")  # what padding rows hold is not read into anything
    check(moe, torch.where(torch.from_numpy(padding).to(device)[:, None], torch.zeros_like(logits), padded), ids, padding, sigmoid, device)
    a = moe.moe_balance_loss(padded, torch.from_numpy(ids).to(device), "sigmoid" if sigmoid else "softmax",
                             torch.from_numpy(padding).to(device))[0]
    assert torch.isfinite(a)
    bad = logits.clone()
    bad[5, 3] = float("nan")
    leaf = bad.requires_grad_()
    a = moe.moe_balance_loss(leaf, torch.from_numpy(ids).to(device), "sigmoid" if sigmoid else "softmax")[0]
    grad, = torch.autograd.grad(a, leaf)
    assert torch.isnan(a) and torch.isnan(grad[5]).any() and torch.isfinite(grad[[1, 2, 3, 4, 7, 8]]).all()


def test_gradient_by_differences(moe, device):
    rng = np.random.default_rng(8)
    logits, ids, _ = make(rng, 6, 10, 2, "fp32", device)
    for sigmoid in (False, True):
        leaf = logits.clone().requires_grad_()
        loss, _ = moe.moe_balance_loss(leaf, torch.from_numpy(ids).to(device), "sigmoid" if sigmoid else "softmax")
        grad, = torch.autograd.grad(loss, leaf)
        l = logits.double().cpu().numpy()
        for t, e in ((0, 0), (3, 7), (5, 9), (2, 4)):
            up, down = l.copy(), l.copy()
            up[t, e] += 1e-5
            down[t, e] -= 1e-5
            d = (B.loss_and_grad(up, ids, sigmoid)[0] - B.loss_and_grad(down, ids, sigmoid)[0]) / 2e-5
            # 1e-8: the differences' own error; the rest FP32
            assert abs(grad[t, e].item() - d) <= 1e-8 + 2.0 ** -18 * (abs(d) + np.abs(grad.cpu().numpy()).max())


def test_strides_types_and_nothing(moe, device):
    rng = np.random.default_rng(3)
    for dtype in TYPES:
        wide, ids, padding = make(rng, 40, 100, 2, dtype, device)
        ids = np.clip(ids, -1, 60)
        for view in (wide[:, 5:65], wide[::2, :61][:20], wide[:1, 3:64]):
            rows = view.shape[0]
            check(moe, view, ids[:rows], padding[:rows], False, device)
    t = torch.from_numpy(ids).to(device)
    a = moe.moe_balance_loss(wide, t.long())[0]
    assert torch.equal(a, moe.moe_balance_loss(wide, t)[0]) and not a.requires_grad
    leaf = wide[:0].detach().requires_grad_()
    loss, counts = moe.moe_balance_loss(leaf, t[:0])
    grad, = torch.autograd.grad(loss, leaf)
    assert loss.item() == 0 and not counts.any() and grad.shape == (0, 100)


def test_deterministic_and_backward_twice(moe, device):
    rng = np.random.default_rng(4)
    logits, ids, padding = make(rng, 3000, 128, 8, "fp32", device)
    t, p = torch.from_numpy(ids).to(device), torch.from_numpy(padding).to(device)
    leaf = logits.requires_grad_()
    loss, _ = moe.moe_balance_loss(leaf, t, is_padding=p)
    g1, = torch.autograd.grad(loss, leaf, retain_graph=True)
    g2, = torch.autograd.grad(loss, leaf, retain_graph=True)
    assert torch.equal(g1, g2)
    g3, = torch.autograd.grad(loss, leaf, torch.full((), 2.0, device=device), retain_graph=True)
    assert torch.equal(g3, 2 * g1)
    for _ in range(3):
        again, _ = moe.moe_balance_loss(leaf, t, is_padding=p)
        assert torch.equal(again, loss)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(loss, leaf, create_graph=True)


def test_expert_counts(moe, device):
    rng = np.random.default_rng(5)
    for rows, experts, topk in ((1, 1, 1), (0, 4, 2), (7, 300, 9), (40000, 64, 8), (1000, 1024, 3)):
        ids = rng.integers(-2, experts + 2, (rows, topk)).astype(np.int32)
        pad = rng.random(rows) < 0.3
        t, p = torch.from_numpy(ids).to(device), torch.from_numpy(pad).to(device)
        want = B.counts(ids, experts, pad)
        got = moe.moe_expert_counts(t, experts, p)
        assert np.array_equal(got.cpu().numpy(), want)
        total = torch.full((experts,), 5_000_000_000, dtype=torch.int64, device=device)
        assert moe.moe_expert_counts(t, experts, p, out=total) is total
        moe.moe_expert_counts(t, experts, out=total)
        assert np.array_equal(total.cpu().numpy(), 5_000_000_000 + want + B.counts(ids, experts))
    same = torch.full((5000, 4), 3, dtype=torch.int32, device=device)
    assert moe.moe_expert_counts(same, 8).tolist() == [0, 0, 0, 20000, 0, 0, 0, 0]


def test_refusals(moe, device):
    l = torch.zeros(6, 8, device=device)
    ids = torch.zeros(6, 2, dtype=torch.int32, device=device)
    pad = torch.zeros(6, dtype=torch.bool, device=device)
    for call in (lambda: moe.moe_balance_loss(l.double(), ids), lambda: moe.moe_balance_loss(l, ids[:5]),
                 lambda: moe.moe_balance_loss(l, ids[:, :0]), lambda: moe.moe_balance_loss(l.t(), ids),
                 lambda: moe.moe_balance_loss(l[:1].expand(6, 8), ids), lambda: moe.moe_balance_loss(l, ids, is_padding=pad[:5]),
                 lambda: moe.moe_balance_loss(l, ids, is_padding=pad.float()), lambda: moe.moe_balance_loss(l, ids.cpu()),
                 lambda: moe.moe_balance_loss(torch.zeros(2, 1025, device=device), ids[:2]),
                 lambda: moe.moe_balance_loss(l[0], ids), lambda: moe.moe_expert_counts(ids, 0), lambda: moe.moe_expert_counts(ids[0], 4),
                 lambda: moe.moe_expert_counts(ids, 4, out=torch.zeros(5, dtype=torch.int64, device=device)),
                 lambda: moe.moe_expert_counts(ids, 4, out=torch.zeros(4, dtype=torch.int32, device=device)),
                 lambda: moe.moe_expert_counts(ids, 4, pad.cpu())):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail("taken")


@pytest.mark.parametrize("rows", [100, 6000])
def test_graph_and_streams(moe, device, rows):
    """Forward and backward captured, replayed with new inputs between eager
    work, and eager calls on two streams at once: equal bits."""
    print(f"balance graph {rows}", flush=True)
    rng = np.random.default_rng(rows)
    sets = []
    for _ in range(3):
        logits, ids, padding = make(rng, rows, 96, 4, "fp32", device)
        sets.append((logits, torch.from_numpy(ids).to(device), torch.from_numpy(padding).to(device)))

    def step(logits, ids, pad):
        leaf = logits.detach().requires_grad_()
        loss, counts = moe.moe_balance_loss(leaf, ids, "sigmoid", pad)
        grad, = torch.autograd.grad(loss, leaf)
        return loss.detach(), counts, grad

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
