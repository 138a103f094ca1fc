"""The dense layer's gradients where the sizes and values of test_gpu_dense.py do not reach.
Tolerances as there."""

import numpy as np
import pytest
import torch

from oracle import dense_oracle as D
from tests.test_gpu_dense import TYPES, close, exact, linear, normal  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [1, 5, 40, 300])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_relu_passes_gradients_where_it_keeps_nan(linear, device, rows, dtype):
    """relu(NaN) is NaN, and dy passes there as it passes torch's relu: dz = dy in the row with a NaN,
    which the type of x holds in full, and the other rows are as they are without it."""
    rng = np.random.default_rng(rows)
    x, w = normal(rng, (rows, 64), dtype, device), normal(rng, (48, 64), dtype, device, 0.1)
    bias = normal(rng, 48, "fp32", device)
    dy = normal(rng, (rows, 48), dtype, device)
    at = rows // 2
    keep = torch.arange(rows, device=device) != at
    bad = x.clone()
    bad[at, 3] = float("nan")
    got = []
    for a in (x, bad):
        leaves = [t.detach().requires_grad_() for t in (a, w, bias)]
        got.append(torch.autograd.grad(linear(*leaves, "relu"), leaves, dy))
    dx, dw, db = got[1]
    assert torch.equal(dx[keep], got[0][0][keep])
    z = torch.from_numpy(exact(bad) @ exact(w).T + exact(bias)).requires_grad_()
    dz, = torch.autograd.grad(torch.relu(z), z, dy.double().cpu())
    assert torch.equal(dz[at], dy[at].double().cpu())
    dz = dz.numpy()
    close(dx[at], dz[at] @ exact(w), D.sum_error(dz[at:at + 1], exact(w).T), "dx of the row with a NaN")
    others, _ = D.backward(exact(x[keep]), exact(w), exact(bias), "relu", exact(dy[keep]), torch.finfo(x.dtype).eps)
    close(db, dz.sum(0), others["bias"][1] + 2.0 ** -23 * np.abs(dz).sum(0), "db")
    # (the NaN is in column 3 of x, and so of dw, alone)
    assert torch.isnan(dw[:, 3]).all() and torch.isfinite(dw[:, :3]).all() and torch.isfinite(dw[:, 4:]).all()


@pytest.mark.parametrize("rows,lines", [(1 << 21, 24), ((1 << 21) - 37, 33), (65536, 256), (100_001, 7)])
def test_bias_gradient_over_many_rows(linear, device, rows, lines):
    """Of gradients of one sign, whose sums go on growing, against 64-bit sums: a workgroup's 64
    rows are 34 additions in FP32, each off by half a step of the sum so far; what is added
    of those must not add to it, but for the result's rounding."""
    g = torch.Generator(device=device).manual_seed(rows)
    x = torch.randn(rows, 8, device=device, generator=g).bfloat16()
    w = torch.randn(lines, 8, device=device, generator=g).bfloat16()
    dy = 0.1 + 0.001 * torch.rand(rows, lines, device=device, generator=g)
    for dtype in ("fp32", "bf16"):
        bias = torch.zeros(lines, device=device, dtype=TYPES[dtype], requires_grad=True)
        db, = torch.autograd.grad(linear(x, w, bias, out_dtype=torch.float32), bias, dy)
        want = dy.double().sum(0).cpu().numpy()
        close(db, want, 34 * 2.0 ** -24 * want, f"db in {dtype}")


@pytest.mark.parametrize("activation", [None, "silu", "swiglu"])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_some_gradients_of_trainable_leaves(linear, device, activation, dtype):
    """Asked for by themselves, gradients have the bits that they have beside the others."""
    rng = np.random.default_rng(21)
    lines = 2 * 60 if activation == "swiglu" else 60
    t = {"x": normal(rng, (100, 72), dtype, device), "w": normal(rng, (lines, 72), dtype, device, 0.1),
         "bias": normal(rng, lines, "fp32", device), "residual": normal(rng, (100, 60), "fp32", device)}
    leaves = {k: v.requires_grad_() for k, v in t.items()}
    dy = normal(rng, (100, 60), dtype, device)
    y = linear(leaves["x"], leaves["w"], leaves["bias"], activation, leaves["residual"], TYPES[dtype])
    every = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy, retain_graph=True)))
    for names in (["x"], ["w"], ["bias"], ["residual"], ["w", "x"], ["residual", "bias"], ["bias", "x"]):
        for name, g in zip(names, torch.autograd.grad(y, [leaves[k] for k in names], dy, retain_graph=True)):
            assert torch.equal(g, every[name]), (names, name)


@pytest.mark.parametrize("activation", [None, "silu", "swiglu"])
def test_frozen_inputs_are_not_kept(linear, device, activation):
    """x written over where only its own and the bias's gradients are asked for, the weights where only
    theirs are: the bits that they have without it."""
    rng = np.random.default_rng(22)
    lines = 2 * 64 if activation == "swiglu" else 64
    for rows in (3, 130):
        x, w, bias = normal(rng, (rows, 72), "fp16", device), normal(rng, (lines, 72), "fp16", device, 0.1), normal(rng, lines, "fp32", device)
        dy = normal(rng, (rows, 64), "fp16", device)
        for names in (["x", "bias"], ["w", "bias"], ["bias"], ["x"], ["w"]):
            got = []
            for change in (False, True):
                t = {k: v.clone().requires_grad_(k in names) for k, v in (("x", x), ("w", w), ("bias", bias))}
                made = {k: (v * 1 if v.requires_grad else v) for k, v in t.items()}
                y = linear(made["x"], made["w"], made["bias"], activation)
                with torch.no_grad():
                    if change:
                        for k, other in (("x", "w"), ("w", "x")):
                            if other not in names:
                                made[k].fill_(float("nan"))
                got.append(torch.autograd.grad(y, [t[k] for k in names], dy))
            assert all(torch.equal(a, b) for a, b in zip(*got)), names


def test_a_residual_alone_keeps_no_memory(linear, device):
    x, w = (torch.zeros(256, k, device=device).half() for k in (64, 64))
    residual = torch.zeros(256, 256, device=device).half().requires_grad_()
    linear(x, w, None, "silu", residual)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated(device)
    y = linear(x, w, None, "silu", residual)
    assert torch.cuda.memory_allocated(device) - before == y.numel() * 2
    dy = torch.ones_like(y)
    assert torch.equal(torch.autograd.grad(y, residual, dy)[0], dy)


@pytest.mark.parametrize("which", ["y", "dx"])
def test_more_results_than_a_launch_has_smallest_tiles(linear, device, which):
    """2^21 and one rows of 8200 columns from 64: the forward's result, and the gradient of as many rows
    as it takes."""
    rows, n, k = (1 << 21) + (which == "y"), 8200, 64
    rng = np.random.default_rng(23)
    g = torch.Generator(device=device).manual_seed(23)
    small = torch.randn(rows, k, device=device, generator=g).bfloat16()
    if which == "y":
        w = normal(rng, (n, k), "bf16", device)
        got, want = linear(small, w), exact(w)
    else:
        w = normal(rng, (k, n), "bf16", device)
        x = torch.zeros(rows, n, device=device, dtype=torch.bfloat16, requires_grad=True)
        got, want = torch.autograd.grad(linear(x, w), x, small)[0], exact(w).T
    some = torch.tensor([0, 1, 127, 128, 65535, 1 << 20, rows - 130, rows - 2, rows - 1], device=device)
    a = exact(small[some])
    close(got[some], a @ want.T, D.sum_error(a, want), which)
    del got
    torch.cuda.empty_cache()


def test_refused_gradients_take_no_memory(linear, device):
    x, w = torch.zeros(1 << 21, 1, device=device).half(), torch.zeros(16448, 1, device=device).half().requires_grad_()
    before = torch.cuda.memory_allocated(device)
    torch.cuda.reset_peak_memory_stats(device)
    with pytest.raises(RuntimeError, match="too many rows and columns"):
        linear(x, w, None, "silu")
    assert torch.cuda.max_memory_allocated(device) == before


def grads_of(linear, x, w, bias, activation, dy):
    leaves = [t.detach().requires_grad_() for t in (x, w, bias)]
    y = linear(*leaves, activation, out_dtype=torch.float32)
    return torch.autograd.grad(y, leaves, dy)


@pytest.mark.parametrize("rows,n,k", [(200, 96, 64), (4000, 40, 72), (30, 3000, 72), (8, 33, 200)])
@pytest.mark.parametrize("activation", [None, "silu", "swiglu"])
def test_fp16_gradients_above_its_range(linear, device, rows, n, k, activation):
    """dz of about 2^20, which FP16 does not hold, and results that it does: dy of 2^20 before x and
    weights of 2^-14.  (Biases keep z, and with it the slopes and up lines, near 1.)"""
    rng = np.random.default_rng(rows + n)
    lines = 2 * n if activation == "swiglu" else n
    x, w = normal(rng, (rows, k), "fp16", device, 2.0 ** -14), normal(rng, (lines, k), "fp16", device, 2.0 ** -14)
    bias, dy = normal(rng, lines, "fp32", device), normal(rng, (rows, n), "fp32", device, 2.0 ** 20)
    wants, dz = D.backward(exact(x), exact(w), exact(bias), activation, exact(dy), torch.finfo(torch.float16).eps)
    assert np.abs(dz).max() > 2 * 65504
    for got, name in zip(grads_of(linear, x, w, bias, activation, dy), ("x", "w", "bias")):
        assert torch.isfinite(got).all() and np.abs(wants[name][0]).max() > 100
        close(got, *wants[name], name)


@pytest.mark.parametrize("rows,n,k", [(200, 96, 64), (4000, 40, 72), (30, 3000, 72), (8, 33, 200)])
@pytest.mark.parametrize("activation", [None, "silu", "swiglu"])
@pytest.mark.parametrize("which", ["x", "w"])
def test_fp16_gradients_below_its_range(linear, device, rows, n, k, activation, which):
    """dz of about 2^-26, which FP16 rounds to zero or its least numbers, and results among its normal ones:
    what dz is multiplied with is 2^13, the other operand as much smaller."""
    rng = np.random.default_rng(rows + n + 1)
    lines = 2 * n if activation == "swiglu" else n
    large, small = (13, -16) if which == "w" else (-16, 13)
    x, w = normal(rng, (rows, k), "fp16", device, 2.0 ** large), normal(rng, (lines, k), "fp16", device, 2.0 ** small)
    bias, dy = normal(rng, lines, "fp32", device), normal(rng, (rows, n), "fp32", device, 2.0 ** -26)
    wants, dz = D.backward(exact(x), exact(w), exact(bias), activation, exact(dy), torch.finfo(torch.float16).eps)
    # (as FP16 by itself would hold it, most of dz is lost)
    assert np.abs(dz.astype(np.float16) - dz).max() > np.abs(dz).max() / 100
    want = wants[which][0]
    assert np.median(np.abs(want)) > 2.0 ** -14
    for got, name in zip(grads_of(linear, x, w, bias, activation, dy), ("x", "w", "bias")):
        close(got, *wants[name], name)
