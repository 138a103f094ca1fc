"""The balance loss around the border between calls in one workgroup and in
several: many rows of few experts, and one row more or less than one workgroup
takes.  Tolerances as in test_gpu_balance.py: FP32 sums of up to 1024 terms, 2^-18
of the magnitudes, then half a step of the type."""

import numpy as np
import pytest
import torch

from oracle import balance_oracle as B

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def loss_of():
    from vllm_mi355x.kernels.moe import moe_balance_loss
    return moe_balance_loss


@pytest.mark.parametrize("rows,experts,topk", [(512, 1, 1), (513, 1, 1), (32768, 1, 1), (512, 8, 2), (513, 8, 2), (4096, 8, 2),
                                               (8192, 4, 2), (512, 40, 3), (513, 40, 3), (256, 100, 4), (257, 100, 4),
                                               (128, 200, 4), (129, 200, 4), (64, 512, 8), (65, 512, 8)])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_around_the_border(loss_of, device, rows, experts, topk, sigmoid):
    print(f"balance border {rows}x{experts} sigmoid={sigmoid}", flush=True)
    rng = np.random.default_rng(rows + experts)
    logits = torch.from_numpy(rng.standard_normal((rows, experts)) * 2).float().to(device).requires_grad_()
    ids = rng.integers(-1, experts, (rows, topk)).astype(np.int32)
    padding = rng.random(rows) < 0.2
    loss, counts = loss_of(logits, torch.from_numpy(ids).to(device), "sigmoid" if sigmoid else "softmax",
                           torch.from_numpy(padding).to(device))
    grad, = torch.autograd.grad(loss, logits, torch.full((), float(rows), device=device))
    l = logits.detach().double().cpu().numpy()
    want, wc, wg = B.loss_and_grad(l, ids, sigmoid, padding)
    assert np.array_equal(counts.cpu().numpy(), wc)
    assert abs(loss.item() - want) <= 2.0 ** -18 * want
    kept = ~padding
    p, d = B.probabilities(l[kept], sigmoid)
    f = wc * (experts / (kept.sum() * topk))
    tol = np.zeros_like(l)
    tol[kept] = 2.0 ** -18 * d * (f + (p @ f)[:, None]) * (rows / kept.sum())
    tol = tol + 2.0 ** -24 * (np.abs(wg * rows) + tol) + 2.0 ** -149
    assert (np.abs(grad.double().cpu().numpy() - wg * rows) <= tol).all()
