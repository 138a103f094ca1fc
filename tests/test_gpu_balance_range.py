"""The balance loss with sigmoids of far negative logits against the FP64 oracle.

A row's p does not change where all its sigmoids are scaled alike, so it has the
same error wherever its logits lie.  With u = 2^-24: a sigmoid is off by 2^-22 (the
exponential) + 2 u (the reciprocal) + u, p by that, by as much again through the
sum, by (E / 64 + 8) u of the additions and 3 u of the quotient and products:
under 38 u up to 1024 experts, and so 2^-18 of p with the products by f.  An
exponential below 2^-126 may count as 0, under a sum of at least 2^-60 (a row is
scaled below that: to a largest of e^l / 2^k > 1/2 over 1 + e^l < 3/2): p then loses less
than 2^-66, which takes up to 2^-66 sum_e f_e from r = sum_e f_e p_e.  A gradient p (1 - s) (f -
r) g / n is off by the same part of its two terms' magnitudes, by what its own p and
r lost, then half a step of its type.
"""

import numpy as np
import pytest
import torch

from oracle import balance_oracle as B

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def loss_of():
    from vllm_mi355x.kernels.moe import moe_balance_loss
    return moe_balance_loss


def far_rows(rng, rows, experts, dtype, device):
    """Rows whose logits all lie around one far negative level, with masks, a few
    larger logits and rows below what leaves anything among them."""
    level = rng.choice([-0.4, -3.0, -30.0, -80.0, -88.0, -93.0, -101.0, -150.0, -300.0, -690.0], (rows, 1))
    x = level + rng.standard_normal((rows, experts)) * 3
    x[rows // 2] = -95.0
    if rows > 8:
        x[0] = np.linspace(-100, -86, experts)
        x[1, ::2] = -np.inf
        x[2, 1:] = float(torch.finfo(TYPES[dtype]).min)
        x[3] = -720.0
        x[4] = -np.inf
        x[5, 0] = 4.0
        x[6] = -np.abs(x[6]) - 760
        x[7] = -88.0
        x[7, -1] = -90.0
    return torch.from_numpy(x).to(TYPES[dtype]).to(device)


@pytest.mark.parametrize("rows,experts", [(1, 1), (1, 8), (12, 2), (40, 8), (200, 40), (130, 256), (20, 600), (10, 1024),
                                          (3000, 16), (700, 100), (200, 250), (100, 512)])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_shares_of_far_negative_logits(loss_of, device, rows, experts, dtype):
    print(f"balance range {rows}x{experts} {dtype}", flush=True)
    rng = np.random.default_rng(rows * 7 + experts)
    logits = far_rows(rng, rows, experts, dtype, device).requires_grad_()
    ids = rng.integers(0, experts, (rows, 2)).astype(np.int32)
    loss, _ = loss_of(logits, torch.from_numpy(ids).to(device), "sigmoid")
    upstream = float(rows)
    grad, = torch.autograd.grad(loss, logits, torch.full((), upstream, device=device))
    l = logits.detach().double().cpu().numpy()
    want, counts, wg = B.loss_and_grad(l, ids, True)
    f = counts * (experts / (rows * 2))
    p, d = B.probabilities(l, True)
    r = (p @ f)[:, None]
    assert abs(loss.item() - want) <= 2.0 ** -18 * want + 2.0 ** -66 * f.sum()
    tol = ((2.0 ** -18 * d + 2.0 ** -66) * (f + r) + d * 2.0 ** -66 * f.sum()) * (upstream / rows)
    info = torch.finfo(TYPES[dtype])
    tol = tol + info.eps / 2 * (np.abs(wg * upstream) + tol) + info.smallest_normal * info.eps
    off = np.abs(grad.double().cpu().numpy() - wg * upstream) - tol
    assert (off <= 0).all(), f"max excess {off.max():.3g} at {np.unravel_index(off.argmax(), off.shape)}"


def test_two_experts_by_hand(loss_of, device):
    """Logits of -88 and -90 share as 1 : e^-2; -720 and masked rows have no shares."""
    logits = torch.tensor([[-88.0, -90.0], [-720.0, -720.0], [-float("inf"), -3.4e38]], device=device)
    ids = torch.zeros(3, 1, dtype=torch.int32, device=device)
    loss, _ = loss_of(logits, ids, "sigmoid")  # f = (2, 0): the mean of 2 p_0
    want = 2 / (1 + np.exp(-2.0)) / 3
    assert abs(loss.item() - want) <= 2.0 ** -18 * want
