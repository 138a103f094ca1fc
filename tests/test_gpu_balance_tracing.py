"""The balance loss traced on the GPU: a recorded graph and a compiled function
give the eager call's bits, for new inputs too."""

import numpy as np
import pytest
import torch
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def loss_of():
    from vllm_mi355x.kernels.moe import moe_balance_loss
    return moe_balance_loss


def inputs(device, seed, rows=300, experts=40):
    rng = np.random.default_rng(seed)
    return (torch.from_numpy(rng.standard_normal((rows, experts)) * 2).bfloat16().to(device),
            torch.from_numpy(rng.integers(-1, experts, (rows, 3)).astype(np.int32)).to(device),
            torch.from_numpy(rng.random(rows) < 0.2).to(device))


@pytest.mark.parametrize("scoring", ["softmax", "sigmoid"])
def test_a_recorded_graph_repeats_the_eager_call(loss_of, device, scoring):
    def step(l, i, p):
        l = l.detach().requires_grad_()
        loss, counts = loss_of(l, i, scoring, p)
        return loss.detach(), counts, torch.autograd.grad(loss, l)[0]

    plain = make_fx(lambda l, i, p: loss_of(l, i, scoring, p))(*inputs(device, 0))
    whole = make_fx(step)(*inputs(device, 0))
    for seed in (0, 1, 2):
        args = inputs(device, seed)
        want = step(*args)
        assert all(torch.equal(a, b) for a, b in zip(whole(*args), want))
        assert all(torch.equal(a, b) for a, b in zip(plain(*args), want[:2]))


def test_a_compiled_function_repeats_the_eager_call(loss_of, device):
    def step(l, i, p):
        loss, counts = loss_of(l, i, "sigmoid", p)
        return 2 * loss, counts

    compiled = torch.compile(step, backend="aot_eager", dynamic=False)
    for seed in (3, 4):
        l, i, p = inputs(device, seed)
        a, b = l.clone().requires_grad_(), l.clone().requires_grad_()
        (x, cx), (y, cy) = step(a, i, p), compiled(b, i, p)
        x.backward()
        y.backward()
        assert torch.equal(x, y) and torch.equal(cx, cy) and torch.equal(a.grad, b.grad)


def test_forward_mode_is_refused(loss_of, device):
    l, i, p = inputs(device, 5)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward-mode"):
            loss_of(forward_ad.make_dual(l, torch.ones_like(l)), i, is_padding=p)
