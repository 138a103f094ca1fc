"""The balance loss under fake tensors, tracers, dispatch modes and forward-mode
derivatives, on the CPU: tensors of a GPU that only pretend, and meta tensors."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx
from torch.utils._python_dispatch import TorchDispatchMode


@pytest.fixture(scope="module")
def loss_of():
    from vllm_mi355x.kernels.moe import moe_balance_loss
    return moe_balance_loss


def inputs(device, requires_grad=False, rows=6, experts=8):
    return (torch.empty(rows, experts, device=device, dtype=torch.bfloat16, requires_grad=requires_grad),
            torch.empty(rows, 2, dtype=torch.int32, device=device), torch.empty(rows, dtype=torch.bool, device=device))


def names(graph):
    return [str(n.target) for n in graph.graph.nodes if n.op == "call_function"]


@pytest.mark.parametrize("requires_grad", [False, True])
def test_fake_gpu_tensors(loss_of, requires_grad):
    with FakeTensorMode():
        logits, ids, pad = inputs("cuda", requires_grad)
        loss, counts = loss_of(logits, ids, "sigmoid", pad)
        assert loss.shape == () and loss.dtype == torch.float32 and loss.device.type == "cuda"
        assert counts.shape == (8,) and counts.dtype == torch.int64 and not counts.requires_grad
        assert loss.requires_grad == requires_grad
        with torch.no_grad():
            assert not loss_of(logits, ids)[0].requires_grad


def test_gradient_of_meta_tensors(loss_of):
    logits, ids, pad = inputs("meta", True)
    grad, = torch.autograd.grad(loss_of(logits, ids, is_padding=pad)[0], logits)
    assert grad.shape == (6, 8) and grad.dtype == torch.bfloat16
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(loss_of(logits, ids)[0], logits, create_graph=True)


@pytest.mark.parametrize("mode", ["real", "symbolic"])
def test_a_trace_holds_the_operators(loss_of, mode):
    """make_fx records what computes the loss and the gradient, not empty outputs."""
    logits, ids, pad = inputs("meta")
    traced = make_fx(lambda l, i, p: loss_of(l, i, "softmax", p), tracing_mode=mode)(logits, ids, pad)
    assert any("_vllm_mi355x.moe_balance" in n for n in names(traced)), names(traced)
    assert not any("aten.empty" in n for n in names(traced))

    def step(l, i, p):
        l = l.detach().requires_grad_()
        loss, counts = loss_of(l, i, "softmax", p)
        return loss.detach(), counts, torch.autograd.grad(loss, l)[0]

    traced = make_fx(step, tracing_mode=mode)(logits, ids, pad)
    got = names(traced)
    assert "_vllm_mi355x.moe_balance_forward.default" in got and "_vllm_mi355x.moe_balance_grad.default" in got, got
    assert not any("aten.empty" in n for n in got)
    out = traced(*inputs("meta"))
    assert [tuple(t.shape) for t in out] == [(), (8,), (6, 8)]


@pytest.mark.parametrize("requires_grad", [False, True])
def test_dispatch_modes_see_it(loss_of, requires_grad):
    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(str(func))
            return func(*args, **(kwargs or {}))

    logits, ids, pad = inputs("meta", requires_grad)
    with Watch():
        loss_of(logits, ids, is_padding=pad)
    assert any("moe_balance" in name for name in seen), seen


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(loss_of, requires_grad):
    """No tangent is dropped: the loss has no forward-mode derivative and says so."""
    logits, ids, _ = inputs("meta", requires_grad)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(logits, torch.ones_like(logits))
        with pytest.raises(RuntimeError, match="forward-mode"):
            loss_of(dual, ids)
        with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
            loss_of(dual, ids)
