"""The dense layer's gradients without a GPU: what a backward pass computes and what the forward
keeps for it, by the operators that are called on meta tensors."""

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode


@pytest.fixture(scope="module")
def linear():
    from vllm_mi355x.kernels.dense import dense_linear
    return dense_linear


class Calls(TorchDispatchMode):
    """The dense layer's operators that run, with their arguments by name."""

    def __init__(self):
        super().__init__()
        self.seen = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        if "dense_linear" in str(func):
            named = dict(zip((a.name for a in func._schema.arguments), args), **(kwargs or {}))
            self.seen.append((func._schema.name.split("::")[1], named))
        return func(*args, **(kwargs or {}))


def leaves(with_bias=True, with_residual=True, lines=5):
    t = {"x": torch.empty(6, 8, device="meta", dtype=torch.half), "w": torch.empty(lines, 8, device="meta", dtype=torch.half)}
    if with_bias:
        t["bias"] = torch.empty(lines, device="meta")
    if with_residual:
        t["residual"] = torch.empty(6, 5, device="meta", dtype=torch.bfloat16)
    return t


@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("activation", [None, "silu"])
def test_a_backward_pass_computes_what_it_is_asked_for(linear, with_bias, with_residual, activation):
    t = {k: v.requires_grad_() for k, v in leaves(with_bias, with_residual).items()}
    y = linear(t["x"], t["w"], t.get("bias"), activation, t.get("residual"))
    for asked in [[k] for k in t] + [["x", "w"], list(t)]:
        with Calls() as calls:
            grads = torch.autograd.grad(y, [t[k] for k in asked], torch.empty_like(y), retain_graph=True)
        assert [(g.shape, g.dtype) for g in grads] == [(t[k].shape, t[k].dtype) for k in asked]
        if asked == ["residual"]:
            assert not calls.seen
            continue
        (name, args), = calls.seen
        assert name == "dense_linear_grad"
        assert (args["need_x"], args["need_w"], args["bias_dtype"] is not None) == ("x" in asked, "w" in asked, "bias" in asked), asked


@pytest.mark.parametrize("which", ["x", "w", "bias", "residual"])
def test_a_single_trainable_input(linear, which):
    t = leaves()
    t[which].requires_grad_()
    y = linear(t["x"], t["w"], t["bias"], "gelu", t["residual"])
    y.backward(torch.empty_like(y))
    assert [k for k, v in t.items() if v.grad is not None] == [which] and t[which].grad.dtype == t[which].dtype
