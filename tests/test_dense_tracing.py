"""The dense layer on meta and fake tensors refuses the shapes and types that it refuses on a GPU, so
that a graph that cannot run is not traced."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx


@pytest.fixture(scope="module")
def linear():
    from vllm_mi355x.kernels.dense import dense_linear
    return dense_linear


def e(*shape, dtype=torch.half, device="meta"):
    return torch.empty(*shape, dtype=dtype, device=device)


def refused(linear, device):
    t = lambda *s, **k: e(*s, device=device, **k)
    x, w, b, r = t(6, 16), t(8, 16), t(8), t(6, 8)
    return [lambda: linear(x, t(8, 15)), lambda: linear(x, t(8, 17)), lambda: linear(t(6, 0), t(8, 0)), lambda: linear(x, t(0, 16)),
            lambda: linear(x, t(7, 16), activation="swiglu"), lambda: linear(x, w, t(7)), lambda: linear(x, w, t(8, 1)),
            lambda: linear(x, w, t(4), "swiglu"), lambda: linear(x, w, t(8, dtype=torch.double)), lambda: linear(x, w, residual=t(5, 8)),
            lambda: linear(x, w, residual=t(6, 7)), lambda: linear(x, w, residual=t(8)), lambda: linear(x, w, activation="swiglu", residual=r),
            lambda: linear(x, w, residual=t(1, 8)), lambda: linear(x, t(8, 16, dtype=torch.bfloat16)), lambda: linear(x.float(), w.float()),
            lambda: linear(x, w, out_dtype=torch.double), lambda: linear(x, t(8)), lambda: linear(x, w, out=t(5, 8)), lambda: linear(x, w, out=t(6, 7)),
            lambda: linear(x, w, out=t(48)), lambda: linear(x, w, out=t(6, 8, dtype=torch.double)), lambda: linear(x, w, out=t(8, 6).t()),
            lambda: linear(x, w, t(7), out=t(6, 8))]


@pytest.mark.parametrize("device", ["meta", "cuda"])
def test_refusals(linear, device):
    with FakeTensorMode():
        for i, call in enumerate(refused(linear, device)):
            with pytest.raises(RuntimeError):
                call()
                pytest.fail(f"call {i} taken")


@pytest.mark.parametrize("activation", [None, "silu", "swiglu"])
def test_refusals_with_gradients(linear, activation):
    """(With k = 0 the number of rows was a division by it.)"""
    for x, w in (((6, 0), (8, 0)), ((6, 16), (8, 15)), ((6, 16), (0, 16))):
        with pytest.raises(RuntimeError):
            linear(e(*x).requires_grad_(), e(*w), activation=activation)
            pytest.fail("taken")


def test_symbolic_sizes(linear):
    """A trace with sizes of no value checks what relates them and keeps them open."""
    step = lambda x, w, b, r: linear(x, w, b, "silu", r)
    args = e(6, 16), e(12, 16), e(12), e(6, 12)
    traced = make_fx(step, tracing_mode="symbolic")(*args)
    assert traced(*args).shape == (6, 12) and traced(e(9, 20), e(32, 20), e(32), e(9, 32)).shape == (9, 32)
    for bad in ((e(6, 16), e(12, 15), e(12), e(6, 12)), (e(6, 16), e(12, 16), e(11), e(6, 12)), (e(6, 16), e(12, 16), e(12), e(5, 12))):
        with pytest.raises(RuntimeError):
            make_fx(step, tracing_mode="symbolic")(*bad)
