"""Routing from logits on meta and fake tensors refuses the shapes and types that it refuses on a GPU, so
that a graph that cannot run is not traced."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.fx.experimental.proxy_tensor import make_fx


@pytest.fixture(scope="module")
def route():
    from vllm_mi355x.kernels.moe import moe_route_logits
    return moe_route_logits


def e(*shape, dtype=torch.half, device="meta"):
    return torch.empty(*shape, dtype=dtype, device=device)


def refused(route, device, trained):
    t = lambda *s, **k: e(*s, device=device, **k)
    l = t(6, 16).requires_grad_(trained)
    f = lambda *s: t(*s, dtype=torch.float32)
    return [lambda: route(l, 17), lambda: route(l, 0), lambda: route(t(6, 128), 65), lambda: route(t(6, 1025), 2), lambda: route(t(6, 0), 1),
            lambda: route(l, 2, num_groups=3), lambda: route(l, 2, num_groups=0), lambda: route(t(6, 128), 2, num_groups=128),
            lambda: route(l, 2, num_groups=4, topk_groups=5), lambda: route(l, 2, num_groups=4, topk_groups=0),
            lambda: route(l, 5, num_groups=4, topk_groups=1), lambda: route(t(6, 16, dtype=torch.double), 2), lambda: route(t(16), 2),
            lambda: route(l, 2, f(15)), lambda: route(l, 2, t(16)), lambda: route(l, 2, f(16, 1)), lambda: route(l, 2, routed_scaling_factor=float("inf")),
            lambda: route(l, 2, routed_scaling_factor=float("nan")), lambda: route(l, 2, is_padding=t(5, dtype=torch.bool)),
            lambda: route(l, 2, is_padding=t(6, dtype=torch.int32)), lambda: route(l, 2, is_padding=t(6, 1, dtype=torch.bool))]


@pytest.mark.parametrize("device", ["meta", "cuda"])
@pytest.mark.parametrize("trained", [False, True])
def test_refusals(route, device, trained):
    with FakeTensorMode():
        for i, call in enumerate(refused(route, device, trained)):
            with pytest.raises(RuntimeError):
                call()
                pytest.fail(f"call {i} taken")


def test_symbolic_sizes(route):
    """A trace with sizes of no value checks what relates them and keeps them open."""
    step = lambda l, b, p: route(l, 2, b, num_groups=2, topk_groups=1, is_padding=p)
    args = lambda m, n: (e(m, n), e(n, dtype=torch.float32), e(m, dtype=torch.bool))
    traced = make_fx(step, tracing_mode="symbolic")(*args(6, 12))
    assert [tuple(t.shape) for t in traced(*args(6, 12))] == [(6, 2)] * 2 and [tuple(t.shape) for t in traced(*args(9, 32))] == [(9, 2)] * 2
    for bad in ((e(6, 13), e(13, dtype=torch.float32), args(6, 1)[2]), (e(6, 12), e(11, dtype=torch.float32), args(6, 1)[2]),
                (*args(6, 12)[:2], args(5, 1)[2]), args(6, 2)):
        with pytest.raises(RuntimeError):
            make_fx(step, tracing_mode="symbolic")(*bad)
