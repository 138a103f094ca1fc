"""Routing from logits without a GPU: the entry points' refusals before anything runs,
and its shapes under meta tensors, tracers and forward-mode derivatives."""

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

A = 1 << 30  # an address that no check follows; the others lie A apart
INF = float("inf")


@pytest.fixture(scope="module")
def lib():
    from vllm_mi355x import _native
    return _native.load()


@pytest.fixture(scope="module")
def route():
    from vllm_mi355x.kernels.moe import moe_route_logits
    return moe_route_logits


def call(logits=A, dtype=2, rows=100, experts=16, stride=16, bias=2 * A, topk=2, groups=4, topk_groups=2, scoring=1, scale=1.0, pad=3 * A,
         weights=4 * A, ids=5 * A):
    return (logits, dtype, rows, experts, stride, bias, topk, groups, topk_groups, scoring, 1, scale, pad, weights, ids, 0)


def grad(logits=A, dtype=2, rows=100, experts=16, stride=16, weights=2 * A, ids=3 * A, topk=2, up=4 * A, out=5 * A):
    return (logits, dtype, rows, experts, stride, weights, ids, topk, 0, 1, up, out, 0)


@pytest.mark.parametrize("name,args,word", [
    ("moe_route_logits", call(dtype=3), "BF16"), ("moe_route_logits", call(rows=-1), "rows"), ("moe_route_logits", call(rows=1 << 31), "rows"),
    ("moe_route_logits", call(experts=0), "experts"), ("moe_route_logits", call(experts=1028, stride=1028), "experts"),
    ("moe_route_logits", call(topk=0), "topk"), ("moe_route_logits", call(topk=17), "topk"),
    ("moe_route_logits", call(experts=128, stride=128, topk=65, groups=1, topk_groups=1), "topk"),
    ("moe_route_logits", call(topk=9), "fit"), ("moe_route_logits", call(groups=3), "groups"), ("moe_route_logits", call(groups=0), "groups"),
    ("moe_route_logits", call(experts=128, stride=128, groups=128), "groups"), ("moe_route_logits", call(topk_groups=0), "topk_groups"),
    ("moe_route_logits", call(topk_groups=5), "topk_groups"), ("moe_route_logits", call(scoring=2), "scoring"),
    ("moe_route_logits", call(scale=INF), "finite"), ("moe_route_logits", call(scale=float("nan")), "finite"),
    ("moe_route_logits", call(stride=15), "stride"), ("moe_route_logits", call(stride=-16), "stride"),
    ("moe_route_logits", call(logits=0), "null"), ("moe_route_logits", call(weights=0), "null"), ("moe_route_logits", call(ids=0), "null"),
    ("moe_route_logits", call(weights=A), "overlap"), ("moe_route_logits", call(ids=4 * A + 796), "overlap"),
    ("moe_route_logits", call(ids=2 * A + 60), "overlap"), ("moe_route_logits", call(weights=3 * A + 96), "overlap"),
    ("moe_route_logits", call(logits=A + 2), "misaligned"), ("moe_route_logits", call(bias=2 * A + 1), "misaligned"),
    ("moe_route_logits", call(ids=5 * A + 2), "misaligned"),
    ("moe_route_grad", grad(out=0), "null"), ("moe_route_grad", grad(up=0), "null"), ("moe_route_grad", grad(out=A), "overlap"),
    ("moe_route_grad", grad(out=5 * A + 8), "misaligned"), ("moe_route_grad", grad(up=5 * A + 6396), "overlap"),
    ("moe_route_grad", grad(topk=20), "topk")])
def test_refusals(lib, name, args, word):
    assert getattr(lib, name)(*args) == 1
    assert word in lib.vllm_mi355x_last_error().decode(), lib.vllm_mi355x_last_error()


def test_no_rows_launch_nothing(lib):
    assert lib.moe_route_logits(*call(rows=0, logits=0, weights=0, ids=0)) == 0
    assert lib.moe_route_grad(*grad(rows=0, logits=0, weights=0, ids=0, up=0, out=0)) == 0


def test_shapes_and_gradient_of_meta_tensors(route):
    logits = torch.empty(6, 8, device="meta", dtype=torch.bfloat16, requires_grad=True)
    w, ids = route(logits, 2, num_groups=4, topk_groups=2)
    assert w.shape == ids.shape == (6, 2) and w.dtype == torch.float32 and ids.dtype == torch.int32 and not ids.requires_grad
    grad, = torch.autograd.grad(w, logits, torch.empty(6, 2, device="meta"))
    assert grad.shape == (6, 8) and grad.dtype == torch.bfloat16
    with pytest.raises(RuntimeError, match="create_graph"):
        w, _ = route(logits, 2)
        torch.autograd.grad(w, logits, torch.empty(6, 2, device="meta"), create_graph=True)
    with FakeTensorMode():
        fake = torch.empty(6, 8, device="cuda")
        w, ids = route(fake, 3, is_padding=torch.empty(6, dtype=torch.bool, device="cuda"))
        assert w.device.type == "cuda" and w.shape == (6, 3) and not w.requires_grad


@pytest.mark.parametrize("mode", ["real", "symbolic"])
def test_a_trace_holds_the_operators(route, mode):
    def step(l, up):
        l = l.detach().requires_grad_()
        w, ids = route(l, 2, scoring="softmax")
        return w.detach(), ids, torch.autograd.grad(w, l, up)[0]

    args = torch.empty(6, 8, device="meta"), torch.empty(6, 2, device="meta")
    traced = make_fx(step, tracing_mode=mode)(*args)
    names = [str(n.target) for n in traced.graph.nodes if n.op == "call_function"]
    assert "_vllm_mi355x.moe_route_logits.default" in names and "_vllm_mi355x.moe_route_grad.default" in names, names
    assert [tuple(t.shape) for t in traced(*args)] == [(6, 2), (6, 2), (6, 8)]


@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode_is_refused(route, requires_grad):
    logits = torch.empty(6, 8, device="meta", requires_grad=requires_grad)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(logits, torch.ones_like(logits))
        with pytest.raises(RuntimeError, match="forward-mode"):
            route(dual, 2)
