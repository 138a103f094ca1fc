"""The dense layer's gradients without a GPU: what a backward pass computes and what the forward
keeps for it, by the operators that are called on meta tensors."""

import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode


@pytest.fixture(scope="module")
def linear():
    from vllm_mi355x.kernels.dense import dense_linear
    return dense_linear


@pytest.fixture(scope="module")
def lib():
    from vllm_mi355x import _native
    return _native.load()


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


def test_a_residual_alone_keeps_nothing(linear):
    t = leaves()
    t["residual"].requires_grad_()
    with Calls() as calls:
        y = linear(t["x"], t["w"], t["bias"], "silu", t["residual"])
    assert [name for name, _ in calls.seen] == ["dense_linear"] and y.requires_grad


@pytest.mark.parametrize("activation", [None, "gelu"])
@pytest.mark.parametrize("trained", [["x"], ["w"], ["bias"], ["x", "bias"], ["w", "bias"], ["residual"], ["x", "w"]])
def test_what_is_not_kept_may_change(linear, activation, trained):
    """The gradient of x is computed from the weights, theirs from x: a frozen one's counterpart is
    neither kept nor found to have changed; the one that is used is."""
    t = {k: v.requires_grad_(k in trained) for k, v in leaves().items()}
    made = {k: (v * 1 if v.requires_grad else v) for k, v in t.items()}  # (leaves cannot be written to)
    y = linear(made["x"], made["w"], made["bias"], activation, made["residual"])
    used = {"x": "w" in trained, "w": "x" in trained, "bias": False, "residual": False}
    with torch.no_grad():
        for k, v in made.items():
            if not used[k]:
                v.add_(1)
    with Calls() as calls:
        grads = torch.autograd.grad(y, [t[k] for k in trained], torch.empty_like(y), retain_graph=True)
    assert [(g.shape, g.dtype) for g in grads] == [(t[k].shape, t[k].dtype) for k in trained]
    for _, args in calls.seen:
        assert (args["x"] is not None) == used["x"] and (args["w"] is not None) == used["w"]
    for k in ("x", "w"):
        if used[k]:
            with torch.no_grad():
                made[k].add_(1)
            with pytest.raises(RuntimeError, match="modified by an inplace operation"):
                torch.autograd.grad(y, [t[k] for k in trained], torch.empty_like(y), retain_graph=True)


def test_null_operands(lib):
    """The entry point takes null for what it does not read: the next check is the workspace's."""
    from tests.test_dense_cpu import grad
    for args, word in ((grad(x=0, dw=0, work=0), "workspace"), (grad(w=0, dx=0, work=0), "workspace"),
                       (grad(x=0, w=0, dx=0, dw=0, work=0), "workspace"), (grad(x=0, work=0), "null"), (grad(w=0, work=0), "null")):
        assert lib.dense_linear_grad(*args) == 1
        assert word in lib.vllm_mi355x_last_error().decode(), lib.vllm_mi355x_last_error()


@pytest.mark.parametrize("rows,k,n", [(1 << 21, 64, 16384), ((1 << 21) + 1, 64, 8200), (1 << 26, 8, 300), (400, 128, 1 << 23), (1 << 21, 192, 16384),
                                      (1 << 22, 64, 20000)])
@pytest.mark.parametrize("residual", [0, 1])
def test_large_results_have_a_plan(lib, rows, k, n, residual):
    """Of few stages the smallest tiles are the fastest, but not more of them than a launch takes
    (2^22): within the sizes that are taken, a result that fits a card is not refused."""
    from tests.test_dense_cpu import plan
    kind, tile_rows, lines, splits, _ = plan(lib, rows, k, n, 0, residual)
    assert kind == 0 and -(-rows // tile_rows) * -(-n // lines) * splits <= 1 << 22


@pytest.mark.parametrize("x,w", [(((1 << 21), 1), (16448, 1)), ((1 << 20, 2, 1), (16448, 1)), ((1 << 21, 16448), (1, 16448)), ((4, 1 << 21), ((1 << 14) + 64, 1 << 21)),
                                 (((1 << 21) + 1, 8), (5, 8)), ((4, 8), ((1 << 21) + 1, 8))])
def test_a_gradient_that_would_be_refused_is_at_the_call(linear, lib, x, w):
    """Not after the forward pass has run; without a gradient the call is taken."""
    rows = torch.empty(*x, device="meta", dtype=torch.half)
    weights = torch.empty(*w, device="meta", dtype=torch.half)
    assert lib.dense_linear_grad_workspace_size(rows.numel() // x[-1], x[-1], w[0], 0, 0, 1, 0) == -1
    assert linear(rows, weights).shape == (*x[:-1], w[0])
    with pytest.raises(RuntimeError, match="too many rows and columns|a gradient takes up to"):
        linear(rows, weights.requires_grad_())
    with pytest.raises(RuntimeError, match="too many rows and columns|a gradient takes up to"):
        linear(rows, weights.detach(), torch.empty(w[0], device="meta", requires_grad=True), "silu")
    # (a residual's gradient needs no product)
    residual = torch.empty(*x[:-1], w[0], device="meta", requires_grad=True)
    assert linear(rows, weights.detach(), None, "silu", residual).requires_grad


def test_every_plan_of_the_gradients_has_a_size(lib):
    """The sizes of test_gpu_dense_grad_plans.py: both products on every kernel, every tile with and
    without K splits (the smallest short ring is for products of few stages, which are not split)."""
    from tests.test_dense_cpu import plan
    from tests.test_gpu_dense_grad_plans import SIZES
    seen = {"x": set(), "w": set()}
    for rows, k, lines, _ in SIZES:
        for name, size in (("x", (rows, lines, k)), ("w", (lines, rows, k))):
            kind, tile_rows, tile_lines, parts, ring = plan(lib, *size, 0, 0)
            seen[name].add((kind, tile_rows, tile_lines, ring, parts > 1) if kind == 0 else (kind,))
    tiles = ((256, 256, 5), (128, 256, 6), (128, 64, 6), (64, 64, 8), (128, 64, 4))
    for name, got in seen.items():
        for shape in tiles:
            assert {(0, *shape, False), (0, *shape, True)} <= got, (name, shape)
        assert (0, 64, 64, 4, False) in got and got & {(1,), (2,)}, name


@pytest.mark.parametrize("trained", [["x"], ["w"], ["bias"], ["residual"], ["x", "residual"]])
@pytest.mark.parametrize("mode", ["real", "symbolic"])
def test_traces_of_some_trainable_inputs(linear, trained, mode):
    """A trace holds the gradient without the operands that it does not read, for other sizes too."""
    from torch.fx.experimental.proxy_tensor import make_fx

    def step(x, w, bias, residual, dy):
        t = {k: v.detach().requires_grad_(k in trained) for k, v in (("x", x), ("w", w), ("bias", bias), ("residual", residual))}
        y = linear(t["x"], t["w"], t["bias"], "swiglu", t["residual"])
        return torch.autograd.grad(y, [t[k] for k in trained], dy)

    def args(rows, k, n):
        return [torch.empty(*s, device="meta", dtype=torch.half) for s in ((rows, k), (2 * n, k), (2 * n,), (rows, n), (rows, n))]

    shapes = lambda a: [tuple(a[("x", "w", "bias", "residual").index(k)].shape) for k in trained]
    traced = make_fx(step, tracing_mode=mode)(*args(6, 8, 5))
    for size in ((6, 8, 5), (9, 24, 7))[:2 if mode == "symbolic" else 1]:
        assert [tuple(g.shape) for g in traced(*args(*size))] == shapes(args(*size))
    calls = [n for n in traced.graph.nodes if "dense_linear_grad" in str(n.target)]
    assert len(calls) == (trained != ["residual"])
    for call in calls:
        assert (call.args[0] is None) == ("w" not in trained) and (call.args[1] is None) == ("x" not in trained)
