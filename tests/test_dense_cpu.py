"""The dense layer without a GPU: the entry points' refusals before anything runs, the plans, and
shapes under meta tensors, tracers and forward-mode derivatives."""

import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
from torch.autograd import forward_ad
from torch.fx.experimental.proxy_tensor import make_fx

A = 1 << 36  # an address that no check follows; the others lie A apart
INF = float("inf")


@pytest.fixture(scope="module")
def lib():
    from vllm_mi355x import _native
    return _native.load()


@pytest.fixture(scope="module")
def linear():
    from vllm_mi355x.kernels.dense import dense_linear
    return dense_linear


def call(x=A, dtype=0, rows=100, k=64, xs=64, w=2 * A, n=32, ws=64, bias=3 * A, bd=2, act=4, limit=INF, res=4 * A, rd=0, rs=32, out=5 * A,
         od=0, z=0, work=6 * A, size=1 << 30):
    return x, dtype, rows, k, xs, w, n, ws, bias, bd, act, limit, res, rd, rs, out, od, z, work, size, 0


def grad(x=A, dtype=0, rows=100, k=64, xs=64, w=2 * A, n=32, ws=64, z=3 * A, act=4, limit=INF, dy=4 * A, dd=0, ds=32, dx=5 * A, dw=6 * A,
         db=7 * A, bd=2, work=8 * A, size=1 << 30):
    return x, dtype, rows, k, xs, w, n, ws, z, act, limit, dy, dd, ds, dx, dw, db, bd, work, size, 0


@pytest.mark.parametrize("name,args,word", [
    ("dense_linear", call(dtype=2), "BF16 or FP16"), ("dense_linear", call(rows=-1), "rows"), ("dense_linear", call(rows=(1 << 26) + 1), "rows"),
    ("dense_linear", call(k=0), "k must"), ("dense_linear", call(k=(1 << 21) + 1), "k must"), ("dense_linear", call(n=0), "columns"),
    ("dense_linear", call(n=(1 << 23) + 1, act=5), "columns"), ("dense_linear", call(act=6), "activation"), ("dense_linear", call(act=-1), "activation"),
    ("dense_linear", call(bd=3), "FP32"), ("dense_linear", call(rd=5), "FP32"), ("dense_linear", call(od=7), "FP32"),
    ("dense_linear", call(x=0), "null"), ("dense_linear", call(w=0), "null"), ("dense_linear", call(out=0), "null"),
    ("dense_linear", call(xs=63), "stride"), ("dense_linear", call(ws=63), "stride"), ("dense_linear", call(rs=31), "stride"),
    ("dense_linear", call(limit=0.0), "limit"), ("dense_linear", call(limit=float("nan")), "limit"),
    ("dense_linear", call(k=4096, xs=4096, ws=4096, size=16), "workspace"), ("dense_linear", call(k=4096, xs=4096, ws=4096, work=0), "workspace"),
    ("dense_linear", call(k=65, xs=65, ws=65, work=6 * A + 8), "workspace"), ("dense_linear", call(xs=66, work=0), "workspace"),
    ("dense_linear", call(out=A), "overlap"), ("dense_linear", call(out=4 * A + 2), "overlap"), ("dense_linear", call(res=5 * A, rs=40), "overlap"),
    ("dense_linear", call(out=4 * A, od=2), "overlap"), ("dense_linear", call(z=5 * A), "overlap"),
    ("dense_linear", call(x=A + 1), "misaligned"), ("dense_linear", call(out=5 * A + 1), "misaligned"), ("dense_linear", call(bias=3 * A + 2), "misaligned"),
    ("dense_linear", call(z=7 * A + 2), "misaligned"),
    ("dense_linear_grad", grad(rows=0), "no rows"), ("dense_linear_grad", grad(dy=0), "null"), ("dense_linear_grad", grad(z=0), "null"),
    ("dense_linear_grad", grad(ds=31), "stride"), ("dense_linear_grad", grad(size=1 << 10), "workspace"), ("dense_linear_grad", grad(work=0), "workspace"),
    ("dense_linear_grad", grad(dx=A), "overlap"), ("dense_linear_grad", grad(dw=5 * A + 100), "overlap"), ("dense_linear_grad", grad(db=4 * A), "overlap"),
    ("dense_linear_grad", grad(rows=(1 << 21) + 1), "2^21"), ("dense_linear_grad", grad(dw=6 * A + 1), "misaligned")])
def test_refusals(lib, name, args, word):
    assert getattr(lib, name)(*args) == 1
    assert word in lib.vllm_mi355x_last_error().decode(), lib.vllm_mi355x_last_error()


def test_no_rows_and_sizes(lib):
    assert lib.dense_linear(*call(rows=0, x=0, w=0, out=0, work=0, size=0)) == 0
    assert lib.dense_linear_workspace_size(A, 0, 64, 64, 2 * A, 32, 64, 0) == 0
    assert lib.dense_linear_workspace_size(A, 1, 64, 64, 2 * A, 32, 64, 0) == 0
    assert lib.dense_linear_workspace_size(A, -1, 64, 64, 2 * A, 32, 64, 0) == -1
    # rows off 16 bytes are packed into it: 100 of 72, and 40 lines
    assert lib.dense_linear_workspace_size(A, 100, 65, 65, 2 * A, 40, 72, 0) >= 100 * 72 * 2 + 40 * 72 * 2
    assert lib.dense_linear_workspace_size(A, 100, 64, 72, 2 * A, 40, 80, 0) == 0
    assert lib.dense_linear_workspace_size(A + 2, 100, 64, 72, 2 * A, 40, 80, 0) >= 100 * 64 * 2
    assert lib.dense_linear_grad_workspace_size(100, 64, 32, 7, 1, 1, 1) == -1
    assert lib.dense_linear_grad_workspace_size((1 << 21) + 1, 64, 32, 0, 1, 1, 1) == -1
    assert lib.dense_linear_grad_workspace_size(1 << 21, 1 << 15, 32, 0, 1, 1, 1) == -1


def plan(lib, *size):
    out = (ctypes.c_int32 * 5)()
    assert lib.dense_linear_plan(*size, out) == 0
    return list(out)


def test_every_plan_has_a_size(lib):
    """The sizes at which test_gpu_dense_plans.py runs reach every kernel and split."""
    from tests.test_gpu_dense_plans import SIZES
    seen = set()
    for rows, k, n, gated in SIZES:
        kind, tile_rows, lines, parts, ring = plan(lib, rows, k, n, 5 if gated else 0, 1)
        seen.add((kind, tile_rows, lines, ring, parts > 1, gated))
    for gated in (False, True):
        for shape in ((256, 256, 5), (128, 256, 6), (128, 64, 6), (64, 64, 8)):
            assert (0, *shape, False, gated) in seen and (0, *shape, True, gated) in seen, (shape, gated)
        assert (0, 128, 64, 4, False, gated) in seen and (0, 64, 64, 4, False, gated) in seen
        assert {s[0] for s in seen if s[-1] == gated} == {0, 1, 2}
    assert {(2, 0, 1, 0, False, False), (2, 0, 1, 0, True, False), (2, 0, 2, 0, False, False), (2, 0, 2, 0, True, True)} <= seen


def test_shapes_and_gradient_of_meta_tensors(linear):
    x = torch.empty(3, 5, 16, device="meta", dtype=torch.half, requires_grad=True)
    w = torch.empty(12, 16, device="meta", dtype=torch.half, requires_grad=True)
    b, r = torch.empty(12, device="meta", requires_grad=True), torch.empty(3, 5, 6, device="meta", dtype=torch.half, requires_grad=True)
    y = linear(x, w, b, "swiglu", r, torch.float32, 7.0)
    assert y.shape == (3, 5, 6) and y.dtype == torch.float32
    grads = torch.autograd.grad(y, (x, w, b, r), torch.empty(3, 5, 6, device="meta"))
    assert [tuple(g.shape) for g in grads] == [(3, 5, 16), (12, 16), (12,), (3, 5, 6)]
    assert [g.dtype for g in grads] == [torch.half, torch.half, torch.float32, torch.half]
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(linear(x, w), x, torch.empty(3, 5, 12, device="meta", dtype=torch.half), create_graph=True)
    with FakeTensorMode():
        y = linear(torch.empty(4, 16, device="cuda", dtype=torch.half), torch.empty(9, 16, device="cuda", dtype=torch.half), activation="gelu")
        assert y.device.type == "cuda" and y.shape == (4, 9) and not y.requires_grad


@pytest.mark.parametrize("mode", ["real", "symbolic"])
def test_a_trace_holds_the_operators(linear, mode):
    def step(x, w, dy):
        x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
        y = linear(x, w, None, "silu")
        return y.detach(), *torch.autograd.grad(y, (x, w), dy)

    args = [torch.empty(*s, device="meta", dtype=torch.half) for s in ((6, 8), (5, 8), (6, 5))]
    traced = make_fx(step, tracing_mode=mode)(*args)
    names = [str(n.target) for n in traced.graph.nodes if n.op == "call_function"]
    assert "_vllm_mi355x.dense_linear_forward.default" in names and "_vllm_mi355x.dense_linear_grad.default" in names, names
    assert [tuple(t.shape) for t in traced(*args)] == [(6, 5), (6, 8), (5, 8)]


@pytest.mark.parametrize("which", range(4))
def test_forward_mode_is_refused(linear, which):
    t = [torch.empty(*s, device="meta", dtype=torch.half) for s in ((6, 8), (5, 8), (5,), (6, 5))]
    with forward_ad.dual_level():
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            linear(t[0], t[1], t[2], "silu", t[3])
        with pytest.raises(RuntimeError, match="forward-mode"):
            linear(t[0], t[1], t[2], "silu", t[3], out=torch.empty(6, 5, device="meta", dtype=torch.half))


def test_a_written_output_is_a_new_version(linear):
    x, w, out = (torch.empty(*s, device="meta", dtype=torch.half) for s in ((6, 8), (5, 8), (6, 5)))
    before = out._version
    assert linear(x, w, out=out) is out and out._version > before
    with pytest.raises(RuntimeError, match="no gradient"):
        linear(x.requires_grad_(), w, out=out)


def test_values_are_refused_by_name(linear):
    x, w = torch.empty(2, 8, device="meta", dtype=torch.half), torch.empty(4, 8, device="meta", dtype=torch.half)
    for kw in ({"activation": "tanh"}, {"clamp_limit": 7.0}, {"activation": "silu", "clamp_limit": 7.0}):
        with pytest.raises(ValueError):
            linear(x, w, **kw)
