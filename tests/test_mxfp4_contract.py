"""The MXFP4 and router-load operators on the CPU: what the C-ABI and the torch
operators refuse, their size functions, and shapes under tracing."""

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from vllm_mi355x import _native
    return _native.load()


def _err(lib):
    return lib.vllm_mi355x_last_error().decode()


P = 1 << 20  # an address that no check follows


@pytest.mark.parametrize("args,word", [
    ((P, 3, 1, 32, 32, 2 * P, 3 * P, 0), "BF16"),
    ((P, 0, 1, 33, 33, 2 * P, 3 * P, 0), "multiple of 32"),
    ((P, 0, 1, 0, 0, 2 * P, 3 * P, 0), "multiple of 32"),
    ((P, 0, -1, 32, 32, 2 * P, 3 * P, 0), "multiple of 32"),
    ((P, 0, 2, 64, 32, 2 * P, 3 * P, 0), "stride"),
    ((0, 0, 2, 64, 64, 2 * P, 3 * P, 0), "null"),
    ((P + 1, 0, 2, 64, 64, 2 * P, 3 * P, 0), "aligned"),
    ((P, 0, 2, 64, 64, 2 * P + 4, 3 * P, 0), "16-byte"),
    ((P, 0, 2, 64, 64, P, 3 * P, 0), "overlap"),
    ((P, 0, 2, 64, 64, 2 * P, 2 * P + 8, 0), "overlap"),
    ((P, 0, 1 << 40, 1 << 30, 1 << 30, 2 * P, 3 * P, 0), "range"),
])
def test_quantize_refusals(lib, args, word):
    assert lib.mxfp4_quantize(*args) == 1 and word in _err(lib)


@pytest.mark.parametrize("args,word", [
    ((P, 2 * P, 1, 32, 3 * P, 7, 0), "BF16"), ((P, 2 * P, 1, 31, 3 * P, 0, 0), "multiple of 32"),
    ((P + 2, 2 * P, 1, 32, 3 * P, 0, 0), "16-byte"), ((P, 2 * P, 1, 32, 3 * P + 1, 0, 0), "aligned"),
    ((P, 2 * P, 1, 32, P, 0, 0), "overlap"), ((P, 0, 1, 32, 3 * P, 0, 0), "null"),
])
def test_dequantize_refusals(lib, args, word):
    assert lib.mxfp4_dequantize(*args) == 1 and word in _err(lib)


def _matmul(a=P, sa=2 * P, rows=2, k=64, w=3 * P, sw=4 * P, n=5, out=5 * P, dt=0, ws=6 * P, wb=1 << 20):
    return (a, sa, rows, k, w, sw, n, out, dt, ws, wb, 0)


@pytest.mark.parametrize("change,word", [
    ({"k": 48}, "multiple of 32"), ({"rows": -1}, "multiple of 32"), ({"dt": 9}, "BF16"),
    ({"w": 0}, "null"), ({"a": 0}, "null"), ({"w": 3 * P + 8}, "16-byte"), ({"a": P + 4}, "16-byte"),
    ({"out": 5 * P + 1}, "aligned"), ({"out": P}, "overlap"), ({"out": 3 * P}, "overlap"),
    ({"rows": 1 << 40, "k": 1 << 30}, "range")])
def test_matmul_refusals(lib, change, word):
    assert lib.mxfp4_matmul(*_matmul(**change)) == 1 and word in _err(lib)


def test_linear_refusals(lib):
    need = lib.mxfp4_linear_workspace_size(300, 4096, 512)
    assert need > 0
    call = lambda ws, nb, out=5 * P, stride=4096: lib.mxfp4_linear(
        1 << 40, 0, 300, 4096, stride, 1 << 41, 1 << 42, 512, out, 0, ws, nb, 0)
    assert call(1 << 43, need - 1) == 1 and "workspace" in _err(lib)
    assert call(0, need) == 1 and "workspace" in _err(lib)
    assert call((1 << 43) + 4, need) == 1 and "workspace" in _err(lib)
    assert call(1 << 41, need) == 1 and "overlap" in _err(lib)
    assert call(1 << 43, need, out=1 << 40) == 1 and "overlap" in _err(lib)
    assert call(1 << 43, need, stride=100) == 1 and "stride" in _err(lib)
    assert lib.mxfp4_linear_workspace_size(1, 40, 4) == -1
    assert lib.mxfp4_matmul_workspace_size(-1, 32, 4) == -1


def _moe(x=1 << 40, dt=0, tokens=2, stride=64, w13=1 << 41, s13=1 << 42, w2=1 << 43, s2=1 << 44, experts=4,
         ids=1 << 45, tw=1 << 46, topk=2, emap=0, mapn=0, hidden=64, inter=32, limit=float("inf"), out=1 << 47,
         ws=1 << 48, wb=1 << 30):
    return (x, dt, tokens, stride, w13, s13, w2, s2, experts, ids, tw, topk, emap, mapn, hidden, inter, limit, out,
            ws, wb, 0)


@pytest.mark.parametrize("change,word", [
    ({"dt": 2}, "bf16"), ({"hidden": 48}, "multiples of 32"), ({"inter": 0}, "multiples of 32"),
    ({"experts": 1025}, "1024"), ({"topk": 0}, "range"), ({"tokens": 1 << 31}, "range"),
    ({"stride": 32}, "stride"), ({"limit": float("nan")}, "limit"), ({"limit": 0.0}, "limit"),
    ({"w2": 0}, "null"), ({"mapn": 4}, "null"), ({"w13": (1 << 41) + 8}, "16-byte"), ({"x": (1 << 40) + 1}, "aligned"),
    ({"wb": 64}, "workspace"), ({"ws": (1 << 48) + 4}, "workspace"), ({"hidden": 65568}, "65536"),
    ({"inter": 1 << 17}, "65536"), ({"ws": 1 << 41}, "overlap"), ({"ws": 1 << 47}, "overlap"), ({"ws": 1 << 40}, "overlap"),
    ({"out": 1 << 43}, "overlap"), ({"out": 1 << 45}, "overlap"), ({"out": 1 << 42}, "overlap")])
def test_moe_refusals(lib, change, word):
    assert lib.mxfp4_moe(*_moe(**change)) == 1 and word in _err(lib)


def test_balance_refusals(lib):
    size = lib.moe_balance_workspace_size(100, 16)
    assert size > 0 and lib.moe_balance_workspace_size(-1, 16) == -1
    assert lib.moe_balance_workspace_size(1, 1025) == -1
    loss = lambda rows=100, e=16, stride=16, k=2, scoring=0, dt=2, ws=P, nb=size, logits=P: lib.moe_balance_loss(
        logits, dt, rows, e, stride, 2 * P, k, 0, scoring, 3 * P, 4 * P, 5 * P, ws, nb, 0)
    for change, word in (({"e": 0}, "experts"), ({"k": 0}, "top_k"), ({"stride": 15}, "stride"), ({"scoring": 2}, "scoring"),
                         ({"dt": 5}, "BF16"), ({"nb": size - 1}, "workspace"), ({"ws": P + 4}, "workspace"),
                         ({"logits": 0}, "null"), ({"rows": 1 << 31}, "rows")):
        assert loss(**change) == 1 and word in _err(lib), change
    assert lib.moe_expert_counts(P, 0, 10, 2, 8, 0, 0, P, 1 << 20, 0) == 1 and "null" in _err(lib)
    assert lib.moe_balance_grad(P, 2, 4, 8, 8, 0, 0, 0, P, P, 0) == 1 and "null" in _err(lib)


def test_cpu_tensors_are_refused():
    from vllm_mi355x.kernels import moe, mxfp4
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    for call in (lambda: mxfp4.mxfp4_quantize(torch.zeros(2, 64)),
                 lambda: mxfp4.mxfp4_dequantize(codes, scales),
                 lambda: mxfp4.mxfp4_linear(torch.zeros(2, 64), codes, scales),
                 lambda: mxfp4.mxfp4_matmul(codes, scales, codes, scales),
                 lambda: moe.moe_balance_loss(torch.zeros(2, 4), torch.zeros(2, 1, dtype=torch.int32)),
                 lambda: moe.moe_expert_counts(torch.zeros(2, 1, dtype=torch.int32), 4)):
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(ValueError):
        moe.moe_balance_loss(torch.zeros(2, 4), torch.zeros(2, 1, dtype=torch.int32), scoring="other")


def test_shapes_under_tracing():
    from vllm_mi355x.kernels import moe, mxfp4
    x = torch.empty(3, 5, 64, dtype=torch.bfloat16, device="meta")
    codes, scales = mxfp4.mxfp4_quantize(x)
    assert codes.shape == (3, 5, 32) and scales.shape == (3, 5, 2) and codes.dtype == torch.uint8
    assert mxfp4.mxfp4_dequantize(codes, scales, torch.float16).shape == (3, 5, 64)
    w, ws = torch.empty(7, 32, dtype=torch.uint8, device="meta"), torch.empty(7, 2, dtype=torch.uint8, device="meta")
    y = mxfp4.mxfp4_linear(x, w, ws)
    assert y.shape == (3, 5, 7) and y.dtype == torch.bfloat16
    assert mxfp4.mxfp4_matmul(codes, scales, w, ws, torch.float32).dtype == torch.float32
    loss, counts = moe.moe_balance_loss(torch.empty(9, 4, device="meta"), torch.empty(9, 2, dtype=torch.int32, device="meta"))
    assert loss.shape == () and counts.shape == (4,) and counts.dtype == torch.int64
