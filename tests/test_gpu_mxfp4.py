"""MXFP4 quantization, dequantization and products on the GPU against the FP64
oracle.

Codes, scales and dequantized values are exact.  A product's FP32 sum of k
products (each exact) is off by at most (k / 32 + 8) 2^-23 of the sum of their
magnitudes: the matrix cores add 32 to 128 products at a time, an FP32 rounding
each (2^-23 allows for truncation), and 8 more join split sums; the output's
rounding adds half a step of its type.
"""

import numpy as np
import pytest
import torch

from oracle import mxfp4_oracle as M

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(scope="module")
def mx():
    from vllm_mi355x.kernels import mxfp4
    return mxfp4


def random_rows(rng, rows, k, dtype):
    """Values over many scales, zeros, exact midpoints and whole zero blocks."""
    x = rng.standard_normal((rows, k)) * np.exp2(rng.integers(-12, 8, (rows, 1)))
    x[rng.random((rows, k)) < 0.05] = 0
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 7, 4, 6])
    pick = rng.random((rows, k)) < 0.1
    x[pick] = rng.choice(ties, pick.sum()) * rng.choice([-1, 1], pick.sum())
    if rows > 1:
        x[rows // 2, : min(k, 64)] = 0
    return torch.from_numpy(x).to(TYPES[dtype])


def random_packed(rng, device, *shape, spread=3):
    """Codes and scales of every kind, as tensors and as FP64 values."""
    code = rng.integers(0, 16, shape).astype(np.uint8)
    byte = rng.integers(127 - spread, 128 + spread, (*shape[:-1], shape[-1] // 32)).astype(np.uint8)
    return (torch.from_numpy(M.pack(code)).to(device), torch.from_numpy(byte).to(device), M.values(code, byte))


def assert_product(got, a, w, dtype, k, extra=0.0):
    want = a @ w.T
    # what the FP32 sum may be off, then the output's rounding of it
    bound = (k / 32 + 8) * 2.0 ** -23 * (np.abs(a) @ np.abs(w).T)
    info = torch.finfo(dtype)
    bound = bound + info.eps / 2 * (np.abs(want) + bound) + info.smallest_normal * info.eps
    got = got.double().cpu().numpy()
    assert got.shape == want.shape
    assert np.isfinite(got).all()
    off = np.abs(got - want) - bound
    assert (off <= 0).all(), f"max excess {off.max():.3g} at {np.unravel_index(off.argmax(), off.shape)}"


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("rows,k", [(1, 32), (3, 96), (17, 4096), (130, 992), (1, 16384), (1000, 64)])
def test_quantize_matches_the_oracle(mx, device, dtype, rows, k):
    print(f"quantize {rows}x{k} {dtype}", flush=True)
    rng = np.random.default_rng(rows * 31 + k)
    x = random_rows(rng, rows, k, dtype)
    codes, scales = mx.mxfp4_quantize(x.to(device))
    code, byte = M.quantize_blocks(x.double().numpy())
    assert codes.shape == (rows, k // 2) and scales.shape == (rows, k // 32)
    assert np.array_equal(scales.cpu().numpy(), byte)
    assert np.array_equal(M.unpack(codes.cpu().numpy()), code)
    for out in TYPES.values():
        back = mx.mxfp4_dequantize(codes, scales, out)
        want = torch.from_numpy(M.values(code, byte)).to(out)
        assert torch.equal(back.cpu(), want)


@pytest.mark.parametrize("dtype", list(TYPES))
def test_quantize_ends_of_the_range(mx, device, dtype):
    info = torch.finfo(TYPES[dtype])
    rows = [[info.max] * 32, [-info.max, info.tiny] * 16, [info.smallest_normal * info.eps] * 32,
            [info.tiny * 1.5] * 32, [0.0] * 32, [-0.0] * 32, [1.0] * 31 + [float("inf")],
            [float("nan")] + [0.0] * 31, [float("-inf")] * 32, [float("nan")] * 32]
    x = torch.tensor(rows, dtype=torch.float64).to(TYPES[dtype])
    codes, scales = mx.mxfp4_quantize(x.to(device))
    code, byte = M.quantize_blocks(x.double().numpy())
    assert np.array_equal(scales.cpu().numpy(), byte)
    assert np.array_equal(M.unpack(codes.cpu().numpy()), code)
    back = mx.mxfp4_dequantize(codes, scales, torch.float32).cpu()
    assert torch.isnan(back[6:]).all() and torch.isfinite(back[:6]).all()


def test_quantize_strides_and_axes(mx, device):
    rng = np.random.default_rng(5)
    for dtype in TYPES:
        big = random_rows(rng, 40, 512, dtype).to(device)
        for view in (big[:, 8:8 + 96], big[:, 3:3 + 64], big[::3, :160], big[7:8, 1:33], big[:0, :64],
                     big.view(4, 10, 512), big.view(4, 10, 512)[:, :, 32:96], big.view(4, 1, 10, 512)):
            codes, scales = mx.mxfp4_quantize(view)
            code, byte = M.quantize_blocks(view.double().cpu().numpy())
            assert np.array_equal(scales.cpu().numpy(), byte)
            assert np.array_equal(M.unpack(codes.cpu().numpy()), code)
        vector = big[3]
        assert torch.equal(mx.mxfp4_quantize(vector)[0], mx.mxfp4_quantize(big[3:4])[0][0])


def test_refusals(mx, device):
    x = torch.zeros(8, 64, device=device, dtype=torch.bfloat16)
    codes, scales = mx.mxfp4_quantize(x)
    bad = [lambda: mx.mxfp4_quantize(x[:, :48]), lambda: mx.mxfp4_quantize(x.t()), lambda: mx.mxfp4_quantize(x.double()),
           lambda: mx.mxfp4_quantize(x[0, 0]), lambda: mx.mxfp4_quantize(x[:1].expand(4, 64)),
           lambda: mx.mxfp4_quantize(x.view(2, 4, 64)[:, :3]), lambda: mx.mxfp4_quantize(x[:, :0]),
           lambda: mx.mxfp4_dequantize(codes, scales[:, :1]), lambda: mx.mxfp4_dequantize(codes.view(torch.int8), scales),
           lambda: mx.mxfp4_dequantize(codes, scales, torch.int32), lambda: mx.mxfp4_dequantize(codes.t(), scales),
           lambda: mx.mxfp4_dequantize(codes, scales.cpu()),
           lambda: mx.mxfp4_linear(x, codes[:, :16].contiguous(), scales[:, :1].contiguous()),
           lambda: mx.mxfp4_linear(x, codes, scales, torch.float64), lambda: mx.mxfp4_linear(x, codes, scales.cpu()),
           lambda: mx.mxfp4_linear(x, codes.view(2, 4, 32), scales.view(2, 4, 2)),
           lambda: mx.mxfp4_matmul(codes, scales, codes[:, ::2], scales), lambda: mx.mxfp4_matmul(codes, scales, codes, scales, torch.int8)]
    for i, call in enumerate(bad):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was taken")
    odd = torch.zeros(8 * 32 + 8, dtype=torch.uint8, device=device)[8:].view(8, 32)
    with pytest.raises(RuntimeError, match="16-byte"):
        mx.mxfp4_linear(x, odd, scales)


SIZES = [(1, 32, 1), (1, 4096, 256), (2, 96, 33), (5, 2592, 77), (8, 1024, 1000), (16, 4128, 130), (17, 736, 515),
         (33, 256, 64), (64, 2048, 512), (100, 992, 300), (129, 512, 257), (257, 1184, 384), (300, 4096, 640), (513, 160, 1031),
         # K split over workgroups, ragged; few rows whose codes come from memory, or
         # are quantized by wide workgroups; row groups of a column group
         (70, 4096, 192), (130, 8224, 331), (16, 8192, 96), (11, 4128, 4100), (3, 2592, 12900), (40, 2080, 777)]


@pytest.mark.parametrize("rows,k,n", SIZES)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear_matches_the_oracle(mx, device, rows, k, n, dtype):
    print(f"linear {rows}x{k}x{n} {dtype}", flush=True)
    rng = np.random.default_rng(rows + k + n)
    x = random_rows(rng, rows, k, dtype)
    w, ws, wv = random_packed(rng, device, n, k)
    xq = M.quantized(x.double().numpy())
    for out in ((None, torch.float32) if dtype != "fp32" else (torch.bfloat16, None)):
        # FP16 holds the sums of values at these scales only where they stay small
        xs = x if out is not None or dtype != "fp16" else x * 2.0 ** -14
        y = mx.mxfp4_linear(xs.to(device), w, ws, out)
        assert y.dtype == (out or TYPES[dtype])
        a = xq if xs is x else M.quantized(xs.double().numpy())
        assert_product(y, a, wv, y.dtype, k)


@pytest.mark.parametrize("rows,k,n,out", [
    (1500, 288, 2200, torch.bfloat16), (1500, 320, 2205, torch.float32), (3600, 288, 3730, torch.bfloat16),
    (3585, 512, 3704, torch.float32), (3600, 544, 3704, torch.float16), (1290, 800, 2304, torch.float16),
    (3600, 4128, 3733, torch.bfloat16), (3590, 2080, 3729, torch.float32)])
def test_many_tiles(mx, device, rows, k, n, out):
    """Enough tiles of every size, ragged on each side, ends of k inside a stage."""
    print(f"tiles {rows}x{k}x{n} {out}", flush=True)
    rng = np.random.default_rng(rows + k)
    a, sa, av = random_packed(rng, device, rows, k, spread=2)
    w, ws, wv = random_packed(rng, device, n, k, spread=2)
    if out is torch.float16:
        sa, av = sa - 6, av / 64  # keeps the sums inside FP16
    assert_product(mx.mxfp4_matmul(a, sa, w, ws, out), av, wv, out, k)


@pytest.mark.parametrize("rows,k,n", SIZES)
def test_matmul_matches_the_oracle_and_the_linear(mx, device, rows, k, n):
    print(f"matmul {rows}x{k}x{n}", flush=True)
    rng = np.random.default_rng(rows * 3 + k + n)
    a, sa, av = random_packed(rng, device, rows, k, spread=5)
    w, ws, wv = random_packed(rng, device, n, k, spread=5)
    for out in TYPES.values():
        if out is torch.float16:
            continue
        assert_product(mx.mxfp4_matmul(a, sa, w, ws, out), av, wv, out, k)
    x = mx.mxfp4_dequantize(a, sa, torch.float32)
    codes, scales = mx.mxfp4_quantize(x)
    y1, y2 = mx.mxfp4_linear(x, w, ws), mx.mxfp4_matmul(codes, scales, w, ws, torch.float32)
    assert_product(y1, av, wv, torch.float32, k)
    assert_product(y2, av, wv, torch.float32, k)


def test_linear_takes_leading_axes_and_nothing(mx, device):
    rng = np.random.default_rng(9)
    w, ws, _ = random_packed(rng, device, 48, 128)
    x = random_rows(rng, 30, 256, "bf16").to(device)
    flat = mx.mxfp4_linear(x[:, :128], w, ws)
    assert torch.equal(mx.mxfp4_linear(x.view(5, 6, 256)[..., :128], w, ws), flat.view(5, 6, 48))
    assert mx.mxfp4_linear(x[:0, :128], w, ws).shape == (0, 48)
    assert mx.mxfp4_linear(x[:, :128], w[:0], ws[:0]).shape == (30, 0)
    assert torch.equal(mx.mxfp4_linear(x[4, :128], w, ws).view(1, 48), mx.mxfp4_linear(x[4:5, :128], w, ws))
    assert mx.mxfp4_matmul(*mx.mxfp4_quantize(x[:0]), *mx.mxfp4_quantize(x)).shape == (0, 30)


@pytest.mark.parametrize("rows", [1, 7, 40, 200])
def test_nan_stays_in_its_row_and_column(mx, device, rows):
    """A NaN block of x makes its output row NaN, one of w its column; all others
    keep their bits."""
    rng = np.random.default_rng(rows)
    k, n = 416, 150
    x = random_rows(rng, rows, k, "bf16").to(device)
    w, ws, _ = random_packed(rng, device, n, k)
    clean = mx.mxfp4_linear(x, w, ws, torch.float32)
    bad = x.clone()
    bad[rows // 2, k - 1] = float("inf")
    bs = ws.clone()
    bs[n - 1, k // 32 - 1] = 255
    y = mx.mxfp4_linear(bad, w, bs, torch.float32)
    assert torch.isnan(y[rows // 2]).all() and torch.isnan(y[:, n - 1]).all()
    keep = torch.ones_like(clean, dtype=torch.bool)
    keep[rows // 2] = False
    keep[:, n - 1] = False
    assert torch.equal(y[keep], clean[keep])


def test_extreme_scales(mx, device):
    """Scale bytes at both ends: products at FP32's range, sums that cancel."""
    k, n = 128, 16
    code = np.full((n, k), 2, np.uint8)  # 1.0
    byte = np.full((n, k // 32), 127, np.uint8)
    byte[0], byte[1] = 0, 250
    w, ws = torch.from_numpy(M.pack(code)).to(device), torch.from_numpy(byte).to(device)
    for scale in (0, 127, 130):
        a = np.full((3, k), 2, np.uint8)
        sa = np.full((3, k // 32), scale, np.uint8)
        y = mx.mxfp4_matmul(torch.from_numpy(M.pack(a)).to(device), torch.from_numpy(sa).to(device), w, ws, torch.float32)
        want = (M.values(a, sa) @ M.values(code, byte).T)
        got = y.double().cpu().numpy()
        over = np.abs(want) > np.finfo(np.float32).max  # the sum itself leaves FP32
        assert over.any() == (scale >= 127) and np.array_equal(np.isposinf(got), over)
        # below the normal range a result may be flushed
        assert (np.abs(got - want)[~over] <= 2.0 ** -126 + 2.0 ** -20 * np.abs(want)[~over]).all()


@pytest.mark.parametrize("rows,k,n", [(1, 4096, 512), (20, 2592, 203), (300, 1024, 500)])
def test_linear_on_a_stream_in_a_graph_and_again(mx, device, rows, k, n):
    """Equal bits eagerly, on another stream beside it, and on every replay of a
    captured graph with new inputs."""
    print(f"graph {rows}x{k}x{n}", flush=True)
    rng = np.random.default_rng(n)
    w, ws, _ = random_packed(rng, device, n, k)
    xs = [random_rows(rng, rows, k, "bf16").to(device) for _ in range(3)]
    want = [mx.mxfp4_linear(x, w, ws, torch.float32) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = mx.mxfp4_linear(xs[0], w, ws, torch.float32)
    second = mx.mxfp4_linear(xs[1], w, ws, torch.float32)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(first, want[0]) and torch.equal(second, want[1])
    static = xs[0].clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = mx.mxfp4_linear(static, w, ws, torch.float32)
        pair = mx.mxfp4_quantize(static)
    for i in (2, 1, 0, 2):
        static.copy_(xs[i])
        graph.replay()
        again = mx.mxfp4_linear(xs[i], w, ws, torch.float32)
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]) and torch.equal(again, want[i])
        assert torch.equal(pair[0], mx.mxfp4_quantize(xs[i])[0])
