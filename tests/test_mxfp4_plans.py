"""Every way in which the MXFP4 products run, against the FP64 oracle.

The kernels' plans (tile, stage buffers, K splits; column tiles, parts and fused
quantization of the few rows' kernel) follow from sizes through a fitted rule, so
the sizes here are checked on the CPU to reach all of them: a change of the rule
that leaves one out fails there.  On the GPU the outputs' rows and columns of every
tile are compared with the product of the codes' values.

Tolerance: products are exact; a sum of k of them is off by at most (k / 32 + 8) 2^-23
of the sum of their magnitudes (the matrix cores add 32 at least at a time, a rounding
of FP32 each, 2^-23 where it truncates; 8 more join parts of K), then half a step of
the output's type.
"""

import ctypes
import math
import random

import numpy as np
import pytest
import torch

from oracle import mxfp4_oracle as M

# rows, k, n: tiles of each size and number of buffers in each number of K splits, most of
# them with ragged ends on all three sides
TILES = [(72, 288, 17), (65, 256, 16), (129, 992, 301), (4856, 5536, 17), (5299, 6656, 16), (76, 3904, 17), (73, 4096, 16),
         (77, 8352, 17), (75, 8960, 16), (72, 8128, 17), (83, 8192, 16),
         (139, 288, 16587), (131, 256, 17263), (300, 4096, 14336), (1500, 2592, 5003), (8227, 10880, 135), (8461, 12800, 134),
         (8447, 10080, 65), (4177, 13376, 66), (67, 11200, 17243), (65, 10016, 8451), (68, 15296, 4135),
         (6616, 288, 130), (7435, 256, 132), (400, 14336, 4096), (401, 14368, 4099), (200, 14336, 4096), (203, 14304, 4093),
         (8053, 8512, 74), (7211, 8064, 18), (4068, 10528, 18), (66, 12544, 2828), (4002, 8032, 17), (3934, 9728, 17),
         (136, 288, 45895), (129, 256, 31116), (2048, 800, 9001), (8155, 18784, 917), (135, 18432, 30869), (140, 27584, 44890),
         (142, 50752, 23097)]
# the few rows' kernel: column tiles, parts of K, fused quantization or not, row groups
FEW = [(1, 32, 1), (17, 32, 1), (1, 544, 1), (17, 544, 33), (15, 1376, 4178), (1, 1568, 7), (17, 1568, 100), (16, 2592, 12),
       (1, 3616, 20), (17, 3616, 31), (11, 3744, 5), (1, 7712, 50), (17, 7712, 3), (5, 8224, 49), (16, 8192, 200),
       (1, 32, 6388), (17, 32, 6447), (1, 544, 6410), (17, 544, 6447), (15, 1376, 8754), (1, 1568, 6398), (17, 1632, 6515),
       (13, 1600, 8457), (1, 3616, 6486), (6, 3616, 8307), (18, 3744, 6495), (16, 4096, 6400),
       (1, 32, 12789), (17, 32, 12809), (12, 864, 56079), (1, 544, 12918), (17, 608, 12862), (15, 1504, 16548), (1, 1568, 13032),
       (11, 1888, 16986), (19, 1568, 12797), (1, 4096, 14336)]
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def plan():
    from vllm_mi355x import _native
    lib = _native.load()
    out = (ctypes.c_int32 * 6)()

    def of(rows, k, n):
        assert lib.mxfp4_matmul_plan(rows, k, n, out) == 0
        return tuple(out)
    return of


def test_the_sizes_here_reach_every_plan(plan):
    """Over random sizes, and those whose stages of K do not split evenly."""
    tiles, few = {plan(*s)[:3] for s in TILES}, {plan(*s)[3:] for s in FEW}
    assert all(plan(*s)[0] for s in TILES) and not any(plan(*s)[0] for s in FEW)
    rng = random.Random(0)

    def log_int(lo, hi):
        return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))

    for i in range(200000):
        rows, n = log_int(1, 16384), log_int(1, 131072)
        k = 32 * (log_int(1, 2048) if i % 2 else rng.randint(257, 288))
        if rows * k * n > 1e15:
            continue
        p = plan(rows, k, n)
        assert p[:3] in tiles if p[0] else p[3:] in few, (rows, k, n, p)


def test_plan_refusals(plan):
    from vllm_mi355x import _native
    lib = _native.load()
    out = (ctypes.c_int32 * 6)()
    assert lib.mxfp4_matmul_plan(4, 33, 5, out) == 1 and lib.mxfp4_matmul_plan(-1, 32, 5, out) == 1
    assert lib.mxfp4_matmul_plan(4, 32, 5, None) == 1


def codes(device, seed, *shape):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randint(0, 256, (*shape[:-1], shape[-1] // 2), dtype=torch.uint8, device=device, generator=g),
            torch.randint(121, 126, (*shape[:-1], shape[-1] // 32), dtype=torch.uint8, device=device, generator=g))


def some(size, most):
    """Places of every 64 on, the ends in full."""
    spread = np.linspace(0, size - 1, min(size, max(most, size // 32))).astype(int)
    return np.unique(np.concatenate([spread, np.arange(min(size, 40)), np.arange(max(0, size - 40), size)]))


def compare(y, a, sa, w, ws, k):
    rows, cols = some(y.shape[0], 70), some(y.shape[1], 70)
    value = lambda c, s, at: M.values(M.unpack(c[at].cpu().numpy()), s[at].cpu().numpy())
    va, vw = value(a, sa, rows), value(w, ws, cols)
    want = va @ vw.T
    bound = (k / 32 + 8) * 2.0 ** -23 * (np.abs(va) @ np.abs(vw).T)
    info = torch.finfo(y.dtype)
    bound = bound + info.eps / 2 * (np.abs(want) + bound) + info.smallest_normal * info.eps
    got = y[torch.from_numpy(rows).to(y.device)][:, torch.from_numpy(cols).to(y.device)].double().cpu().numpy()
    off = np.abs(got - want) - bound
    assert np.isfinite(got).all() and (off <= 0).all(), f"max excess {off.max():.3g} at {np.unravel_index(off.argmax(), off.shape)}"


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", TILES + FEW)
def test_products_of_every_plan(plan, device, rows, k, n):
    from vllm_mi355x.kernels import mxfp4
    print(f"plan {rows}x{k}x{n} {plan(rows, k, n)}", flush=True)
    a, sa = codes(device, rows, rows, k)
    w, ws = codes(device, n + 1, n, k)
    for out in TYPES if rows * n < 1 << 22 else TYPES[:2]:
        compare(mxfp4.mxfp4_matmul(a, sa, w, ws, out), a, sa, w, ws, k)
    # (values that the format holds: quantizing them changes the codes at most, not the values)
    x = mxfp4.mxfp4_dequantize(a, sa, torch.bfloat16)
    compare(mxfp4.mxfp4_linear(x, w, ws, torch.float32), a, sa, w, ws, k)
