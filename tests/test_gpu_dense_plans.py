"""The dense layer on every kernel that its sizes choose from, with and without K splits, and past
32-bit offsets.  Tolerances as in test_gpu_dense.py."""

import pytest
import torch

from tests.test_gpu_dense import TYPES, check, close, exact, linear, normal  # noqa: F401
from oracle import dense_oracle as D

pytestmark = pytest.mark.gpu

# rows, k, n, gated: (test_dense_cpu.py holds that they reach all plans)
SIZES = [(1, 4096, 300, False), (2, 8200, 65, False), (3, 520, 8200, False), (7, 1024, 40, True), (8, 100, 9000, True), (1, 300, 5000, False),
         (9, 2056, 100, False), (16, 520, 70, True), (12, 4100, 33, True), (40, 4096, 200, False), (40, 192, 700, False), (60, 4096, 100, True),
         (60, 200, 500, True), (700, 1024, 1100, False), (64, 14336, 4096, False), (1000, 2048, 4096, False), (190, 14336, 4100, False),
         (2040, 256, 4096, False), (700, 1024, 600, True), (64, 14336, 2050, True), (1000, 2048, 2050, True), (190, 14336, 2050, True),
         (2040, 256, 2050, True), (2048, 512, 6000, False), (2048, 512, 3000, True), (700, 4096, 4096, False), (700, 4096, 2048, True),
         (4096, 192, 4100, False), (4096, 192, 2049, True), (300, 8192, 8192, False), (300, 8192, 4096, True), (100, 4096, 14336, False),
         (100, 4096, 7168, True), (600, 14336, 4096, False), (600, 14336, 2048, True), (1500, 8192, 3000, False), (1500, 8192, 1500, True), (500, 4096, 1500, False),
         (500, 4096, 750, True), (700, 8192, 750, True), (500, 8192, 1500, False), (2500, 192, 1250, True), (3000, 4096, 3000, False),
         (3000, 4096, 1500, True), (40, 64, 100, False), (6, 4096, 9000, False), (12, 8192, 2100, True), (16, 5000, 300, False),
         (3, 8192, 4200, False), (9, 8192, 5000, False)]


@pytest.mark.parametrize("rows,k,n,gated", SIZES)
def test_every_plan(linear, device, rows, k, n, gated):
    """All outputs of few rows and columns; of large calls the first, last and some rows between,
    against the same rows of a 64-bit product."""
    import numpy as np
    print(f"dense plan {rows}x{k}x{n} gated={gated}", flush=True)
    rng = np.random.default_rng(rows + k)
    g = torch.Generator(device=device).manual_seed(rows + k)
    lines = 2 * n if gated else n
    for dtype in ("bf16", "fp16"):
        x = torch.randn(rows, k, device=device, generator=g).to(TYPES[dtype])
        w = (torch.randn(lines, k, device=device, generator=g) * k ** -0.5).to(TYPES[dtype])
        bias, residual = normal(rng, lines, dtype, device), normal(rng, (rows, n), dtype, device)
        act = "swiglu" if gated else "gelu"
        y = linear(x, w, bias, act, residual)
        again = linear(x, w, bias, act, residual)
        assert torch.equal(y, again)
        some = sorted({0, rows - 1, rows // 2, rows // 3, min(rows - 1, 128), min(rows - 1, 255)})
        want, tol = D.forward(exact(x[some]), exact(w), exact(bias), act, exact(residual[some]))
        close(y[some], want, tol, "rows")


def test_weights_and_outputs_past_32_bits(linear, device):
    """Weights of over 2^32 elements through every kernel, and an output of as many."""
    lines, k = 70000, 65536
    w = torch.empty(lines, k, dtype=torch.bfloat16, device=device).normal_(generator=torch.Generator(device=device).manual_seed(3))
    some = [0, 1, 32767, 65535, 65536, lines - 1]
    for rows in (2, 12, 40):
        x = torch.randn(rows, k, device=device, generator=torch.Generator(device=device).manual_seed(rows)).bfloat16()
        y = linear(x, w, out_dtype=torch.float32)
        want, tol = D.forward(exact(x), exact(w[some]), None, None, None)
        close(y[:, some], want, tol, f"{rows} rows")
        if rows == 12:  # off 16 bytes
            y = linear(x[:, 1:], w[:, 1:], out_dtype=torch.float32)
            want, tol = D.forward(exact(x[:, 1:]), exact(w[some, 1:]), None, None, None)
            close(y[:, some], want, tol, f"{rows} rows off 16 bytes")
    del w
    x = torch.randn(66000, 8, device=device, generator=torch.Generator(device=device).manual_seed(5)).half()
    w = torch.randn(66000, 8, device=device, generator=torch.Generator(device=device).manual_seed(6)).half()
    y = linear(x, w)
    some = torch.tensor([0, 31, 65534, 65999], device=device)
    want, tol = D.forward(exact(x[some]), exact(w), None, None, None)
    close(y[some], want, tol, "rows")
