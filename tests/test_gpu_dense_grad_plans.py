"""The dense layer's gradients on every kernel and number of K splits that their two products choose
from, in BF16 and in FP16, whose power of two is taken out again in each of the kernels' ends.
Tolerances as in test_gpu_dense.py."""

import numpy as np
import pytest
import torch

from oracle import dense_oracle as D
from tests.test_gpu_dense import TYPES, close, exact, linear, normal  # noqa: F401

pytestmark = pytest.mark.gpu

# rows, k, lines, activation: (test_dense_grad_cpu.py holds that dx and dW reach all plans)
SIZES = [(34, 34, 32, "gelu"), (135, 33, 34, "swiglu"), (36, 32, 138, "swiglu"), (3905, 33, 35, "relu"), (33, 34, 3821, None),
         (34, 9105, 513, "gelu_tanh"), (1733, 2899, 36, "swiglu"), (10227, 1047, 1406, "swiglu"), (11086, 66, 8904, "silu"), (520, 4377, 459, "silu"),
         (714, 2898, 516, None), (6680, 1349, 482, "gelu"), (462, 1388, 6982, "swiglu"), (130, 8477, 730, "relu"), (747, 8337, 129, None),
         (6493, 2247, 935, "gelu"), (597, 2219, 9270, "swiglu"), (338, 7581, 1563, "silu"), (1963, 6209, 321, None), (8140, 2745, 1462, "swiglu"),
         (1421, 2749, 8063, "gelu_tanh"), (5, 200, 33, "silu"), (200, 2048, 6, "swiglu")]


@pytest.mark.parametrize("rows,k,lines,activation", SIZES)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_every_plan(linear, device, rows, k, lines, activation, dtype):
    """Some rows of dx and some lines of dW and db against 64 bits, equal bits from call to call, and of y
    (written beside z)."""
    print(f"dense gradient {rows}x{k}x{lines} {dtype} {activation}", flush=True)
    rng = np.random.default_rng(rows + k + lines)
    g = torch.Generator(device=device).manual_seed(rows + k + lines)
    n = lines // 2 if activation == "swiglu" else lines
    x = torch.randn(rows, k, device=device, generator=g).to(TYPES[dtype])
    w = (torch.randn(lines, k, device=device, generator=g) * k ** -0.5).to(TYPES[dtype])
    bias = normal(rng, lines, "fp32", device)
    dy = torch.randn(rows, n, device=device, generator=g).to(TYPES[dtype])
    leaves = [t.requires_grad_() for t in (x, w, bias)]
    y = linear(x, w, bias, activation)
    dx, dw, db = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, dy)
    assert all(torch.equal(a, b) for a, b in zip((dx, dw, db), again))
    eps = torch.finfo(x.dtype).eps
    # (FP16's bound is of dz's largest magnitude: those of the rows and lines here are above a
    # quarter of the whole's, which the bound's factor of four covers)
    some = sorted({i for i in (0, 1, rows // 2, rows // 3, 127, 128, 255, 256, rows - 2, rows - 1) if i < rows})
    want, tol = D.forward(exact(x[some]), exact(w), exact(bias), activation, None)
    close(y[some], want, tol, "y")
    wants, _ = D.backward(exact(x[some]), exact(w), exact(bias), activation, exact(dy[some]), eps)
    close(dx[some], *wants["x"], "dx")
    at = sorted({i for i in (0, 1, n // 2, n // 3, 63, 64, 255, 256, n - 2, n - 1) if 0 <= i < n})
    of = at + [n + i for i in at] if activation == "swiglu" else at
    wants, _ = D.backward(exact(x), exact(w[of]), exact(bias[of]), activation, exact(dy[:, at]), eps)
    close(dw[of], *wants["w"], "dW")
    close(db[of], *wants["bias"], "db")
