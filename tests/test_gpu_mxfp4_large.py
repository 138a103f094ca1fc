"""Offsets past 32 bits: quantization, products, the fused MoE and the balance
loss on tensors of more than 2^31 elements or bytes, whose far ends have to
equal the same calls on small copies of these ends."""

import numpy as np
import pytest
import torch

from oracle import balance_oracle as B

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mx():
    from vllm_mi355x.kernels import mxfp4
    yield mxfp4
    torch.cuda.empty_cache()


def codes(device, *shape, seed=0):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randint(0, 256, (*shape[:-1], shape[-1] // 2), dtype=torch.uint8, device=device, generator=g),
            torch.randint(124, 129, (*shape[:-1], shape[-1] // 32), dtype=torch.uint8, device=device, generator=g))


def test_quantize_and_dequantize(mx, device):
    print("quantize 70000x32768", flush=True)
    x = torch.randn(70000, 32768, dtype=torch.bfloat16, device=device)
    c, s = mx.mxfp4_quantize(x)
    for rows in (slice(0, 3), slice(65534, 65540), slice(69990, 70000)):
        cs, ss = mx.mxfp4_quantize(x[rows].clone())
        assert torch.equal(c[rows], cs) and torch.equal(s[rows], ss)
    del x
    y = mx.mxfp4_dequantize(c, s, torch.float16)
    for rows in (slice(0, 3), slice(65534, 65540), slice(69990, 70000)):
        assert torch.equal(y[rows], mx.mxfp4_dequantize(c[rows].clone(), s[rows].clone(), torch.float16))


def test_rows_far_apart(mx, device):
    """A row stride whose last rows lie past 2^31 elements."""
    base = torch.randn(3, 1 << 30, dtype=torch.bfloat16, device=device)
    x = base[:, 77:77 + 512]
    w, ws = codes(device, 96, 512)
    assert torch.equal(mx.mxfp4_linear(x, w, ws), mx.mxfp4_linear(x.contiguous(), w, ws))
    assert torch.equal(mx.mxfp4_quantize(x)[0], mx.mxfp4_quantize(x.contiguous())[0])


@pytest.mark.parametrize("rows", [1, 16, 40, 300])
def test_weights(mx, device, rows):
    """140000 columns of 32768 (2.3 GB of codes): the last ones, as a product of
    their own.  Sums of the same products in another order: off by at most (k /
    32 + 8) 2^-23 of the sum of magnitudes each (at most 6 * 6 * 2 * 2 * k), then
    half a step of the output."""
    print(f"linear {rows}x32768x140000", flush=True)
    k = 32768
    w, ws = codes(device, 140000, k, seed=1)
    x = torch.randn(rows, k, dtype=torch.bfloat16, device=device)
    y = mx.mxfp4_linear(x, w, ws, torch.float32)
    xq = mx.mxfp4_dequantize(*mx.mxfp4_quantize(x), torch.float32).double()
    for cols in (slice(0, 40), slice(131060, 131090), slice(139900, 140000)):
        v = mx.mxfp4_dequantize(w[cols].clone(), ws[cols].clone(), torch.float32).double()
        want, size = (xq[:, None] * v[None]).sum(-1), (xq[:, None] * v[None]).abs().sum(-1)
        bound = (k / 32 + 8) * 2.0 ** -23 * size
        assert ((y[:, cols].double() - want).abs() <= bound + 2.0 ** -24 * (want.abs() + bound)).all()


def test_outputs(mx, device):
    """20000 x 140000 outputs (2.8e9): the last rows and columns equal a product of
    theirs (one stage of k, the same order of sums)."""
    print("matmul 20000x256x140000", flush=True)
    a, sa = codes(device, 20000, 256, seed=2)
    w, ws = codes(device, 140000, 256, seed=3)
    y = mx.mxfp4_matmul(a, sa, w, ws)
    for rows in (slice(0, 300), slice(15300, 15600), slice(19700, 20000)):
        z = mx.mxfp4_matmul(a[rows].clone(), sa[rows].clone(), w[-1000:].clone(), ws[-1000:].clone())
        assert torch.equal(y[rows, -1000:], z)


@pytest.mark.parametrize("tokens", [2, 20, 600])
def test_experts(mx, device, tokens):
    """64 experts of 8192 x 8192 (6.4 GB of codes), tokens on the last four: as in a
    layer of these four."""
    print(f"moe {tokens} on the last of 64 experts of 8192 x 8192", flush=True)
    w1, s1 = codes(device, 64, 16384, 8192, seed=4)
    w2, s2 = codes(device, 64, 8192, 8192, seed=5)
    s1, s2 = s1 - 6, s2 - 6  # keeps the sums inside the type
    x = torch.randn(tokens, 8192, dtype=torch.bfloat16, device=device)
    ids = torch.randint(0, 4, (tokens, 1), dtype=torch.int32, device=device)
    tw = torch.ones(tokens, 1, device=device)
    y = mx.fused_mxfp4_moe(x, w1, w2, s1, s2, tw, ids + 60)
    z = mx.fused_mxfp4_moe(x, *(t[60:].clone() for t in (w1, w2, s1, s2)), tw, ids)
    assert torch.isfinite(y).all() and y.abs().max() > 0
    assert torch.equal(y, z)


def test_balance(device):
    """2.2 million rows of 1024: the loss's counts, and the last rows' gradient from
    the formula."""
    from vllm_mi355x.kernels.moe import moe_balance_loss
    print("balance 2200000x1024", flush=True)
    rows, experts = 2_200_000, 1024
    logits = torch.randn(rows, experts, dtype=torch.bfloat16, device=device).requires_grad_()
    ids = torch.randint(0, experts, (rows, 2), dtype=torch.int32, device=device)
    loss, counts = moe_balance_loss(logits, ids)
    assert torch.equal(counts, torch.bincount(ids.flatten().long(), minlength=experts))
    grad, = torch.autograd.grad(loss * rows, logits)
    f = counts.double().cpu().numpy() * experts / (rows * 2)
    for at in (0, 2_097_150, rows - 20):
        p, _ = B.probabilities(logits[at:at + 20].detach().double().cpu().numpy(), False)
        r = p @ f
        want = p * (f - r[:, None])
        tol = 2.0 ** -18 * p * (f + r[:, None])
        tol = tol + 2.0 ** -8 * (np.abs(want) + tol) + 2.0 ** -133
        assert (np.abs(grad[at:at + 20].double().cpu().numpy() - want) <= tol).all()
