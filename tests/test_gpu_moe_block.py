"""A mixture-of-experts block as a model runs it: the router's dense layer, the choice from its
logits, the balance loss, the routed experts and the shared expert with their sum as its
residual.  Each step is held to its FP64 oracle at the inputs that the step itself had, with
the tolerances of the steps' own tests; gradients likewise, at the upstream gradients that
arrived."""

import numpy as np
import pytest
import torch

from oracle import balance_oracle as B
from oracle import dense_oracle as D
from oracle import mxfp4_oracle as X
from oracle import route_logits_oracle as L
from tests.test_gpu_dense import close, exact, normal

pytestmark = pytest.mark.gpu

E, K, N, TOPK, GROUPS = 16, 256, 128, 4, 4


def packed(rng, device, *shape):
    code = rng.integers(0, 16, shape).astype(np.uint8)
    byte = rng.integers(119, 123, (*shape[:-1], shape[-1] // 32)).astype(np.uint8)
    return torch.from_numpy(X.pack(code)).to(device), torch.from_numpy(byte).to(device), X.values(code, byte)


@pytest.mark.parametrize("rows,padded", [(1, 0), (7, 2), (40, 9), (300, 60)])
def test_a_serving_block(device, rows, padded):
    """The last `padded` rows are a batch's padding: no experts, so the shared expert alone."""
    from vllm_mi355x.kernels import mxfp4
    from vllm_mi355x.kernels.dense import dense_linear
    from vllm_mi355x.kernels.moe import moe_route_logits

    rng = np.random.default_rng(rows)
    x = normal(rng, (rows, K), "bf16", device)
    router, bias = normal(rng, (E, K), "bf16", device, K ** -0.5), rng.normal(0, 0.1, E).astype(np.float32)
    (w13, s13, v13), (w2, s2, v2) = packed(rng, device, E, 2 * N, K), packed(rng, device, E, K, N)
    up, down = normal(rng, (2 * N, K), "bf16", device, K ** -0.5), normal(rng, (K, N), "bf16", device, N ** -0.5)
    padding = np.arange(rows) >= rows - padded
    mask = torch.from_numpy(padding).to(device)
    correction = torch.from_numpy(bias).to(device)

    def block(x):
        logits = dense_linear(x, router, out_dtype=torch.float32)
        weights, ids = moe_route_logits(logits, TOPK, correction, GROUPS, 2, True, 2.5, mask)
        routed = mxfp4.fused_mxfp4_moe(x, w13, w2, s13, s2, weights, ids)
        hidden = dense_linear(x, up, activation="swiglu", clamp_limit=7.0)
        return logits, weights, ids, routed, hidden, dense_linear(hidden, down, residual=routed)

    got = block(x)
    logits, weights, ids, routed, hidden, y = got
    close(logits, *D.forward(exact(x), exact(router), None, None, None), "logits")
    want_ids, want_weights = L.route(exact(logits), TOPK, True, bias, GROUPS, 2, True, 2.5, padding)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    assert (np.abs(exact(weights) - want_weights) <= 2.0 ** -18 * want_weights).all()
    assert (want_ids[padding] == -1).all() and not exact(routed)[padding].any()
    want, tol = X.moe(exact(x), ids.cpu().numpy(), weights.cpu().numpy(), v13, v2)
    close(routed, want, tol, "routed experts")
    close(hidden, *D.forward(exact(x), exact(up), None, "swiglu", None, 7.0), "shared expert's hidden rows")
    close(y, *D.forward(exact(hidden), exact(down), None, None, exact(routed)), "y")

    # captured: one graph of the whole block, replayed on new rows beside eager calls
    static, graph = x.clone(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        outs = block(static)
    for i in range(4):
        fresh = x if i == 2 else normal(rng, (rows, K), "bf16", device)
        static.copy_(fresh)
        graph.replay()
        eager = block(fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, eager)), i


@pytest.mark.parametrize("rows", [1, 50, 400])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
def test_a_training_block(device, rows, scoring):
    """The loss's gradients through the weighted sum, the choice, the balance loss and the router to
    the rows; the experts are a dense layer each, on all rows."""
    from vllm_mi355x.kernels.dense import dense_linear
    from vllm_mi355x.kernels.moe import moe_balance_loss, moe_route_logits

    rng = np.random.default_rng(rows)
    x = normal(rng, (rows, 96), "bf16", device).requires_grad_()
    router = normal(rng, (8, 96), "bf16", device, 0.1).requires_grad_()
    experts = [normal(rng, (64, 96), "bf16", device, 0.1).requires_grad_() for _ in range(8)]
    target = normal(rng, (rows, 32), "fp32", device)
    xs = [x.detach().requires_grad_() for _ in range(9)]  # a leaf a use: their gradients by themselves
    logits = dense_linear(xs[8], router, out_dtype=torch.float32)
    weights, ids = moe_route_logits(logits, 2, scoring=scoring, routed_scaling_factor=1.5)
    outs = [dense_linear(xs[e], experts[e], activation="swiglu", out_dtype=torch.float32) for e in range(8)]
    y = (torch.stack(outs, 1).gather(1, ids.long()[..., None].expand(-1, -1, 32)) * weights[..., None]).sum(1)
    balance, counts = moe_balance_loss(logits, ids, scoring=scoring)
    mse = ((y - target) ** 2).mean()
    (mse + 0.01 * balance).backward(retain_graph=True, inputs=[*xs, router, *experts])
    parts = torch.autograd.grad(mse, [weights, *outs], retain_graph=True)
    by_route, = torch.autograd.grad(weights, logits, parts[0], retain_graph=True)
    by_balance, = torch.autograd.grad(balance, logits, torch.tensor(0.01, device=device), retain_graph=True)

    l, w = exact(logits), exact(weights)
    want_ids, want = L.route(l, 2, scoring == "sigmoid", scale=1.5)
    assert np.array_equal(ids.cpu().numpy(), want_ids) and (np.abs(w - want) <= 2.0 ** -18 * want).all()
    up = exact(parts[0])
    for t in range(rows):
        g = L.gradient(l[t], want_ids[t], want[t], up[t], scoring == "sigmoid", True, 1.5)
        # 2^-18 and the weights' errors, 2^-18, of terms of twice the sum at most
        assert (np.abs(exact(by_route[t]) - g) <= 2.0 ** -16 * np.abs(want[t] * up[t]).sum()).all()
    loss, c, g = B.loss_and_grad(l, want_ids, scoring == "sigmoid")
    assert np.array_equal(counts.cpu().numpy(), c) and abs(balance.item() - loss) <= 2.0 ** -17 * loss
    assert np.abs(exact(by_balance) - 0.01 * g).max() <= 2.0 ** -16 * 0.01 * np.abs(g).max()
    # the router's own gradients from the two's sum, the experts' from theirs
    eps = torch.finfo(torch.bfloat16).eps
    wants, _ = D.backward(exact(x), exact(router), None, None, exact(by_route + by_balance), eps)
    close(xs[8].grad, *wants["x"], "x through the router")
    close(router.grad, *wants["w"], "router")
    for e in range(8):
        wants, _ = D.backward(exact(x), exact(experts[e]), None, "swiglu", exact(parts[1 + e]), eps)
        close(xs[e].grad, *wants["x"], f"x through expert {e}")
        close(experts[e].grad, *wants["w"], f"expert {e}")
