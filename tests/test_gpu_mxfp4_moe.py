"""The fused MoE in MXFP4 on the GPU against the FP64 oracle, whose tolerance
follows FP32 sums through the intermediate's quantization
(oracle/mxfp4_oracle.py), plus the output's rounding."""

import math

import numpy as np
import pytest
import torch

from oracle import mxfp4_oracle as M

pytestmark = pytest.mark.gpu

TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


@pytest.fixture(scope="module")
def mx():
    from vllm_mi355x.kernels import mxfp4
    return mxfp4


class Layer:
    def __init__(self, rng, experts, hidden, inter, device):
        self.experts, self.hidden, self.inter = experts, hidden, inter

        def packed(*shape):
            code = rng.integers(0, 16, shape).astype(np.uint8)
            byte = rng.integers(119, 123, (*shape[:-1], shape[-1] // 32)).astype(np.uint8)
            return (torch.from_numpy(M.pack(code)).to(device), torch.from_numpy(byte).to(device), M.values(code, byte))

        self.w13, self.s13, self.v13 = packed(experts, 2 * inter, hidden)
        self.w2, self.s2, self.v2 = packed(experts, hidden, inter)

    def run(self, mx, x, weights, ids, **kw):
        return mx.fused_mxfp4_moe(x, self.w13, self.w2, self.s13, self.s2, weights, ids, **kw)


def routing(rng, tokens, experts, topk):
    ids = np.stack([rng.permutation(experts)[:topk] for _ in range(tokens)]) if tokens else np.zeros((0, topk))
    weights = rng.random((tokens, topk)) + 0.1
    return ids.astype(np.int32), (weights / weights.sum(1, keepdims=True)).astype(np.float32)


def check(layer, got, x, ids, weights, dtype, limit=math.inf):
    want, tol = M.moe(x.double().cpu().numpy(), ids, weights, layer.v13, layer.v2, limit)
    info = torch.finfo(dtype)
    tol = tol + info.eps / 2 * (np.abs(want) + tol) + info.smallest_normal * info.eps
    off = np.abs(got.double().cpu().numpy() - want) - tol
    assert (off <= 0).all(), f"max excess {off.max():.3g} of {np.abs(want).max():.3g}"


CASES = [  # experts, hidden, inter, topk, tokens
    (1, 32, 32, 1, 1), (4, 64, 32, 2, 3), (8, 256, 96, 2, 1), (8, 288, 160, 8, 1), (16, 128, 64, 3, 2),
    (16, 512, 256, 4, 5), (8, 416, 224, 2, 40), (4, 256, 128, 1, 70), (64, 128, 64, 6, 33), (3, 160, 96, 3, 150),
    (2, 384, 320, 1, 300), (40, 96, 32, 5, 20), (128, 64, 32, 8, 17), (300, 64, 32, 4, 30),
    # few rows' kernels: several tasks of 16 rows an expert, listed and looked for; whole
    # blocks a wavefront, by expert and by slot; more than eight and 64 slots a token
    (64, 128, 64, 6, 200), (8, 160, 96, 2, 100), (64, 256, 512, 2, 40), (128, 64, 512, 2, 62), (32, 128, 64, 20, 2),
    (100, 64, 32, 64, 1), (100, 64, 32, 65, 1), (100, 64, 32, 40, 2), (4, 64, 2080, 2, 1), (6, 64, 4128, 1, 4),
    # rows so long that LDS holds fewer than 16 (and one)
    (2, 8192, 64, 1, 30), (4, 96, 8192, 1, 80), (2, 8192, 64, 2, 600), (1, 65536, 32, 1, 2), (1, 32, 65536, 1, 2),
    # tiles: several an expert, a few rows of many experts, sizes that end inside a stage
    (2, 256, 256, 1, 700), (3, 288, 416, 2, 450), (200, 256, 256, 8, 150), (16, 256, 288, 4, 16), (16, 256, 288, 4, 17)]


@pytest.mark.parametrize("experts,hidden,inter,topk,tokens", CASES)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_matches_the_oracle(mx, device, experts, hidden, inter, topk, tokens, dtype):
    print(f"moe E={experts} H={hidden} I={inter} k={topk} T={tokens} {dtype}", flush=True)
    rng = np.random.default_rng(experts + hidden + tokens)
    layer = Layer(rng, experts, hidden, inter, device)
    ids, weights = routing(rng, tokens, experts, topk)
    x = torch.from_numpy(rng.standard_normal((tokens, hidden))).to(TYPES[dtype]).to(device)
    limit = 2.0 if tokens % 2 else math.inf
    got = layer.run(mx, x, torch.from_numpy(weights).to(device), torch.from_numpy(ids).to(device),
                    clamp_limit=None if math.isinf(limit) else limit)
    check(layer, got, x, ids, weights, TYPES[dtype], limit)


@pytest.mark.parametrize("hidden,inter", [(192, 96), (288, 320)])
@pytest.mark.parametrize("tokens", [1, 6, 90])
def test_expert_map_masked_slots_and_repeats(mx, device, tokens, hidden, inter):
    """A part of the layer's experts, ids out of range, one expert twice in a
    row, rows with no slot left (zeros), all slots on one expert."""
    rng = np.random.default_rng(tokens)
    layer = Layer(rng, 6, hidden, inter, device)
    emap = np.array([-1, 3, 0, -1, 5, 2, 77, 1, 4, -5], np.int32)
    ids = rng.integers(-2, 12, (tokens, 4)).astype(np.int32)
    ids[0] = [1, 1, 4, 4]
    if tokens > 2:
        ids[1] = -1
        ids[2] = [0, 3, 6, 11]
    weights = rng.random((tokens, 4)).astype(np.float32)
    local = np.where((ids >= 0) & (ids < len(emap)), emap[np.clip(ids, 0, len(emap) - 1)], -1)
    x = torch.from_numpy(rng.standard_normal((tokens, hidden))).bfloat16().to(device)
    tw = torch.from_numpy(weights).to(device)
    got = layer.run(mx, x, tw, torch.from_numpy(ids).to(device), expert_map=torch.from_numpy(emap).to(device))
    check(layer, got, x, local, weights, torch.bfloat16)
    if tokens > 2:
        assert not got[1].any() and not got[2].any()
    same = layer.run(mx, x, tw, torch.from_numpy(ids).long().to(device), expert_map=torch.from_numpy(emap).long().to(device))
    assert torch.equal(same, got)
    none = layer.run(mx, x, tw, torch.full((tokens, 4), -1, dtype=torch.int32, device=device))
    assert not none.any()
    one = torch.full((tokens, 4), 5, dtype=torch.int32, device=device)
    check(layer, layer.run(mx, x, tw, one), x, np.full((tokens, 4), 5), weights, torch.bfloat16)


@pytest.mark.parametrize("inter", [128, 288])
def test_rows_do_not_depend_on_each_other(mx, device, inter):
    """A NaN row, and one of infinities, leave the other rows' bits; row strides."""
    rng = np.random.default_rng(0)
    layer = Layer(rng, 8, 256, inter, device)
    ids, weights = routing(rng, 50, 8, 2)
    ti, tw = torch.from_numpy(ids).to(device), torch.from_numpy(weights).to(device)
    wide = torch.from_numpy(rng.standard_normal((50, 300))).bfloat16().to(device)
    x = wide[:, 8:264]
    clean = layer.run(mx, x.contiguous(), tw, ti)
    assert torch.equal(layer.run(mx, x, tw, ti), clean)
    odd = wide[:, 3:259]
    assert torch.equal(layer.run(mx, odd, tw, ti), layer.run(mx, odd.contiguous(), tw, ti))
    bad = x.contiguous().clone()
    bad[7, 100] = float("nan")
    bad[31] = float("inf")
    got = layer.run(mx, bad, tw, ti)
    assert torch.isnan(got[7]).all() and torch.isnan(got[31]).all()
    keep = [t for t in range(50) if t not in (7, 31)]
    assert torch.equal(got[keep], clean[keep])


@pytest.mark.parametrize("size,copies", [(128, 1), (256, 1), (256, 7)])
def test_weights_with_a_nan_expert(mx, device, size, copies):
    rng = np.random.default_rng(2)
    layer = Layer(rng, 4, size, size, device)
    ids = torch.tensor([[0, 1], [2, 3], [1, 2]] * copies, dtype=torch.int32, device=device)
    tw = torch.full((3 * copies, 2), 0.5, device=device)
    x = torch.from_numpy(rng.standard_normal((3 * copies, size)) * 0.1).half().to(device)
    clean = layer.run(mx, x, tw, ids)
    assert torch.isfinite(clean).all()
    layer.s13[3, 10, 1] = 255  # a gate row: h's block is NaN, and so every output
    got = layer.run(mx, x, tw, ids)
    hit = torch.arange(3 * copies, device=device) % 3 == 1
    assert torch.isnan(got[hit]).all() and torch.equal(got[~hit], clean[~hit])


def test_refusals(mx, device):
    rng = np.random.default_rng(3)
    layer = Layer(rng, 4, 128, 64, device)
    x = torch.zeros(3, 128, dtype=torch.bfloat16, device=device)
    ids = torch.zeros(3, 2, dtype=torch.int32, device=device)
    tw = torch.ones(3, 2, device=device)
    ok = (x, layer.w13, layer.w2, layer.s13, layer.s2, tw, ids)
    for i, bad in ((0, x.float()), (0, x[:, :64]), (0, x.t().contiguous().t()), (1, layer.w13[:3]), (2, layer.w2[:, :64]),
                   (3, layer.s13[:, :, :1]), (1, layer.w13.view(torch.int8)), (5, tw[:2]), (6, ids[:2]), (4, layer.s2.cpu())):
        args = list(ok)
        args[i] = bad
        with pytest.raises(RuntimeError):
            mx.fused_mxfp4_moe(*args)
            pytest.fail(f"argument {i} was taken")
    for kw in ({"clamp_limit": -1.0}, {"clamp_limit": float("nan")}, {"output": x[:2]}, {"output": x.float()},
               {"expert_map": ids}):
        with pytest.raises(RuntimeError):
            mx.fused_mxfp4_moe(*ok, **kw)
            pytest.fail(f"{kw} was taken")
    assert mx.fused_mxfp4_moe(x[:0], *ok[1:5], tw[:0], ids[:0]).shape == (0, 128)
    out = torch.empty_like(x)
    assert mx.fused_mxfp4_moe(*ok, output=out) is out


@pytest.mark.parametrize("inter", [128, 256])
@pytest.mark.parametrize("tokens", [1, 3, 64, 200, 700])
def test_streams_workspace_and_graph(mx, device, tokens, inter):
    """Equal bits on another stream, with a workspace that a larger call left,
    and on every replay of a graph with new inputs and new routing."""
    print(f"moe graph T={tokens} I={inter}", flush=True)
    rng = np.random.default_rng(tokens + 1)
    layer = Layer(rng, 16, 256, inter, device)
    sets = []
    for _ in range(3):
        ids, weights = routing(rng, tokens, 16, 4)
        sets.append((torch.from_numpy(rng.standard_normal((tokens, 256))).bfloat16().to(device),
                     torch.from_numpy(weights).to(device), torch.from_numpy(ids).to(device)))
    want = [layer.run(mx, *s) for s in sets]
    ws = {}
    big = torch.from_numpy(rng.standard_normal((300, 256))).bfloat16().to(device)
    bi, bw = routing(rng, 300, 16, 4)
    layer.run(mx, big, torch.from_numpy(bw).to(device), torch.from_numpy(bi).to(device), workspace=ws)
    for s, y in zip(sets, want):
        assert torch.equal(layer.run(mx, *s, workspace=ws), y)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = layer.run(mx, *sets[0])
    second = layer.run(mx, *sets[1])
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(first, want[0]) and torch.equal(second, want[1])
    static = tuple(t.clone() for t in sets[0])
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out = layer.run(mx, *static)
    for i in (1, 2, 0, 1):
        for dst, src in zip(static, sets[i]):
            dst.copy_(src)
        graph.replay()
        again = layer.run(mx, *sets[i])
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]) and torch.equal(again, want[i])


@pytest.mark.parametrize("inter", [128, 256])
def test_a_graph_outlives_its_workspace(mx, device, inter):
    """Calls captured with a workspace, which later calls replace by larger ones
    and whose memory others then write; two graphs replayed in turn; the output
    in the place of the input."""
    print("moe graphs and a workspace", flush=True)
    rng = np.random.default_rng(8)
    layer = Layer(rng, 8, 256, inter, device)
    def call(tokens):
        ids, weights = routing(rng, tokens, 8, 2)
        return (torch.from_numpy(rng.standard_normal((tokens, 256))).bfloat16().to(device),
                torch.from_numpy(weights).to(device), torch.from_numpy(ids).to(device))
    small, large = call(5), call(90)
    want = [layer.run(mx, *small), layer.run(mx, *large)]
    ws, graphs, outs = {}, [], []
    layer.run(mx, *small, workspace=ws)
    torch.cuda.synchronize()
    for args in (small, large):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(layer.run(mx, *args, workspace=ws))
        graphs.append(graph)
    layer.run(mx, *call(600), workspace=ws)
    taken = [torch.full((1 << 16,), 255, dtype=torch.uint8, device=device) for _ in range(64)]
    for i in (0, 1, 1, 0):
        outs[i].zero_()
        graphs[i].replay()
        layer.run(mx, *large, workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(outs[i], want[i])
    assert all(bool((t == 255).all()) for t in taken)
    for args, y in zip((small, large), want):
        x = args[0].clone()
        assert layer.run(mx, x, *args[1:], output=x) is x and torch.equal(x, y)


def test_router_load_and_experts_together(mx, device):
    """A layer as it runs: route, the router's load and loss, the experts."""
    from oracle import balance_oracle as B
    from vllm_mi355x.kernels.moe import moe_balance_loss, moe_expert_counts, moe_route
    rng = np.random.default_rng(4)
    tokens, experts, hidden, inter, topk = 37, 16, 256, 128, 4
    layer = Layer(rng, experts, hidden, inter, device)
    x = torch.from_numpy(rng.standard_normal((tokens, hidden))).bfloat16().to(device)
    gate = torch.from_numpy(rng.standard_normal((experts, hidden)) * 0.1).bfloat16().to(device)
    pad = torch.zeros(tokens, dtype=torch.bool, device=device)
    pad[[3, 36]] = True
    logits, weights, ids, *_ = moe_route(x, gate, None, topk=topk, num_experts=experts, scoring="softmax",
                                         routed_scaling_factor=1.0, is_padding=pad)
    y = layer.run(mx, x, weights, ids)
    check(layer, y, x, ids.cpu().numpy(), weights.cpu().numpy(), torch.bfloat16)
    assert not y[pad].any()
    logits.requires_grad_()
    loss, counts = moe_balance_loss(logits, ids, is_padding=pad)
    loss.backward()
    want, wc, wg = B.loss_and_grad(logits.detach().double().cpu().numpy(), ids.cpu().numpy(), False, pad.cpu().numpy())
    assert abs(loss.item() - want) <= 2.0 ** -18 * want and np.array_equal(counts.cpu().numpy(), wc)
    assert np.abs(logits.grad.double().cpu().numpy() - wg).max() <= 2.0 ** -18 * np.abs(wg).max() * 4
    assert torch.equal(moe_expert_counts(ids, experts), counts) and int(counts.sum()) == (tokens - 2) * topk
