"""The fused MXFP4 MoE where a task's rows just fit LDS, or just do not: tasks of 16
rows and a few more, of rows up to 7168 elements and above; and few tokens whose slots are
many to an expert, or more than a workgroup lists.  Tolerance as the oracle
gives it, then half a step of the type."""

import numpy as np
import pytest
import torch

from oracle import mxfp4_oracle as M

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def mx():
    from vllm_mi355x.kernels import mxfp4
    return mxfp4


@pytest.mark.parametrize("experts,hidden,inter,topk,tokens", [(2, 6656, 32, 1, 40), (2, 7168, 32, 1, 40), (2, 7200, 32, 1, 40),
                                                              (1, 7168, 64, 1, 16), (1, 7168, 64, 1, 17), (2, 64, 7168, 2, 33),
                                                              (3, 6688, 32, 2, 700), (40, 7168, 32, 8, 8),
                                                              # tiles for few tokens, many to an expert; long lists of few tokens
                                                              (4, 256, 288, 4, 12), (2, 512, 256, 2, 16), (200, 64, 32, 100, 12)])
def test_rows_that_just_fit(mx, device, experts, hidden, inter, topk, tokens):
    print(f"moe rows E={experts} H={hidden} I={inter} k={topk} T={tokens}", flush=True)
    rng = np.random.default_rng(hidden + tokens)

    def packed(*shape):
        code = rng.integers(0, 16, shape).astype(np.uint8)
        byte = rng.integers(119, 123, (*shape[:-1], shape[-1] // 32)).astype(np.uint8)
        return torch.from_numpy(M.pack(code)).to(device), torch.from_numpy(byte).to(device), M.values(code, byte)

    w13, s13, v13 = packed(experts, 2 * inter, hidden)
    w2, s2, v2 = packed(experts, hidden, inter)
    ids = np.stack([rng.permutation(experts)[:topk] for _ in range(tokens)]).astype(np.int32)
    weights = (rng.random((tokens, topk)) + 0.1).astype(np.float32)
    x = torch.from_numpy(rng.standard_normal((tokens, hidden))).bfloat16().to(device)
    got = mx.fused_mxfp4_moe(x, w13, w2, s13, s2, torch.from_numpy(weights).to(device), torch.from_numpy(ids).to(device))
    want, tol = M.moe(x.double().cpu().numpy(), ids, weights, v13, v2)
    tol = tol + 2.0 ** -8 * (np.abs(want) + tol) + 2.0 ** -133
    off = np.abs(got.double().cpu().numpy() - want) - tol
    assert (off <= 0).all(), f"max excess {off.max():.3g} of {np.abs(want).max():.3g}"
