"""CPU statement of MXFP4 (blocks of 32, E2M1 codes under an E8M0 scale byte),
its product and the routed experts in it, in FP64 NumPy.

TEST INFRASTRUCTURE ONLY.  Only tests/ may import this module;
the product path (vllm-cmp170hx_amd/) never does.

Pinned by closed forms (tests/test_oracle_mxfp4.py): every code's value, the
midpoints' ties, scales at the ends of the range, blocks with NaN or infinity.
"""

from __future__ import annotations

import numpy as np

BLOCK = 32
GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def quantize_blocks(x):
    """x [..., k] FP64 -> (codes 0..15 [..., k], scale bytes [..., k / 32])."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], x.shape[-1] // BLOCK, BLOCK)
    top = np.abs(b).max(-1)
    finite = np.isfinite(b).all(-1)
    _, e = np.frexp(np.where(finite & (top > 0), top, 1.0))  # top = m 2^e, m in [0.5, 1)
    byte = np.where(top > 0, np.maximum(e - 1 - 2 + 127, 0), 0)
    byte = np.where(finite, byte, 255).astype(np.int64)
    with np.errstate(invalid="ignore", over="ignore"):
        a = np.ldexp(np.abs(b), (127 - byte)[..., None])
    # nearest of the grid, a tie to the even code
    lower = np.clip(np.searchsorted(GRID, a, side="right") - 1, 0, 6)
    mid = (GRID[lower] + GRID[lower + 1]) / 2
    up = (a > mid) | ((a == mid) & (lower % 2 == 1))
    code = lower + up
    code = np.where(np.signbit(b), code + 8, code)
    code = np.where(finite[..., None], code, 0)
    return code.reshape(x.shape).astype(np.uint8), byte.astype(np.uint8)


def pack(code):
    return (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8)


def unpack(packed):
    return np.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], 2 * packed.shape[-1])


def values(code, byte):
    """Codes and scale bytes -> FP64 values."""
    v = np.where(code >= 8, -1.0, 1.0) * GRID[code & 7]
    s = np.where(byte == 255, np.nan, np.ldexp(1.0, byte.astype(np.int64) - 127))
    return (v.reshape(*byte.shape, BLOCK) * s[..., None]).reshape(code.shape)


def quantized(x):
    return values(*quantize_blocks(x))


def silu(g):
    with np.errstate(over="ignore"):
        return g / (1.0 + np.exp(-g))


def moe(x, ids, weights, w13, w2, limit=np.inf):
    """x [T, K] (quantized here), ids [T, k] local experts (others: no part),
    w13 [E, 2 I, K], w2 [E, K, I] FP64 values -> (out [T, K], tolerance [T, K]).

    tolerance: what FP32 sums may make of it.  A sum of n products is off by at
    most n 2^-23 of the sum of their magnitudes; that moves h, and where h then
    lies nearer than that to a midpoint of its grid (or its block's largest
    magnitude to a power of two), its code may be its neighbour's: one step of
    the grid (two where the scale may change)."""
    xq = quantized(x)
    T, K = x.shape
    inter = w2.shape[2]
    out, tol = np.zeros((T, K)), np.zeros((T, K))
    unit = 2.0 ** -23
    for t in range(T):
        for slot in range(ids.shape[1]):
            e = ids[t, slot]
            if e < 0 or e >= w13.shape[0]:
                continue
            gu = w13[e] @ xq[t]
            d = (K / 32 + 8) * unit * (np.abs(w13[e]) @ np.abs(xq[t]))
            g, u = gu[:inter], gu[inter:]
            gc, uc = np.minimum(g, limit), np.clip(u, -limit, limit)
            h = silu(gc) * uc
            dh = 1.1 * d[:inter] * (np.abs(uc) + d[inter:]) + np.abs(silu(gc)) * d[inter:] \
                + 2.0 ** -20 * np.abs(h)
            code, byte = quantize_blocks(h)
            hq = values(code, byte)
            b = byte.astype(np.int64) - 127
            scale = np.ldexp(1.0, b)[:, None]
            a, da = np.abs(h).reshape(-1, BLOCK) / scale, dh.reshape(-1, BLOCK) / scale
            mids = (GRID[1:] + GRID[:-1]) / 2
            near = (np.abs(a[..., None] - mids) <= da[..., None]).any(-1)
            step = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
            step = np.where(np.abs(a - 2) <= da, 1.0, np.where(np.abs(a - 4) <= da, 2.0, step))
            at = a.argmax(-1)[:, None]
            top, dtop = np.take_along_axis(a, at, -1), da.max(-1, keepdims=True)
            moved = (np.abs(top - 8) <= dtop) | (np.abs(top - 4) <= dtop)
            slack = (np.where(moved, 2 * np.maximum(step, 1.0), np.where(near, step, 0.0)) * scale).reshape(-1)
            y = w2[e] @ hq
            wt = float(weights[t, slot])
            out[t] += wt * y
            tol[t] += abs(wt) * (np.abs(w2[e]) @ (slack + (inter / 32 + 8) * unit * np.abs(hq))
                                 + 2.0 ** -22 * np.abs(y))
    return out, tol
