"""The oracle of routing from logits against hand-made rows, the router's own
oracle and differences."""

import numpy as np
import pytest

from oracle import route_logits_oracle as L
from oracle import route_oracle as R


def test_groups_and_ties_by_hand():
    row = np.array([1.0, 5.0, 2.0, 2.0, 4.0, 0.0, 3.0, 3.0])
    assert L.choice(row, 3, False).tolist() == [1, 4, 6]
    assert L.choice(row, 2, False, groups=4, topk_groups=1).tolist() == [1, 0]
    # without a bias groups score 5, 2, 4, 3; with one (of zeros) by two sigmoids
    assert L.choice(row, 4, False, groups=4, topk_groups=2).tolist() == [1, 4, 0, 5]
    s = 1 / (1 + np.exp(-row))
    pairs = s.reshape(4, 2).sum(1)
    best = int(pairs.argmax())
    assert L.choice(row, 2, True, np.zeros(8, np.float32), 4, 1).tolist() == sorted(
        (2 * best, 2 * best + 1), key=lambda e: (-s[e], e))
    assert L.choice(np.zeros(6), 3, True, groups=3, topk_groups=2).tolist() == [0, 1, 2]


def test_masks_by_hand():
    low = np.finfo(np.float32).min
    row = np.array([-np.inf, 1.0, low, -800.0])
    assert L.choice(row, 3, True).tolist() == [1, -1, -1]
    assert L.choice(np.full(4, low), 2, False).tolist() == [0, 1]
    assert L.choice(np.full(4, low), 2, True).tolist() == [-1, -1]
    assert L.choice(np.array([1.0, np.nan, 2.0]), 3, False).tolist() == [2, 0, -1]
    bias = np.array([0, -np.inf, np.nan, 9], np.float32)
    assert L.choice(np.zeros(4), 4, True, bias).tolist() == [3, 0, -1, -1]
    assert np.isnan(L.weigh(np.array([1.0, np.nan, 2.0]), np.array([2, 0, -1]), False, True, 1.0)[:2]).all()


@pytest.mark.parametrize("sigmoid", [False, True])
def test_agrees_with_the_routers_oracle(sigmoid):
    rng = np.random.default_rng(1)
    logits = rng.standard_normal((50, 40)).astype(np.float32) * 2
    bias = rng.standard_normal(40).astype(np.float32) if sigmoid else None
    ids, w = L.route(logits, 6, sigmoid, bias, scale=2.5)
    want, ww, _ = R.route(logits, 6, sigmoid, bias, scale=2.5)
    assert np.array_equal(ids, want) and np.allclose(w, ww, rtol=1e-5)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("renormalize", [False, True])
def test_gradient_by_differences(sigmoid, renormalize):
    rng = np.random.default_rng(2)
    row, up = rng.standard_normal(9) * 2, rng.standard_normal(4)
    ids = np.array([3, 0, 7, -1], np.int32)
    grad = L.gradient(row, ids, L.weigh(row, ids, sigmoid, renormalize, 2.5), up, sigmoid, renormalize, 2.5)
    for e in range(9):
        d = np.zeros(9)
        d[e] = 1e-6
        diff = sum((up * (L.weigh(row + d, ids, sigmoid, renormalize, 2.5) - L.weigh(row - d, ids, sigmoid, renormalize, 2.5)))) / 2e-6
        assert abs(grad[e] - diff) <= 1e-8
