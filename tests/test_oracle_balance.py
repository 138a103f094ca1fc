"""Pins of the balance-loss oracle: even and one-sided load by hand, the gradient
by central differences."""

import numpy as np
import pytest

from oracle import balance_oracle as B


def test_even_load_gives_one():
    ids = np.arange(12).reshape(6, 2) % 4
    assert B.loss_and_grad(np.zeros((6, 4)), ids)[0] == pytest.approx(1.0, abs=1e-15)


def test_all_rows_on_one_expert():
    logits = np.log(np.array([[0.7, 0.2, 0.1]] * 5))
    loss, counts, _ = B.loss_and_grad(logits, np.zeros((5, 1), int))
    assert loss == pytest.approx(3 * 0.7) and counts.tolist() == [5, 0, 0]


def test_nothing_left():
    logits = np.full((2, 3), -np.inf)
    ids = np.array([[0], [1]])
    for sigmoid in (False, True):
        loss, _, grad = B.loss_and_grad(logits, ids, sigmoid)
        assert loss == 0 and not grad.any()
    loss, counts, grad = B.loss_and_grad(np.zeros((2, 3)), ids, padding=np.array([True, True]))
    assert loss == 0 and not counts.any() and not grad.any()


@pytest.mark.parametrize("sigmoid", [False, True])
def test_gradient_by_differences(sigmoid):
    rng = np.random.default_rng(1)
    logits = rng.standard_normal((5, 6)) * 2
    ids = rng.integers(-1, 6, (5, 2))
    pad = np.array([False, True, False, False, False])
    _, _, grad = B.loss_and_grad(logits, ids, sigmoid, pad)
    step = 1e-5
    for t in range(5):
        for e in range(6):
            up, down = logits.copy(), logits.copy()
            up[t, e] += step
            down[t, e] -= step
            d = (B.loss_and_grad(up, ids, sigmoid, pad)[0] - B.loss_and_grad(down, ids, sigmoid, pad)[0]) / (2 * step)
            assert abs(d - grad[t, e]) < 1e-8
