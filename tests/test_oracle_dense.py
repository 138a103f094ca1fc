"""The dense layer's oracle: slopes and gradients against differences, activations against
torch's in 64 bits."""

import numpy as np
import pytest
import torch

from oracle import dense_oracle as D


@pytest.mark.parametrize("name", [None, "relu", "gelu", "gelu_tanh", "silu"])
def test_activations_and_slopes(name):
    z = np.linspace(-9, 9, 400)
    f = torch.nn.functional
    t = torch.from_numpy(z)
    want = {None: t, "relu": f.relu(t), "gelu": f.gelu(t), "gelu_tanh": f.gelu(t, approximate="tanh"), "silu": f.silu(t)}[name]
    assert np.allclose(D.activate(name, z), want.numpy(), rtol=1e-9, atol=1e-12)
    d = (D.activate(name, z + 1e-6) - D.activate(name, z - 1e-6)) / 2e-6
    assert np.allclose(D.slope(name, z), d, atol=1e-7)
    assert np.abs(D.slope(name, z)).max() <= D.STEEP
    bend = np.abs(D.slope(name, z[1:]) - D.slope(name, z[:-1])) / np.diff(z)
    if name != "relu":
        assert bend.max() <= D.BEND[name] + 1e-9


@pytest.mark.parametrize("activation", [None, "relu", "gelu", "gelu_tanh", "silu", "swiglu"])
def test_gradient_by_differences(activation):
    rng = np.random.default_rng(1)
    lines = 8 if activation == "swiglu" else 4
    x, w, b = rng.standard_normal((3, 5)), rng.standard_normal((lines, 5)), rng.standard_normal(lines)
    dy = rng.standard_normal((3, 4))
    limit = 1.0 if activation == "swiglu" else np.inf
    grads, _ = D.backward(x, w, b, activation, dy, 0.0, limit)
    loss = lambda: (D.forward(x, w, b, activation, None, limit)[0] * dy).sum()
    for name, a in (("x", x), ("w", w), ("bias", b)):
        for at in np.ndindex(a.shape):
            old = a[at]
            a[at] = old + 1e-6
            up = loss()
            a[at] = old - 1e-6
            diff = (up - loss()) / 2e-6
            a[at] = old
            assert abs(grads[name][0][at] - diff) <= 1e-7


@pytest.mark.parametrize("name", [None, "relu", "gelu", "gelu_tanh", "silu"])
def test_slopes_at_nan(name):
    """As torch's: an activation that keeps a NaN does not drop its gradient."""
    f = torch.nn.functional
    z = torch.tensor([float("nan")], dtype=torch.float64, requires_grad=True)
    y = {None: z * 1, "relu": f.relu(z), "gelu": f.gelu(z), "gelu_tanh": f.gelu(z, approximate="tanh"), "silu": f.silu(z)}[name]
    want, = torch.autograd.grad(y, z)
    assert torch.isnan(y) and np.isnan(D.activate(name, z.detach().numpy())).all()
    assert np.array_equal(D.slope(name, z.detach().numpy()), want.numpy(), equal_nan=True)
