"""Pins of the MXFP4 oracle by closed forms."""

import numpy as np

from oracle import mxfp4_oracle as M


def test_every_code_stands_for_itself():
    for byte in (0, 1, 100, 127, 200, 252):
        x = np.zeros(32)
        x[:16] = np.concatenate([M.GRID, -M.GRID]) * 2.0 ** (byte - 127)
        code, b = M.quantize_blocks(x)
        assert b[0] == byte
        assert np.array_equal(code[:16], np.arange(16))
        assert np.array_equal(M.values(code, b), x)


def test_ties_go_to_even_codes_and_large_values_saturate():
    x = np.zeros(32)
    x[:10] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 5.01, 7.0, 7.99]
    assert list(M.quantized(x)[:10]) == [0, 1, 1, 2, 2, 4, 4, 6, 6, 6]
    assert np.array_equal(M.quantized(-x), -M.quantized(x))
    x[10] = 8.0  # the block's scale doubles
    assert list(M.quantized(x)[:11]) == [0, 1, 1, 2, 2, 4, 4, 6, 8, 8, 8]


def test_ends_of_the_range():
    x = np.zeros((3, 32))
    x[0, 0] = 2.0 ** -149
    x[1, 3] = np.nan
    x[2, 5] = -np.inf
    code, byte = M.quantize_blocks(x)
    assert byte.reshape(-1).tolist() == [0, 255, 255]
    assert not code.any()
    assert np.isnan(M.values(code, byte)[1:]).all()
    big = np.full(32, float(np.finfo(np.float32).max))
    assert M.quantize_blocks(big)[1][0] == 252
    assert M.quantized(big)[0] == 6 * 2.0 ** 125


def test_packing():
    code = np.arange(64, dtype=np.uint8).reshape(2, 32) % 16
    packed = M.pack(code)
    assert packed[0, 0] == 0x10 and packed[0, 1] == 0x32
    assert np.array_equal(M.unpack(packed), code)


def test_error_is_at_most_half_a_step():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 96)) * np.exp(rng.standard_normal((50, 1)) * 5)
    code, byte = M.quantize_blocks(x)
    scale = np.repeat(np.ldexp(1.0, byte.astype(int) - 127), 32, -1)
    a = np.abs(x) / scale
    step = np.where(a < 2, 0.5, np.where(a < 4, 1, 2))
    off = np.abs(M.values(code, byte) - x) / scale
    assert (off <= np.where(a > 6, a - 6, step / 2)).all()
