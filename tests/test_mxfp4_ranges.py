"""Sizes past what the MXFP4 products count in, on the CPU: refused, with addresses
that no check follows."""

import pytest


@pytest.fixture(scope="module")
def lib():
    from vllm_mi355x import _native
    return _native.load()


@pytest.mark.parametrize("k", [(1 << 32) + 32, 1 << 36, 1 << 37, (1 << 37) + 4096])
def test_products_of_too_long_rows(lib, k):
    """(A row of 2^36 elements has 2^31 blocks.)"""
    a, sa, w, sw, out, ws = (i << 50 for i in range(1, 7))
    error = lambda: lib.vllm_mi355x_last_error().decode()
    assert lib.mxfp4_matmul(a, sa, 1, k, w, sw, 1, out, 2, ws, 1 << 40, 0) == 1 and "range" in error()
    assert lib.mxfp4_linear(a, 0, 1, k, k, w, sw, 1, out, 2, ws, 1 << 45, 0) == 1 and "range" in error()
    assert lib.mxfp4_matmul_workspace_size(1, k, 1) == -1 and "2^32" in error()
    assert lib.mxfp4_linear_workspace_size(1, k, 1) == -1 and "2^32" in error()
