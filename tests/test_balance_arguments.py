"""The balance entry points' arrays, on the CPU: outputs that overlap another array, and
pointers off their elements, are refused before anything runs."""

import pytest

A = 1 << 30  # an address that no check follows; the others lie A apart


@pytest.fixture(scope="module")
def lib():
    from vllm_mi355x import _native
    return _native.load()


def error(lib):
    return lib.vllm_mi355x_last_error().decode()


def counts(ids=A, pad=2 * A, out=3 * A, ws=4 * A):
    return ids, pad, 100, 2, 16, 0, out, ws, 1 << 20, 0


def loss(logits=A, ids=2 * A, pad=3 * A, out=4 * A, counts=5 * A, stats=6 * A, ws=7 * A, stride=16):
    return logits, 2, 100, 16, stride, ids, 2, pad, 0, out, counts, stats, ws, 1 << 20, 0


def grad(logits=A, pad=2 * A, stats=3 * A, up=4 * A, out=5 * A, stride=16):
    return logits, 2, 100, 16, stride, pad, 0, stats, up, out, 0


@pytest.mark.parametrize("call,args,word", [
    ("moe_expert_counts", counts(out=A + 8), "overlap"), ("moe_expert_counts", counts(out=2 * A - 8), "overlap"),
    ("moe_expert_counts", counts(ws=A), "overlap"), ("moe_expert_counts", counts(ws=3 * A), "overlap"),
    ("moe_expert_counts", counts(ids=A + 2), "misaligned"), ("moe_expert_counts", counts(out=3 * A + 4), "misaligned"),
    ("moe_balance_loss", loss(out=A + 6400 - 4), "overlap"), ("moe_balance_loss", loss(stats=5 * A + 64), "overlap"),
    ("moe_balance_loss", loss(counts=3 * A), "overlap"), ("moe_balance_loss", loss(ws=A), "overlap"),
    ("moe_balance_loss", loss(ws=A + 99 * 80 + 64 - 8, stride=20), "overlap"),
    ("moe_balance_loss", loss(logits=A + 2), "misaligned"), ("moe_balance_loss", loss(out=4 * A + 2), "misaligned"),
    ("moe_balance_loss", loss(counts=5 * A + 4), "misaligned"), ("moe_balance_loss", loss(stats=6 * A + 1), "misaligned"),
    ("moe_balance_grad", grad(out=A + 64), "overlap"), ("moe_balance_grad", grad(out=A, stride=20), "overlap"),
    ("moe_balance_grad", grad(out=3 * A), "overlap"), ("moe_balance_grad", grad(up=5 * A + 32), "overlap"),
    ("moe_balance_grad", grad(out=2 * A - 16), "overlap"), ("moe_balance_grad", grad(up=4 * A + 2), "misaligned"),
    ("moe_balance_grad", grad(logits=A + 1), "misaligned")])
def test_refusals(lib, call, args, word):
    assert getattr(lib, call)(*args) == 1 and word in error(lib), error(lib)


def test_expert_map_off_its_elements(lib):
    at = [(i + 1) << 40 for i in range(10)]
    args = (at[0], 0, 2, 64, at[1], at[2], at[3], at[4], 4, at[5], at[6], 2, at[7] + 2, 8, 64, 32, float("inf"), at[8],
            at[9], 1 << 30, 0)
    assert lib.mxfp4_moe(*args) == 1 and "misaligned" in error(lib)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,experts", [(7, 5), (300, 64), (2500, 256)])
@pytest.mark.parametrize("scoring", [0, 1])
def test_gradient_in_place_of_the_logits(lib, device, rows, experts, scoring):
    """The bits of a gradient beside them."""
    import torch

    g = torch.Generator(device=device).manual_seed(rows)
    logits = torch.randn(rows, experts, device=device, generator=g) * 3 - 20 * scoring
    logits[rows // 2] -= 300
    stats = torch.rand(experts + 1, device=device, generator=g)
    up = torch.full((1,), 2.0, device=device)
    out, place = torch.empty_like(logits), logits.clone()
    stream = torch.cuda.current_stream(device).cuda_stream
    for x, y in ((logits, out), (place, place)):
        assert lib.moe_balance_grad(x.data_ptr(), 2, rows, experts, experts, 0, scoring, stats.data_ptr(), up.data_ptr(),
                                    y.data_ptr(), stream) == 0
    assert torch.isfinite(out).all() and torch.equal(out, place)
