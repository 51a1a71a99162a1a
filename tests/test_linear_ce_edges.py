"""The linear cross entropy where its tiles, signs and ranges meet: results of several tiles a block, rows that
are sure of their target, tokens far below the likeliest, sums over many rows, infinite logits.  The formula
in 64 bits and the bounds are those of the tests of its values; a tighter bound is derived where it is used."""

import pytest
import torch

from tests.test_linear_ce import F16, _bounds, _call, _check, _make, _truth

gpu = pytest.mark.gpu


@pytest.fixture(scope="module")
def eng(cuda_ctx):
    from ferrotensor_b200.engine import ComputeEngine
    return ComputeEngine(cuda_ctx)


@gpu
@pytest.mark.parametrize("mode", ["F16", "F16X2"])
@pytest.mark.parametrize("vocab_major", [False, True])
@pytest.mark.parametrize("rows,hidden", [(64, 576), (300, 576), (64, 896), (300, 960), (130, 64)])
def test_f16_weight_gradients_of_many_tiles(cuda_ctx, eng, mode, vocab_major, rows, hidden):
    """Hidden sizes whose tiles give a warp an odd number of 32-column blocks (192, 224 and 64 columns), few
    rows (a tile is multiplied sooner than it is stored) and several tiles for every block: each element
    of every tile, and the same bits each time."""
    x, w, y, a = _make(rows, hidden, 30208, (F16, F16), vocab_major, "half", 700 + hidden)
    q = _truth(x, w, y, a, 512.0, vocab_major)
    tols = _bounds(q, mode, (F16, F16), (F16, F16))
    first = _call(cuda_ctx, eng, mode, x, w, y, a, 512.0, vocab_major, (F16, F16))
    _check(first, q, tols, vocab_major)
    for _ in range(4):
        again = _call(cuda_ctx, eng, mode, x, w, y, a, 512.0, vocab_major, (F16, F16))
        assert all(torch.equal(p, r) for p, r in zip(first, again))
