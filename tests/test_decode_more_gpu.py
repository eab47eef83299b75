"""Cache append, paged attention and adapters, continued: rows, orders and values that the first file of tests does not meet.
Tolerances are those of test_decode_gpu.py where nothing else is said (u = 2^-23)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(__file__))
from test_decode_gpu import attend, batch, check_attention, status  # noqa: E402

pytestmark = pytest.mark.gpu


# ---- runs of pages ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("page,dim", [(1, 48), (3, 16), (5, 80), (24, 48), (40, 96), (64, 144)])
@pytest.mark.parametrize("i8", [0, 1])
@pytest.mark.parametrize("lens", [[9000], [700, 0, 1, 3000, 33, 0, 2], [5, 90, 0, 31] * 40])
def test_attention_of_many_runs(page, dim, i8, lens):
    """Rows of which some lanes copy nothing, and pages so small, or units so short, that a warp goes on to another run after
    every few steps: the same bits in every call."""
    cache, q, table, length = batch(page + dim, lens, (page, 3, dim, i8, "hnd", 0), 6)
    got, lse = attend(cache, q, table, length)
    assert status() == 0
    check_attention(cache, q, table, length, got, lse)
    for _ in range(10):
        again, lse_again = attend(cache, q, table, length)
        same = torch.equal(got, again), torch.equal(lse, lse_again)
        assert same == (True, True)
