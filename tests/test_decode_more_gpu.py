"""Cache append, paged attention and adapters, continued: rows, orders and values that the first file of tests does not meet.
Tolerances are those of test_decode_gpu.py where nothing else is said (u = 2^-23)."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(__file__))
import bolt_b200 as B  # noqa: E402
from test_decode_gpu import DT, U, attend, batch, check_attention, status  # noqa: E402

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


# ---- sums that do not drift ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("x_dt", [torch.float32, torch.uint8])
@pytest.mark.parametrize("rows,n,k,rank", [(1, 768, 768, 8), (16, 768, 768, 16), (16, 1024, 1024, 32), (16, 1024, 4096, 16), (64, 512, 8192, 8),
                                           (64, 512, 4096, 24), (64, 512, 4096, 64), (64, 512, 4096, 128), (300, 515, 1001, 40)])
def test_lora_sums_of_one_sign(x_dt, rows, n, k, rank):
    """Positive x, A and B: what is cut off, and not rounded, adds up.  A result may be too small by this much on the average: t,
    u / 2 for each of the two instructions that go into one register before the sum is rounded to nearest, u; the outer sum, u / 2
    (1/4 + 2/4 + 3/4 + 1) for four of them, 5/4 u; what is rounded to nearest (x, t, the sums, y) has no share in a mean but for
    its noise: 3 u together."""
    g = torch.Generator(device="cuda")
    g.manual_seed(k + rank + rows)
    pos = lambda *s: 0.5 + 0.5 * torch.rand(s, device="cuda", generator=g)  # noqa: E731
    ka = (k + 7) // 8 * 8
    a, b = (pos(1, rank, ka) * k ** -0.5).half(), (pos(1, n, rank) * rank ** -0.5).half()
    if x_dt == torch.float32:
        x = pos(rows, k)
        exact = x.double()
    else:
        x = torch.randint(129, 256, (rows, k), device="cuda", generator=g, dtype=torch.uint8)
        exact = (x.double() - 128) / 32.0
    y = torch.zeros(rows, n, device="cuda")
    first, adapter = torch.tensor([0, rows], dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    call = B.Lora(rows, n, k, rank, 1, 1, DT[x_dt], x.data_ptr(), y.data_ptr(), k, n, a.data_ptr(), b.data_ptr(), ka, None, first.data_ptr(),
                  adapter.data_ptr(), 32.0, None, None)
    nb = B.lora_tmp_bytes(call)
    tmp = torch.empty(nb, dtype=torch.uint8, device="cuda")
    B.lora(call, nb, tmp.data_ptr())
    assert status() == 0
    want = (exact @ a[0, :, :k].double().T) @ b[0].double().T
    mean = float(((y.double() - want) / want).mean()) / U
    assert abs(mean) <= 3, mean
