"""Cache append, paged attention and adapters, continued: rows, orders and values that the first file of tests does not meet.
Tolerances are those of test_decode_gpu.py where nothing else is said (u = 2^-23)."""
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(__file__))
import bolt_b200 as B  # noqa: E402
from test_decode_gpu import DT, U, Cache, attend, batch, check_attention, perm, rand, status  # noqa: E402

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


# ---- caches of bytes whose rows differ -------------------------------------------------------------------------------
def filled(i8, k, v, page):
    """a cache of one sequence made by kv_append; k, v: [tokens, heads, dim] in binary32"""
    n, kv, dim = k.shape
    cache = Cache(1, -(-n // page), page, kv, dim, i8)
    table = perm(2, cache.pages).int()[None, :].contiguous()
    rows = torch.cat((k.reshape(n, -1), v.reshape(n, -1)), 1).contiguous()
    seq, pos = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    p = rows.data_ptr()
    B.kv_append(cache.desc(), B.KvAppend(n, 0, B.DT_F32, B.DT_F32, None, p, p + 4 * kv * dim, None, 0, 2 * kv * dim, 2 * kv * dim, 0, seq.data_ptr(),
                                         pos.data_ptr(), table.data_ptr(), 1, table.shape[1], 0, 0, 0, None, None))
    return cache, table


@pytest.mark.parametrize("kv,group,dim", [(2, 4, 128), (1, 1, 64), (1, 8, 256), (1, 12, 128), (3, 2, 80)])
@pytest.mark.parametrize("small", [1e-2, 1e-4, 1e-6, 1e-8, 1e-20])
@pytest.mark.parametrize("heavy", ["zeros", "ones", "large"])
def test_attention_values_beside_a_heavy_row(kv, group, dim, small, heavy):
    """Rows of small values beside rows that weigh most, are zeros and therefore have scale 1, or weigh next to nothing and are
    large: the small ones keep their bits.  (ones: rows whose scale is 1, too, and that are no zeros count.)"""
    n, heads = 700, kv * group
    q = rand(3, 1, heads, dim)
    k, v = rand(4, n, kv, dim), small * rand(5, n, kv, dim)
    one = q[0].view(kv, group, dim).sum(1)
    one = 16 * group ** 0.5 * one / one.norm(dim=-1, keepdim=True)      # a key whose score is about 16 for all heads of the group
    spots = [0, 17, 300, 650, 699]
    for t in spots:
        k[t] = -2 * one if heavy == "large" else one
        v[t] = 0 if heavy == "zeros" else (127 * rand(6 + t, kv, dim).sign() if heavy == "ones" else rand(6 + t, kv, dim))
    length = torch.tensor([n], dtype=torch.int32, device="cuda")
    cache, table = filled(1, k, v, 16)
    if heavy != "large":
        assert bool((cache.vs[table[0, 1], :, 1] == 1).all())
    got, lse = attend(cache, q, table, length)
    assert status() == 0
    check_attention(cache, q, table, length, got, lse)
    if small < 1e-3:
        return                                                          # (below binary16)
    # A cache of binary16: a weight is two binary16 numbers in units in which a head's largest is 2^14, the second a multiple of
    # 2^-24 at worst: off by 2^-25, which is 2^-39 of the largest weight.
    cache, table = filled(0, k, v, 16)
    got, lse = attend(cache, q, table, length)
    check_one(cache, q, table, n, got, lse, weight=2.0 ** -39)


def check_one(cache, q, table, n, got, lse, query=0.0, weight=0.0):
    """check_attention of one sequence, and what a query is off by, of its head's largest element, and a weight, of the largest"""
    dim, group = q.shape[2], q.shape[1] // cache.heads
    kk, vv = (cache.rows(x, table[0], 0, n).repeat_interleave(group, 0) for x in "kv")
    scale = np.float32(dim ** -0.5).item()
    qq = q[0].double()
    s = torch.einsum("hd,htd->ht", qq, kk) * scale
    off = ((dim + 16) * U * torch.einsum("hd,htd->ht", qq.abs(), kk.abs()) + query * qq.abs().amax(-1)[:, None] * kk.abs().sum(-1)).amax(-1) * scale
    top = torch.logsumexp(s, -1)
    p = torch.exp(s - top[:, None])
    tol = 2 * (off[:, None] + (n / 16 + 72) * U) * torch.einsum("ht,htd->hd", p, vv.abs()) + n * 2.0 ** -126 * vv.abs().amax(1)
    tol += weight * p.amax(-1)[:, None] * vv.abs().sum(1)
    n_bad = int((~((got[0].double() - torch.einsum("ht,htd->hd", p, vv)).abs() <= tol)).sum())
    n_lse = int((~((lse[0].double() - top).abs() <= off + (n / 16 + 72) * U + 2 * U * top.abs())).sum())
    assert (n_bad, n_lse) == (0, 0)


@pytest.mark.parametrize("kv,group,dim", [(2, 4, 128), (1, 1, 64), (1, 12, 128), (1, 8, 256)])
@pytest.mark.parametrize("i8", [0, 1])
@pytest.mark.parametrize("ratio", [2.0 ** 8, 2.0 ** 15, 2.0 ** 20])
def test_attention_queries_of_different_magnitude(kv, group, dim, i8, ratio):
    """Heads in which some elements are by far the largest, where the keys are nothing (and the others decide) or alike.  Whole
    numbers for bytes are rounded to half a unit, 2^-30 of an element that has 2^29 units or more; the second of two binary16 numbers to
    2^-25 beside 2^13 or more, 2^-38."""
    n = 600
    for big in (0.0, 1.0 / ratio, 1.0):
        q = rand(3, 1, kv * group, dim)
        k, v = rand(4, n, kv, dim), rand(5, n, kv, dim)
        q[..., 3::40] *= ratio
        k[..., 3::40] *= big
        if big == 1:
            q *= 8 / ratio                                             # (scores of some 10)
        cache, table = filled(i8, k, v, 16)
        length = torch.tensor([n], dtype=torch.int32, device="cuda")
        got, lse = attend(cache, q, table, length)
        assert status() == 0
        check_one(cache, q, table, n, got, lse, query=2.0 ** -30 if i8 and group <= 8 else 2.0 ** -38)


# ---- what other tests would let through ------------------------------------------------------------------------------
@pytest.mark.parametrize("i8", [0, 1])
@pytest.mark.parametrize("sequences,longest", [(256, 70), (257, 70), (1025, 70), (5000, 40), (65535, 3)])
def test_attention_of_many_sequences_leaves_no_nan(i8, sequences, longest):
    """every number of every sequence, those without tokens among them, is one"""
    page, heads, dim = 8, 3, 32
    g = torch.Generator(device="cuda")
    g.manual_seed(sequences)
    length = torch.randint(0, longest + 1, (sequences,), device="cuda", generator=g, dtype=torch.int32)
    length[1::3] = 0
    tp = -(-longest // page)
    cache = Cache(1, 3000, page, 1, dim, i8)
    table = torch.randint(0, 3000, (sequences, tp), device="cuda", generator=g, dtype=torch.int32)
    table[torch.arange(tp, device="cuda")[None, :] * page >= length[:, None]] = -1
    q = rand(5, sequences, heads, dim)
    got, lse = attend(cache, q, table, length)
    assert status() == 0
    empty = length == 0
    assert bool((got[empty] == 0).all()) and bool((lse[empty] == -math.inf).all())
    assert bool(got.isfinite().all()) and bool(lse[~empty].isfinite().all())
    t = torch.arange(longest, device="cuda")
    pages, at = table.clamp(min=0).long()[:, t // page], (t % page)[None, :].expand(sequences, -1)
    k, v = (x[pages, 0, at].double() / (s[pages, 0, at].double()[..., None] if i8 else 1) for x, s in ((cache.k, cache.ks), (cache.v, cache.vs)))
    live = t[None, None, :] < length[:, None, None]
    scale = np.float32(dim ** -0.5).item()
    off = ((dim + 16) * U * scale * torch.einsum("bhd,btd->bht", q.double().abs(), k.abs()) * live).amax(-1)
    s = torch.where(live, torch.einsum("bhd,btd->bht", q.double(), k) * scale, -math.inf)
    top = torch.logsumexp(s, -1)
    p = torch.where(live, torch.exp(s - top[..., None]), 0.0)
    tol = 2 * (off[..., None] + (longest / 16 + 72) * U) * torch.einsum("bht,btd->bhd", p, v.abs()) + longest * 2.0 ** -126 * v.abs().amax()
    n_bad = int((~((got.double() - torch.einsum("bht,btd->bhd", p, v)).abs() <= tol)).sum())
    n_lse = int((~((lse.double() - top).abs() <= off + (longest / 16 + 72) * U + 2 * U * top.abs()))[~empty].sum())
    assert (n_bad, n_lse) == (0, 0)


@pytest.mark.parametrize("rows,n,k,rank,segments", [(64, 1000, 2048, 16, 64), (600, 700, 4096, 32, 3), (5, 768, 768, 8, 2), (40, 512, 28672, 128, 1)])
def test_lora_of_bytes_gives_the_same_bits_again(rows, n, k, rank, segments):
    g = torch.Generator(device="cuda")
    g.manual_seed(rows)
    x = torch.randint(0, 256, (rows, k), device="cuda", generator=g, dtype=torch.uint8)
    a, b, y = rand(1, segments, rank, k, dtype=torch.float16), rand(2, segments, n, rank, dtype=torch.float16), rand(3, rows, n)
    scale, row_scale = rand(4, segments), 20 + torch.rand(rows, device="cuda", generator=g)
    first = torch.tensor([rows * i // segments for i in range(segments + 1)], dtype=torch.int32, device="cuda")
    adapter = torch.arange(segments, dtype=torch.int32, device="cuda")
    results = []
    for fill in (0, 0xFF, 0x5A):
        out = y.clone()
        call = B.Lora(rows, n, k, rank, segments, segments, B.DT_U8_Q, x.data_ptr(), out.data_ptr(), k, n, a.data_ptr(), b.data_ptr(), k, scale.data_ptr(),
                      first.data_ptr(), adapter.data_ptr(), 1.0, None, row_scale.data_ptr())
        nb = B.lora_tmp_bytes(call)
        tmp = torch.full((nb,), fill, dtype=torch.uint8, device="cuda")
        B.lora(call, nb, tmp.data_ptr())
        assert status() == 0
        results.append(out)
    assert not torch.equal(results[0], y)
    same = [torch.equal(r, results[0]) for r in results]
    assert same == [True] * 3


@pytest.mark.parametrize("heads,n", [(8, 96), (32, 96), (8, 30000)])
@pytest.mark.parametrize("out", [torch.uint8, torch.float32])
def test_results_that_the_next_call_reads(heads, n, out):
    """Attention into x of the adapters, whose first kernel starts beside the end of attention's last, over and over into the same
    arrays, and a page table that a copy in front has written: the bits of calls that wait for one another."""
    seqs, kv, dim, rank = 6, 2, 64, 16
    cache, _, table, length = batch(5, [900, 33, 1, 517, 0, 64], (16, kv, dim, 0, "hnd", 0), heads)
    tables = [table.clone(), table.clone()]
    tables[1][0, :40] = table[0, :40].flip(0)
    qs = [rand(s, seqs, heads * dim) for s in range(6)]
    a, b = rand(1, 2, rank, heads * dim, dtype=torch.float16, scale=0.1), rand(2, 2, n, rank, dtype=torch.float16)
    first, adapter = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 2, 6], [1, 0]))
    q, x, y = torch.empty_like(qs[0]), torch.empty(seqs, heads * dim, dtype=out, device="cuda"), torch.zeros(seqs, n, device="cuda")
    tmp = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    attention = B.PagedAttention(seqs, heads, B.DT_F32, DT[out], q.data_ptr(), x.data_ptr(), None, heads * dim, heads * dim, table.data_ptr(), length.data_ptr(),
                                 table.shape[1], 0, 0.125, 60.0)
    lora = B.Lora(seqs, n, heads * dim, rank, 2, 2, DT[out], x.data_ptr(), y.data_ptr(), heads * dim, n, a.data_ptr(), b.data_ptr(), heads * dim, None,
                  first.data_ptr(), adapter.data_ptr(), 60.0, None, None)

    def steps(wait):
        kept = []
        y.zero_()
        for i in range(24):
            q.copy_(qs[i % 6])
            table.copy_(tables[i % 2])
            for call in (lambda: B.paged_attention(cache.desc(), attention, tmp.numel(), tmp.data_ptr()), lambda: B.lora(lora, tmp.numel(), tmp.data_ptr())):
                call()
                if wait:
                    torch.cuda.synchronize()
            kept.append(y.clone())
        assert status() == 0
        return kept

    want = steps(True)
    for _ in range(3):
        same = [torch.equal(u, v) for u, v in zip(steps(False), want)]
        assert same == [True] * 24
