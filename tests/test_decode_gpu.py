"""Cache append, paged attention and adapters against plain 64-bit computations, at the sizes and masks where they can go wrong.

Tolerances (u = 2^-23, twice the unit roundoff of binary32, which also covers sums that truncate):
  append     every step is one binary32 operation of defined order: equal bits.
  attention  a score of dim products is off by at most (dim + 16) u sum |q_i k_i| scale (products, sums, 22-bit operands, the
             multiplication with the scale; a cache of bytes may round queries at 2^-30 of a head's largest element instead,
             which is less for the noise that is used here); its exponential by that much relative, plus 8 u; the sum over n tokens adds
             16 at a time: (n / 16 + 64) u sum p |v|.  Numerator and denominator together: twice that.  Exponentials below
             2^-126, the smallest normal number, may count as nothing: n 2^-126 max |v|.
  lora       inner sums: (K / 16 + 40) u sum |x a|; outer: (rank / 16 + 40) u sum |t b|; y itself: 2 u |y|.
A result in binary16 is rounded once more (half of torch.finfo.eps, 2^-25 below the normal numbers), one in bytes by 1/2.
"""
import ctypes as C
import math
import os
import sys

import numpy as np
import pytest
import torch

sys.path.insert(0, os.path.dirname(__file__))
import bolt_b200 as B  # noqa: E402

pytestmark = pytest.mark.gpu
U = 2.0 ** -23
DT = {torch.float32: B.DT_F32, torch.float16: B.DT_F16, torch.int8: B.DT_I8, torch.uint8: B.DT_U8_Q}


def rand(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (scale * torch.randn(shape, device="cuda", generator=g)).to(dtype)


def perm(seed, n):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randperm(n, device="cuda", generator=g)


def ptr(t):
    return None if t is None else t.data_ptr()


def status():
    torch.cuda.synchronize()
    return B.lib().bolt_b200_device_status()


class Cache:
    """pages of finite noise; `poison`: what lies between rows and (later) behind the sequences"""

    def __init__(self, seed, pages, page, heads, dim, i8, order="hnd", gap=0):
        dt = torch.int8 if i8 else torch.float16
        shape = (pages, heads, page, dim + gap) if order == "hnd" else (pages, page, heads, dim + gap)
        make = (lambda s: torch.randint(-127, 128, shape, device="cuda", dtype=torch.int8)) if i8 else (lambda s: rand(s, *shape, dtype=dt))
        torch.manual_seed(seed)
        self.k_all, self.v_all = make(seed), make(seed + 1)
        if gap and not i8:
            self.k_all[..., dim:] = self.v_all[..., dim:] = math.nan
        self.k, self.v = self.k_all[..., :dim], self.v_all[..., :dim]
        self.i8, self.order, self.page, self.heads, self.dim, self.pages = i8, order, page, heads, dim, pages
        self.ks = self.vs = None
        if i8:
            self.ks, self.vs = (20 + 100 * torch.rand((pages, heads, page), device="cuda") for _ in range(2))

    def desc(self):
        s = self.k.stride()
        token, head = (s[2], s[1]) if self.order == "hnd" else (s[1], s[2])
        return B.KvCache(B.DT_I8 if self.i8 else B.DT_F16, self.pages, self.page, self.heads, self.dim, s[0], token, head,
                         ptr(self.k), ptr(self.v), ptr(self.ks), ptr(self.vs))

    def rows(self, which, table_row, begin, end):
        """[heads, tokens, dim] in 64 bits"""
        t = torch.arange(begin, end, device="cuda")
        page, at = table_row[t // self.page].long(), t % self.page
        x, s = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        r = (x[page, :, at] if self.order == "hnd" else x[page, at]).double()
        if self.i8:
            r = r / s[page, :, at].double()[..., None]
        return r.transpose(0, 1)


# ---- append --------------------------------------------------------------------------------------------------------
def turned(x, pos, cos, sin, rotary, interleaved):
    """x [rows, heads, dim], numpy binary32 operations one by one"""
    x = x.astype(np.float32)
    if rotary == 0:
        return x
    c, s = cos[pos][:, None, :], sin[pos][:, None, :]
    y = x.copy()
    ia, ib = (np.arange(0, rotary, 2), np.arange(1, rotary, 2)) if interleaved else (np.arange(rotary // 2), np.arange(rotary // 2, rotary))
    a, b = x[..., ia], x[..., ib]
    y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
    return y


def quantized(rows):
    top = np.abs(rows).max(-1)
    with np.errstate(divide="ignore"):
        s = np.where(top == 0, np.float32(1), np.float32(127) / top).astype(np.float32)
    return np.clip(np.rint(rows * s[..., None]), -127, 127).astype(np.int8), s


def append_case(tokens, heads, kv, dim, i8, page, order, dt, rotary, interleaved, gap=0, offset=0, in_place=False, with_seq=True, pad=True, q_out=None, pad_every=0):
    seqs, tp = 3, 6
    cap = tp * page
    tokens = min(tokens, seqs * cap)
    cache = Cache(7, seqs * tp + 1, page, kv, dim, i8, order, gap)
    table = perm(3, seqs * tp + 1)[: seqs * tp].int().view(seqs, tp).contiguous()
    place = perm(5, seqs * cap)[:tokens]
    if not with_seq:
        tokens = min(tokens, seqs)
        place = torch.arange(tokens, device="cuda") * cap + perm(6, cap)[:1]
    seq, pos = (place // cap).int(), (place % cap).int()
    if pad and tokens > 2:
        pos[1] = -1
    if pad_every:
        pos[::pad_every] = -1
    width = (heads + 2 * kv) * dim + offset
    qkv = rand(11, tokens, width, dtype=dt)[:, offset:]
    qkv[0, heads * dim: (heads + 1) * dim] = 0                      # a row of zeros has scale 1
    width = qkv.stride(0)
    cos, sin = (rand(s, cap, max(rotary // 2, 1)).contiguous() for s in (21, 22))
    before_k, before_v = cache.k_all.clone(), cache.v_all.clone()
    before_s = [x.clone() for x in (cache.ks, cache.vs)] if i8 else []
    src = qkv.clone()
    qo = qkv if in_place else torch.full((tokens, heads * dim), 9.0, dtype=q_out or dt, device="cuda")
    p, e = qkv.data_ptr(), qkv.element_size()
    call = B.KvAppend(tokens, heads, DT[dt], DT[qo.dtype], p, p + heads * dim * e, p + (heads + kv) * dim * e, qo.data_ptr(), width, width, width,
                      qo.stride(0), seq.data_ptr() if with_seq else None, pos.data_ptr(), table.data_ptr(), seqs, tp, rotary, interleaved,
                      cap if rotary else 0, ptr(cos) if rotary else None, ptr(sin) if rotary else None)
    B.kv_append(cache.desc(), call)
    assert status() == 0
    # what it has to be
    live = (pos >= 0).cpu().numpy()
    ps, sq = pos.cpu().numpy(), seq.cpu().numpy()
    x = src.cpu().numpy().reshape(tokens, heads + 2 * kv, dim)
    y = turned(x, np.maximum(ps, 0), cos.cpu().numpy(), sin.cpu().numpy(), rotary, interleaved)
    want_q = src.cpu().numpy()[:, : heads * dim].copy() if in_place else np.full((tokens, heads * dim), 9.0, np.float32)
    want_q[live] = y[live, :heads].reshape(int(live.sum()), heads * dim)
    got_q = qo.cpu()[:, : heads * dim]
    assert torch.equal(got_q, torch.from_numpy(want_q).to(got_q.dtype))
    if in_place:
        assert torch.equal(qo.cpu()[:, heads * dim:], src.cpu()[:, heads * dim:])
    tab = table.cpu().numpy()
    page_i, at = tab[sq[live], ps[live] // page], ps[live] % page
    for got, before, rows, scales, sb in ((cache.k_all, before_k, y[live, heads: heads + kv], cache.ks, before_s[:1]),
                                          (cache.v_all, before_v, x[live, heads + kv:].astype(np.float32), cache.vs, before_s[1:])):
        want, got = before.cpu().numpy().copy(), got.cpu().numpy()
        if i8:
            rows, s = quantized(rows)
            ws = sb[0].cpu().numpy().copy()
            ws[page_i, :, at] = s
            assert ws.tobytes() == scales.cpu().numpy().tobytes()
        if order == "hnd":
            want[page_i, :, at, :dim] = rows
        else:
            want[page_i, at, :, :dim] = rows
        assert want.tobytes() == got.tobytes()


@pytest.mark.parametrize("heads,kv,dim", [(1, 1, 16), (12, 12, 64), (8, 2, 128), (5, 1, 256), (4, 4, 80), (3, 3, 48), (0, 2, 192), (6, 2, 96)])
@pytest.mark.parametrize("i8", [0, 1])
@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
@pytest.mark.parametrize("order,page,tokens", [("hnd", 16, 40), ("nhd", 7, 100), ("hnd", 1, 5), ("nhd", 33, 1)])
def test_append(heads, kv, dim, i8, dt, order, page, tokens):
    for rotary, interleaved in ((dim, 0), (dim, 1), (0, 0), (dim // 2, 0)):
        append_case(tokens, heads, kv, dim, i8, page, order, dt, rotary, interleaved)


@pytest.mark.parametrize("i8", [0, 1])
@pytest.mark.parametrize("interleaved", [0, 1])
def test_append_off_the_grid(i8, interleaved):
    """halves that are no multiple of four, rows at odd addresses, gaps between the cache's rows, queries in place and in another type"""
    for rotary in (2, 6, 10, 36):
        append_case(9, 4, 2, 48, i8, 5, "hnd", torch.float32, rotary, interleaved)
    for offset in (1, 2, 3):
        append_case(9, 4, 2, 64, i8, 5, "nhd", torch.float16, 64, interleaved, offset=offset)
        append_case(9, 4, 2, 256, i8, 5, "hnd", torch.float32, 256, interleaved, offset=offset)
    append_case(9, 4, 2, 64, i8, 5, "nhd", torch.float32, 32, interleaved, gap=16)
    append_case(9, 4, 2, 128, i8, 5, "hnd", torch.float32, 128, interleaved, in_place=True)
    append_case(9, 4, 2, 128, i8, 5, "hnd", torch.float16, 64, interleaved, in_place=True, offset=1)
    append_case(9, 4, 2, 128, i8, 5, "hnd", torch.float32, 64, interleaved, q_out=torch.float16)
    append_case(9, 4, 2, 128, i8, 5, "hnd", torch.float16, 64, interleaved, q_out=torch.float32)
    append_case(3, 4, 2, 128, i8, 5, "hnd", torch.float16, 64, interleaved, with_seq=False, pad=False)


@pytest.mark.parametrize("heads,kv,dim", [(12, 2, 64), (8, 2, 128), (5, 1, 256), (7, 3, 80), (0, 9, 192), (33, 5, 48)])
@pytest.mark.parametrize("i8", [0, 1])
@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
def test_append_of_prompts(heads, kv, dim, i8, dt):
    """more rows than run at a time: every group of lanes goes through several tokens, some of them padding"""
    for tokens, rotary, interleaved, in_place in ((3601, dim, 0, False), (5000, dim // 2, 1, True), (4999, 0, 0, False)):
        append_case(tokens, heads, kv, dim, i8, 300, "hnd" if in_place else "nhd", dt, rotary, interleaved, in_place=in_place, pad_every=7)


def test_append_refuses_on_the_device_what_leads_outside():
    """sequence, position, page and angle out of range: nothing is written for these tokens, the others are done"""
    cache = Cache(1, 4, 8, 2, 64, 0)
    table = torch.tensor([[0, 1], [2, 99], [-5, 3]], dtype=torch.int32, device="cuda")
    #      good  sequence sequence position page -5   page 99  angle   good
    seq = torch.tensor([0, 3, -1, 0, 2, 1, 0, 2], dtype=torch.int32, device="cuda")
    pos = torch.tensor([3, 0, 0, 16, 1, 9, 15, 8], dtype=torch.int32, device="cuda")
    kv = rand(1, 8, 4 * 64, dtype=torch.float16)
    cos, sin = rand(2, 15, 32), rand(3, 15, 32)
    before = cache.k.clone(), cache.v.clone()
    q = torch.full((8, 64), 5.0, device="cuda", dtype=torch.float16)
    call = B.KvAppend(8, 1, B.DT_F16, B.DT_F16, kv.data_ptr(), kv.data_ptr(), kv.data_ptr() + 256, q.data_ptr(), 256, 256, 256, 64, seq.data_ptr(),
                      pos.data_ptr(), table.data_ptr(), 3, 2, 64, 0, 15, cos.data_ptr(), sin.data_ptr())
    B.kv_append(cache.desc(), call)
    assert B.lib().bolt_b200_synchronize() == B.UNKNOWN
    changed = [(cache.k != before[0]).any(-1).any(1), (cache.v != before[1]).any(-1).any(1)]     # [page, token]
    want = torch.zeros((4, 8), dtype=torch.bool, device="cuda")
    want[0, 3] = want[3, 0] = True
    assert torch.equal(changed[0], want) and torch.equal(changed[1], want)
    assert ((q != 5).any(1)).tolist() == [True] + [False] * 6 + [True]
    assert status() == 0


# ---- attention ---------------------------------------------------------------------------------------------------
def attend(cache, q, table, length, window=0, scale=None, out=torch.float32, out_scale=1.0, lse=True, q_stride=None, out_gap=0):
    """one call; (out [sequences, heads, dim], lse)"""
    b, h, d = q.shape
    o_all = torch.full((b, h * d + out_gap), 77, dtype=out, device="cuda")
    l = torch.full((b, h), 5.0, device="cuda") if lse else None
    call = B.PagedAttention(b, h, DT[q.dtype], DT[out], q.data_ptr(), o_all.data_ptr(), ptr(l), q.stride(0), o_all.stride(0), table.data_ptr(),
                            length.data_ptr(), table.shape[1], window, scale if scale is not None else d ** -0.5, out_scale)
    n = B.paged_attention_tmp_bytes(cache.desc(), call)
    tmp = torch.full((n + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    B.paged_attention(cache.desc(), call, n, tmp.data_ptr())
    if out_gap:
        assert bool((o_all[:, h * d:] == 77).all())
    assert bool((tmp[n:] == 0xA5).all())
    return o_all[:, : h * d].view(b, h, d) if not out_gap else o_all[:, : h * d].reshape(b, h, d), l


def check_attention(cache, q, table, length, got, lse, window=0, scale=None, out_scale=None):
    b, h, d = q.shape
    scale = np.float32(scale if scale is not None else d ** -0.5).item()
    group = h // cache.heads
    for i, end in enumerate(length.tolist()):
        begin = max(0, end - window) if window else 0
        if end == 0:
            want, tol = torch.zeros((h, d), device="cuda", dtype=torch.float64), torch.zeros((h, d), device="cuda", dtype=torch.float64)
            if lse is not None:
                assert bool((lse[i] == -math.inf).all())
        else:
            k, v = (cache.rows(x, table[i], begin, end).repeat_interleave(group, 0) for x in "kv")
            qq = q[i].double()
            s = torch.einsum("hd,htd->ht", qq, k) * scale
            off = ((d + 16) * U * abs(scale) * torch.einsum("hd,htd->ht", qq.abs(), k.abs())).amax(-1)     # of a score
            top = torch.logsumexp(s, -1)
            p = torch.exp(s - top[:, None])
            want = torch.einsum("ht,htd->hd", p, v)
            n = end - begin
            tol = 2 * (off[:, None] + (n / 16 + 72) * U) * torch.einsum("ht,htd->hd", p, v.abs()) + n * 2.0 ** -126 * v.abs().amax(1)
            if lse is not None:
                assert bool(((lse[i].double() - top).abs() <= off + (n / 16 + 72) * U + 2 * U * top.abs()).all()), (i, end)
        g = got[i].double()
        if got.dtype == torch.float16:
            tol = tol + want.abs() * 2.0 ** -11 + 2.0 ** -25
        if got.dtype == torch.uint8:
            want, tol = (want * out_scale).clamp(-127, 127) + 128, tol * out_scale + 0.5
        bad = ~((g - want).abs() <= tol * (1 + 1e-9))
        n_bad = int(bad.sum())
        assert n_bad == 0, (i, end, n_bad, float((g - want).abs()[bad].max()), float(tol[bad].min()))


def batch(seed, lens, cache_args, heads, q_dt=torch.float32, q_scale=1.0, poison=True):
    """cache, queries, table and lengths of a batch; what the pages hold behind a sequence is poison"""
    page, kv, dim, i8, order, gap = cache_args
    tp = max(1, max(-(-n // page) for n in lens))
    need = [-(-n // page) for n in lens]
    cache = Cache(seed, sum(need) + 1, page, kv, dim, i8, order, gap)
    order_ = perm(seed, sum(need) + 1)
    table = torch.full((len(lens), tp), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order_[at: at + n].int()
        at += n
        if poison and lens[i] % page:
            last, tail = int(table[i, n - 1]), lens[i] % page
            for x in (cache.k, cache.v):
                dst = x[last, :, tail:] if order == "hnd" else x[last, tail:]
                dst.fill_(127 if i8 else math.nan)
            if i8:
                cache.ks[last, :, tail:] = 0.0
                cache.vs[last, :, tail:] = math.nan
    q = rand(seed + 9, len(lens), heads, dim, dtype=q_dt, scale=q_scale)
    return cache, q, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


LENS = [0, 1, 2, 15, 16, 17, 31, 33, 64, 127, 128, 129, 255, 257, 300, 0, 513, 1025]


@pytest.mark.parametrize("dim", [8, 16, 32, 48, 64, 80, 96, 112, 128, 144, 192, 256])
@pytest.mark.parametrize("kv,group", [(1, 1), (2, 2), (1, 5), (3, 8), (2, 9), (1, 16), (1, 20), (1, 40)])
@pytest.mark.parametrize("i8", [0, 1])
def test_attention_heads(dim, kv, group, i8):
    if i8 and dim % 16:
        pytest.skip("rows of a cache of bytes are multiples of 16")
    page, order = ((16, "hnd"), (5, "nhd"), (100, "hnd"))[(dim // 8 + group) % 3]
    lens = LENS[(dim + group) % 5::2] + [700]
    cache, q, table, length = batch(dim + group, lens, (page, kv, dim, i8, order, 0), kv * group, (torch.float32, torch.float16)[group % 2])
    got, lse = attend(cache, q, table, length)
    assert status() == 0
    check_attention(cache, q, table, length, got, lse)


@pytest.mark.parametrize("page", [1, 3, 16, 24, 64, 1000])
@pytest.mark.parametrize("order,gap", [("hnd", 0), ("nhd", 0), ("nhd", 16)])
@pytest.mark.parametrize("i8", [0, 1])
@pytest.mark.parametrize("out", [torch.float32, torch.float16, torch.uint8])
def test_attention_pages_and_outputs(page, order, gap, i8, out):
    cache, q, table, length = batch(page, LENS + [2000], (page, 2, 64, i8, order, gap), 8)
    for window in (0, 1, 20, 300, 5000):
        got, lse = attend(cache, q, table, length, window=window, out=out, out_scale=100.0, lse=window != 20, out_gap=window % 3)
        assert status() == 0
        check_attention(cache, q, table, length, got, lse, window, out_scale=100.0)


@pytest.mark.parametrize("i8", [0, 1])
@pytest.mark.parametrize("lens", [[40000], [30000, 5, 1, 0, 17000], [257] * 70, [3] * 700, [0, 0, 0], [0], [1], [1025] * 149])
def test_attention_splits(i8, lens):
    """few long sequences, many short ones, none with a token"""
    cache, q, table, length = batch(4, lens, (16, 2, 128, i8, "hnd", 0), 16)
    got, lse = attend(cache, q, table, length)
    again, _ = attend(cache, q, table, length)
    assert status() == 0
    check_attention(cache, q, table, length, got, lse)
    assert torch.equal(got, again)          # no order of arrival in the result


@pytest.mark.parametrize("i8", [0, 1])
def test_attention_values(i8):
    """peaked softmax, large and small queries, one value far above the rest, negative scales, equal scores"""
    for q_scale, scale in ((1e-6, None), (30.0, None), (1e5, 1e-6), (1e-30, 1e29), (1.0, -0.5), (1.0, 0.0)):
        cache, q, table, length = batch(8, [900, 1, 77], (16, 2, 64, i8, "hnd", 0), 8, q_scale=q_scale)
        got, lse = attend(cache, q, table, length, scale=scale)
        check_attention(cache, q, table, length, got, lse, scale=scale)
    cache, q, table, length = batch(9, [900, 1, 77], (16, 2, 64, i8, "hnd", 0), 8)
    if i8:
        cache.vs *= torch.pow(10.0, -6 + 9 * torch.rand_like(cache.vs))       # rows of very different magnitude
        cache.vs[int(table[0, 3]), :, 5] = 1e-3
    else:
        cache.v *= 1e-3
        cache.v[int(table[0, 3]), :, 5] = 60000.0
        cache.k[int(table[0, 0]), :, 0] = 200.0 * q[0, 0].sign().half()
    got, lse = attend(cache, q, table, length)
    check_attention(cache, q, table, length, got, lse)


@pytest.mark.parametrize("group", [2, 12])
def test_attention_rows_that_are_not_finite_stay_with_their_sequence(group):
    """live rows have to be finite; where one is not, the other sequences and key heads are as they would be"""
    for bad in (math.nan, math.inf, -math.inf):
        cache, q, table, length = batch(3, [700, 90, 300, 900], (16, 2, 64, 0, "hnd", 0), 2 * group)
        cache.k[int(table[1, 2]), 0, 5] = bad
        cache.v[int(table[3, 20]), 1, 7] = bad
        got, lse = attend(cache, q, table, length)
        cache.k[int(table[1, 2]), 0, 5] = 0
        cache.v[int(table[3, 20]), 1, 7] = 0
        clean, clean_lse = attend(cache, q, table, length)
        got[1, :group], lse[1, :group], got[3, group:] = clean[1, :group], clean_lse[1, :group], clean[3, group:]
        same = torch.equal(got, clean), torch.equal(lse, clean_lse)
        assert same == (True, True)


@pytest.mark.parametrize("i8", [0, 1])
@pytest.mark.parametrize("group", [2, 12])
def test_attention_queries_that_are_not_finite_stay_with_their_head(i8, group):
    for bad in (math.nan, math.inf, -math.inf):
        cache, q, table, length = batch(4, [700, 33], (16, 2, 64, i8, "hnd", 0), 2 * group)
        clean, clean_lse = attend(cache, q, table, length)
        q[0, 1, 5] = q[1, group, 63] = bad
        got, lse = attend(cache, q, table, length)
        for i, h in ((0, 1), (1, group)):
            assert bool(got[i, h].isnan().all()) and bool(lse[i, h].isnan())
            got[i, h], lse[i, h] = clean[i, h], clean_lse[i, h]
        same = torch.equal(got, clean), torch.equal(lse, clean_lse)
        assert same == (True, True)


def test_attention_refuses_on_the_device_what_leads_outside():
    """a page outside the cache is left out, a length beyond the table is cut, a negative one is none"""
    cache, q, table, length = batch(2, [100, 100, 100, 64], (16, 2, 64, 0, "hnd", 0), 4)
    good = table.clone()
    table[0, 2], table[1, 0] = cache.pages, -7
    length[2], length[3] = 1 << 30, -1
    table[2] = table[0, 3]
    got, _ = attend(cache, q, table, length)
    assert B.lib().bolt_b200_synchronize() == B.UNKNOWN
    for i, lost in ((0, range(32, 48)), (1, range(16))):
        keep = torch.tensor([t for t in range(100) if t not in lost], device="cuda")
        k, v = (cache.rows(x, good[i], 0, 100)[:, keep].repeat_interleave(2, 0) for x in "kv")
        want = torch.softmax(torch.einsum("hd,htd->ht", q[i].double(), k) / 8, -1)
        assert float((got[i].double() - torch.einsum("ht,htd->hd", want, v)).abs().max()) < 1e-4
    assert bool((got[3] == 0).all())
    attend(cache, q, good, torch.tensor([100, 100, 100, 64], dtype=torch.int32, device="cuda"))
    length.fill_(10)
    attend(cache, q, good, length)
    assert status() == 0


def test_attention_far_into_a_large_cache():
    """rows behind 2^32 bytes and 2^31 elements"""
    pages, page, kv, dim = 70000, 64, 4, 128                       # 2.3 G elements, 4.6 GB per cache
    cache = Cache.__new__(Cache)
    cache.k_all = cache.k = torch.empty((pages, kv, page, dim), dtype=torch.float16, device="cuda")
    cache.v_all = cache.v = torch.empty((pages, kv, page, dim), dtype=torch.float16, device="cuda")
    cache.i8, cache.order, cache.page, cache.heads, cache.dim, cache.pages, cache.ks, cache.vs = 0, "hnd", page, kv, dim, pages, None, None
    table = torch.tensor([[pages - 1, 0, pages - 2, 65536]], dtype=torch.int32, device="cuda")
    for x, s in ((cache.k, 1), (cache.v, 2)):
        x[table[0].long()] = rand(s, 4, kv, page, dim, dtype=torch.float16)
    row = rand(5, 1, 3 * kv * dim)
    pos, zero = torch.tensor([63], dtype=torch.int32, device="cuda"), None
    call = B.KvAppend(1, kv, B.DT_F32, B.DT_F32, row.data_ptr(), row.data_ptr() + 4 * kv * dim, row.data_ptr() + 8 * kv * dim, row.data_ptr(),
                      3 * kv * dim, 3 * kv * dim, 3 * kv * dim, 3 * kv * dim, zero, pos.data_ptr(), table.data_ptr(), 1, 4, 0, 0, 0, None, None)
    B.kv_append(cache.desc(), call)
    assert torch.equal(cache.k[pages - 1, :, 63].reshape(-1), row[0, kv * dim: 2 * kv * dim].half())
    q, length = rand(6, 1, 8, dim), torch.tensor([250], dtype=torch.int32, device="cuda")
    got, lse = attend(cache, q, table, length)
    check_attention(cache, q, table, length, got, lse)
    assert status() == 0


def test_attention_in_a_graph_follows_lengths_and_tables():
    """captured once, replayed for other lengths; two graphs with a workspace each on two streams"""
    works = []
    for s in (1, 2):
        cache, q, table, length = batch(s, [600, 900, 3], (16, 2, 128, s - 1, "hnd", 0), 8, poison=False)
        out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
        call = B.PagedAttention(3, 8, B.DT_F32, B.DT_F32, q.data_ptr(), out.data_ptr(), lse.data_ptr(), q.stride(0), out.stride(0), table.data_ptr(),
                                length.data_ptr(), table.shape[1], 0, 128 ** -0.5, 0.0)
        n = B.paged_attention_tmp_bytes(cache.desc(), call)
        tmp = torch.empty(n + 16, dtype=torch.uint8, device="cuda")
        B.paged_attention(cache.desc(), call, n, tmp.data_ptr())
        torch.cuda.synchronize()
        stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            B.lib().bolt_b200_set_stream(C.c_void_p(torch.cuda.current_stream().cuda_stream))
            B.paged_attention(cache.desc(), call, n, tmp.data_ptr())
            B.lib().bolt_b200_set_stream(None)
        works.append((cache, q, table, length, out, lse, stream, graph, tmp))
    for lens in ([600, 900, 3], [1, 0, 3], [256, 17, 2], [0, 0, 0], [599, 900, 1]):
        for w in works:
            w[3].copy_(torch.tensor(lens, dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(5):
            for w in works:
                with torch.cuda.stream(w[6]):
                    w[7].replay()
        torch.cuda.synchronize()
        for cache, q, table, length, out, lse, *_ in works:
            check_attention(cache, q, table, length, out, lse)
    assert status() == 0


# ---- adapters ------------------------------------------------------------------------------------------------------
def lora_case(rows, n, k, rank, bounds, adapters, x_dt, seed=1, which=None, scale=True, unit="row", x_gap=0, y_gap=0, x_off=0, y_off=0, a_gap=0, values=1.0):
    seg = len(bounds) - 1
    which = which or [i % adapters for i in range(seg)]
    first, adapter = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in (bounds, which))
    if x_dt == torch.uint8:
        x_all = torch.randint(0, 256, (rows, k + x_gap + x_off), device="cuda", dtype=torch.uint8)
    else:
        x_all = rand(seed, rows, k + x_gap + x_off, scale=values)
        x_all[:, :x_off] = x_all[:, x_off + k:] = math.nan
    x = x_all[:, x_off: x_off + k]
    y_all = rand(seed + 1, rows, n + y_gap + y_off)
    y = y_all[:, y_off: y_off + n]
    a_all = rand(seed + 2, adapters, rank, (k + 7) // 8 * 8 + a_gap, dtype=torch.float16, scale=k ** -0.5)
    a_all[:, :, k:] = math.nan
    b = rand(seed + 3, adapters, n, rank, dtype=torch.float16, scale=rank ** -0.5)
    s = 0.5 + torch.rand(adapters, device="cuda") if scale else None
    row_scale = 10 + 50 * torch.rand(rows, device="cuda") if unit == "row" else None
    d_sA = torch.full((1,), 33.0, device="cuda") if unit == "device" else None
    before = y_all.clone()
    call = B.Lora(rows, n, k, rank, adapters, seg, DT[x_dt], x.data_ptr(), y.data_ptr(), x.stride(0), y.stride(0), a_all.data_ptr(), b.data_ptr(),
                  a_all.shape[2], ptr(s), first.data_ptr(), adapter.data_ptr(), 21.0, ptr(d_sA), ptr(row_scale))
    nb = B.lora_tmp_bytes(call)
    tmp = torch.full((nb + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    B.lora(call, nb, tmp.data_ptr())
    torch.cuda.synchronize()
    assert bool((tmp[nb:] == 0xA5).all())
    want, tol = before.double(), torch.zeros_like(before, dtype=torch.float64)
    wy, ty = want[:, y_off: y_off + n], tol[:, y_off: y_off + n]
    for i, ad in enumerate(which):
        if ad < 0 or ad >= adapters or not max(0, *bounds[:i + 1]) <= bounds[i] <= bounds[i + 1] <= rows:
            continue
        r = slice(bounds[i], bounds[i + 1])
        xx = x[r].double()
        if x_dt == torch.uint8:
            xx = (xx - 128) / (row_scale[r].double()[:, None] if unit == "row" else (33.0 if unit == "device" else 21.0))
        aa, bb, ss = a_all[ad, :, :k].double(), b[ad].double(), float(s[ad]) if scale else 1.0
        t, dt = xx @ aa.T, (k / 16 + 40) * U * (xx.abs() @ aa.abs().T)
        add = ss * (t @ bb.T)
        ty[r] = ss * (dt @ bb.abs().T + (rank / 16 + 40) * U * (t.abs() @ bb.abs().T)) + 2 * U * (wy[r].abs() + add.abs())
        wy[r] += add
    bad = ~((y_all.double() - want).abs() <= tol)
    n_bad = int(bad.sum())
    assert n_bad == 0, (rows, n, k, rank, n_bad, float((y_all.double() - want).abs()[bad].max()), float(tol[bad].min()))
    return before, y_all


@pytest.mark.parametrize("rank", [8, 16, 24, 32, 40, 64, 72, 128])
@pytest.mark.parametrize("x_dt", [torch.float32, torch.uint8])
@pytest.mark.parametrize("n,k", [(1, 8), (7, 33), (64, 64), (100, 515), (1001, 40), (768, 768), (130, 4100)])
def test_lora_sizes(rank, x_dt, n, k):
    lora_case(1, n, k, rank, [0, 1], 1, x_dt)
    lora_case(70, n, k, rank, [0, 1, 1, 18, 34, 65], 3, x_dt)


@pytest.mark.parametrize("x_dt", [torch.float32, torch.uint8])
def test_lora_segments(x_dt):
    """no rows, rows in front and behind, requests without an adapter, one adapter twice, many requests"""
    for bounds, which in (([7, 7, 7], None), ([0, 10, 20], [-1, -1])):
        before, after = lora_case(20, 48, 64, 16, bounds, 2, x_dt, which=which)
        same = torch.equal(before, after)
        assert same
    lora_case(100, 200, 128, 16, [5, 40, 41, 60, 90], 3, x_dt, which=[2, -1, 0, 2])
    lora_case(300, 96, 128, 8, list(range(301)), 7, x_dt)
    lora_case(333, 200, 264, 32, [0] + sorted(int(i) for i in perm(4, 333)[:40]), 5, x_dt)
    lora_case(1500, 300, 300, 16, [0, 1400], 1, x_dt)
    assert status() == 0


@pytest.mark.parametrize("x_dt", [torch.float32, torch.uint8])
@pytest.mark.parametrize("rank", [8, 16, 32, 56, 128])
def test_lora_of_more_steps_than_run_at_a_time(rank, x_dt):
    """CTAs that go on from unit to unit, in the middle of rows of B too; few rows to a request, and many"""
    lora_case(1003, 4101, 1030, rank, [3, 100, 101, 400, 990], 3, x_dt, which=[2, 0, -1, 1], y_gap=3)
    lora_case(200, 3001, 520, rank, list(range(0, 201, 2)), 9, x_dt)
    lora_case(200, 512 if x_dt == torch.float32 else 1020, 250, rank, list(range(0, 201, 2)), 9, x_dt)     # (short K)
    assert status() == 0


@pytest.mark.parametrize("x_dt", [torch.float32, torch.uint8])
def test_lora_strides_and_units(x_dt):
    for x_off in (0, 1, 2, 3, 4):
        lora_case(37, 65, 120, 16, [0, 20, 37], 2, x_dt, x_off=x_off, x_gap=3, y_off=x_off % 3, y_gap=x_off, a_gap=8)
    for unit in ("row", "device", "host"):
        lora_case(37, 64, 128, 16, [0, 20, 37], 2, x_dt, unit=unit, scale=unit != "device")
    for values in (1e-20, 1e-6, 1e6, 1e20):
        lora_case(37, 64, 128, 16, [0, 20, 37], 2, torch.float32, values=values)


def test_lora_refuses_on_the_device_what_leads_outside():
    """segments that fall or leave the rows, adapters that do not exist: left out, the others are done"""
    for bounds, which in (([0, 10, 41], [0, 1]), ([-1, 5, 20], [0, 1]), ([0, 10, 20], [0, 2]), ([0, 30, 20, 40], [0, 1, 1]), ([0, 10, 1 << 30], [1, 0])):
        lora_case(40, 64, 64, 16, bounds, 2, torch.float32, which=which)
        assert status() == 53
    lora_case(40, 64, 64, 16, [0, 40], 2, torch.float32)
    assert B.lib().bolt_b200_synchronize() == B.SUCCESS


def test_lora_gives_the_same_bits_again():
    for args in ((64, 1000, 2048, 16, list(range(65)), 64), (600, 700, 4096, 32, [0, 100, 590], 2)):
        a, b = (lora_case(*args, torch.uint8 if args[3] == 16 else torch.float32, seed=3, scale=False, unit="host") for _ in range(2))
        if args[3] == 32:                       # (bytes of x come from the generator's state)
            assert torch.equal(a[1], b[1])


# ---- many sequences, streams, host memory, all of them together ------------------------------------------------------
@pytest.mark.parametrize("i8", [0, 1])
@pytest.mark.parametrize("sequences,longest", [(256, 70), (257, 70), (1024, 70), (1025, 70), (5000, 40), (65535, 3)])
def test_attention_of_many_sequences(i8, sequences, longest):
    """more than a warp counts for itself, up to the most that a call takes; every third has no tokens"""
    page, kv, dim, heads = 8, 1, 32, 3
    g = torch.Generator(device="cuda")
    g.manual_seed(sequences)
    length = torch.randint(0, longest + 1, (sequences,), device="cuda", generator=g, dtype=torch.int32)
    length[::3] = 0
    tp = -(-longest // page)
    cache = Cache(1, 3000, page, kv, dim, i8)
    table = torch.randint(0, 3000, (sequences, tp), device="cuda", generator=g, dtype=torch.int32)
    table[torch.arange(tp, device="cuda")[None, :] * page >= length[:, None]] = -1
    q = rand(5, sequences, heads, dim)
    got, lse = attend(cache, q, table, length)
    assert status() == 0
    t = torch.arange(longest, device="cuda")
    pages, at = table.clamp(min=0).long()[:, t // page], (t % page)[None, :].expand(sequences, -1)
    k, v = (x[pages, 0, at].double() / (s[pages, 0, at].double()[..., None] if i8 else 1) for x, s in ((cache.k, cache.ks), (cache.v, cache.vs)))
    live = t[None, :] < length[:, None]
    s = torch.einsum("bhd,btd->bht", q.double(), k) * np.float32(dim ** -0.5).item()
    off = ((dim + 16) * U * dim ** -0.5 * torch.einsum("bhd,btd->bht", q.double().abs(), k.abs()) * live[:, None, :]).amax(-1)
    s = torch.where(live[:, None, :], s, -math.inf)
    top = torch.logsumexp(s, -1)
    p = torch.where(live[:, None, :], torch.exp(s - top[..., None]), 0.0)
    want, tol = torch.einsum("bht,btd->bhd", p, v), 2 * (off[..., None] + (longest / 16 + 72) * U) * torch.einsum("bht,btd->bhd", p, v.abs()) + 1e-30
    n_bad = int(((got.double() - want).abs() > tol).sum())
    n_lse = int(((lse.double() - top).abs() > off + (longest / 16 + 72) * U + 2 * U * top.abs()).sum()) + int((lse.isinf() != (length == 0)[:, None]).sum())
    assert (n_bad, n_lse) == (0, 0)


def test_calls_on_two_streams_do_not_mix():
    """eager calls of all three operators, each stream with tensors and workspaces of its own"""
    def make(seed):
        cache, q, table, length = batch(seed, [900, 33, 0, 2000], (16, 2, 128, seed % 2, "hnd", 0), 16)
        qkv = rand(seed + 1, 4, (16 + 4) * 128)
        pos = (length.clamp(min=1) - 1).int()
        pos[2] = -1
        cos, sin = rand(seed + 2, 2048, 64), rand(seed + 3, 2048, 64)
        out, tmp = torch.empty_like(q), torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
        a, b, y = rand(seed + 4, 2, 16, 2048, dtype=torch.float16), rand(seed + 5, 2, 512, 16, dtype=torch.float16), torch.zeros(4, 512, device="cuda")
        first, adapter = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1, 4], [1, 0]))
        qo = torch.empty_like(q)
        e = qkv.data_ptr()

        def run():
            B.kv_append(cache.desc(), B.KvAppend(4, 16, B.DT_F32, B.DT_F32, e, e + 4 * 2048, e + 4 * 2304, qo.data_ptr(), 2560, 2560, 2560, 2048, None,
                                                 pos.data_ptr(), table.data_ptr(), 4, table.shape[1], 128, 0, 2048, cos.data_ptr(), sin.data_ptr()))
            B.paged_attention(cache.desc(), B.PagedAttention(4, 16, B.DT_F32, B.DT_F32, qo.data_ptr(), out.data_ptr(), None, 2048, 2048, table.data_ptr(),
                                                             length.data_ptr(), table.shape[1], 0, 0.09, 1.0), tmp.numel(), tmp.data_ptr())
            B.lora(B.Lora(4, 512, 2048, 16, 2, 2, B.DT_F32, out.data_ptr(), y.data_ptr(), 2048, 512, a.data_ptr(), b.data_ptr(), 2048, None, first.data_ptr(),
                          adapter.data_ptr(), 1.0, None, None), tmp.numel(), tmp.data_ptr())
        return run, (out, y, cache, q, qkv, pos, cos, sin, tmp, a, b, first, adapter, qo, table, length)

    works = [make(10), make(21)]
    qo_rows = []
    for run, keep in works:
        keep[13].zero_()
        run()
        torch.cuda.synchronize()
        qo_rows.append((keep[0].clone(), keep[1].clone()))
    streams = [torch.cuda.Stream() for _ in works]
    for _ in range(20):
        for _, keep in works:
            keep[1].zero_()
        torch.cuda.synchronize()
        for (run, _), st in zip(works, streams):
            B.lib().bolt_b200_set_stream(C.c_void_p(st.cuda_stream))
            run()
            B.lib().bolt_b200_set_stream(None)
        torch.cuda.synchronize()
        same = [torch.equal(k[0], o) and torch.equal(k[1], y) for (_, k), (o, y) in zip(works, qo_rows)]
        assert same == [True, True]
    assert status() == 0


def test_host_memory_is_refused():
    cache, q, table, length = batch(3, [20], (16, 1, 64, 0, "hnd", 0), 2)
    host = torch.zeros(1 << 16, dtype=torch.float32)
    call = B.PagedAttention(1, 2, B.DT_F32, B.DT_F32, q.data_ptr(), host.data_ptr(), None, 128, 128, table.data_ptr(), length.data_ptr(), table.shape[1], 0, 0.1, 1.0)
    tmp = torch.empty(1 << 23, dtype=torch.uint8, device="cuda")
    lib = B.lib()
    assert lib.bolt_b200_paged_attention(cache.desc(), call, tmp.numel(), tmp.data_ptr()) == B.NOT_MATCH
    call.out = q.data_ptr()
    assert lib.bolt_b200_paged_attention(cache.desc(), call, tmp.numel(), host.data_ptr()) == B.NOT_MATCH
    d = cache.desc()
    d.k = host.data_ptr()
    assert lib.bolt_b200_paged_attention(d, call, tmp.numel(), tmp.data_ptr()) == B.NOT_MATCH
    ap = B.KvAppend(1, 0, B.DT_F32, B.DT_F32, None, q.data_ptr(), q.data_ptr(), None, 0, 0, 0, 0, None, host.data_ptr(), table.data_ptr(), 1, 2, 0, 0, 0, None, None)
    assert lib.bolt_b200_kv_append(cache.desc(), ap) == B.NOT_MATCH
    lo = B.Lora(1, 64, 64, 8, 1, 1, B.DT_F32, q.data_ptr(), tmp.data_ptr(), 64, 64, host.data_ptr(), tmp.data_ptr(), 64, None, length.data_ptr(), length.data_ptr(),
                1.0, None, None)
    assert lib.bolt_b200_lora(lo, tmp.numel() // 2, tmp.data_ptr() + tmp.numel() // 2) == B.NOT_MATCH
    assert status() == 0


def packed(seed, k, n):
    """a pre-packed u8 x s8 weight: (bytes [k, n], packed, offset of its offsets, scale per column)"""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    w = torch.randint(-127, 128, (k, n), dtype=torch.int8, device="cuda", generator=g)
    desc = B.tensor2df(B.DT_I8, B.DF_NORMAL, k, n)
    nbytes, rhs = B.matrix_matrix_multiply_transform_rhs_bytes(desc)
    p = torch.zeros(nbytes, dtype=torch.uint8, device="cuda")
    B.matrix_matrix_multiply_transform_rhs(desc, w.data_ptr(), p.data_ptr())
    return w, p, rhs, 800.0 + 200 * torch.rand(n, device="cuda", generator=g)


def project(x, row_scale, weight, y):
    """y = x W of the quantized product, a scale for every row of x and column of W"""
    w, p, rhs, col = weight
    ep = B.GemmEpilogue()
    ep.out_dt, ep.out_scale, ep.row_scale, ep.col_scale, ep.sA, ep.sB = B.DT_F32, 1.0, row_scale.data_ptr(), col.data_ptr(), 1.0, 1.0
    m, k = x.shape
    B.CHECK_STATUS(B.lib().bolt_b200_gemm_u8s8_ex(w.shape[1], m, k, x.data_ptr(), p.data_ptr(), p.data_ptr() + rhs, y.data_ptr(), C.byref(ep)), "gemm")


@pytest.mark.parametrize("i8", [0, 1])
@pytest.mark.parametrize("graph", [0, 1])
def test_decoding_steps(i8, graph):
    """Prompts, then one token at a time: quantized projection with adapters, append, attention in 8 bits, projection with
    adapters.  Every stage against 64 bits from the stage before it; the steps also as one captured graph."""
    seqs, heads, kv, dim, hidden, page, tp, rank = 3, 8, 2, 64, 256, 16, 8, 8
    width = (heads + 2 * kv) * dim
    w_in, w_out = packed(1, hidden, width), packed(2, heads * dim, hidden)
    cache = Cache(3, seqs * tp, page, kv, dim, i8)
    table = perm(4, seqs * tp).int().view(seqs, tp).contiguous()
    ang = torch.arange(tp * page, device="cuda", dtype=torch.float64)[:, None] * 1000.0 ** (-torch.arange(dim // 2, device="cuda") / (dim // 2))[None, :]
    cos, sin = ang.cos().float().contiguous(), ang.sin().float().contiguous()
    adapters = [(rand(5, 2, rank, k, dtype=torch.float16, scale=k ** -0.5), rand(6, 2, n, rank, dtype=torch.float16, scale=rank ** -0.5))
                for k, n in ((hidden, width), (heads * dim, hidden))]
    out_scale = 60.0
    prompt = [5, 40, 17]
    x_all = torch.randint(0, 256, (seqs, 64, hidden), dtype=torch.uint8, device="cuda", generator=torch.Generator(device="cuda").manual_seed(9))
    tmp = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")

    def layer(x, row_scale, first, adapter, seq, pos, length, bufs):
        """x [m, hidden] of any number of sequences; attention (decoding) if length is given"""
        m = x.shape[0]
        qkv, q, ctx, ones, y = bufs
        project(x, row_scale, w_in, qkv)
        (a, b), n_seg = adapters[0], first.numel() - 1
        B.lora(B.Lora(m, width, hidden, rank, 2, n_seg, B.DT_U8_Q, x.data_ptr(), qkv.data_ptr(), hidden, width, a.data_ptr(), b.data_ptr(), hidden, None,
                      first.data_ptr(), adapter.data_ptr(), 1.0, None, row_scale.data_ptr()), tmp.numel(), tmp.data_ptr())
        e = qkv.data_ptr()
        B.kv_append(cache.desc(), B.KvAppend(m, heads, B.DT_F32, B.DT_F32, e, e + 4 * heads * dim, e + 4 * (heads + kv) * dim, q.data_ptr(), width, width, width,
                                             heads * dim, ptr(seq), pos.data_ptr(), table.data_ptr(), seqs, tp, dim, 0, tp * page, cos.data_ptr(), sin.data_ptr()))
        if length is None:
            return
        B.paged_attention(cache.desc(), B.PagedAttention(seqs, heads, B.DT_F32, B.DT_U8_Q, q.data_ptr(), ctx.data_ptr(), None, heads * dim, heads * dim,
                                                         table.data_ptr(), length.data_ptr(), tp, 0, dim ** -0.5, out_scale), tmp.numel(), tmp.data_ptr())
        project(ctx, ones, w_out, y)
        a, b = adapters[1]
        B.lora(B.Lora(m, hidden, heads * dim, rank, 2, n_seg, B.DT_U8_Q, ctx.data_ptr(), y.data_ptr(), heads * dim, hidden, a.data_ptr(), b.data_ptr(),
                      heads * dim, None, first.data_ptr(), adapter.data_ptr(), out_scale, None, None), tmp.numel(), tmp.data_ptr())

    def buffers(m):
        return (torch.zeros(m, width, device="cuda"), torch.zeros(m, heads * dim, device="cuda"), torch.zeros(m, heads * dim, dtype=torch.uint8, device="cuda"),
                torch.full((m,), out_scale, device="cuda"), torch.zeros(m, hidden, device="cuda"))

    def exact_projection(x, row_scale, weight, ad, which):
        xx = (x.double() - 128) / row_scale.double()[:, None]
        y = xx @ (weight[0].double() / weight[3].double()[None, :])
        for i, w in enumerate(which):
            if w >= 0:
                y[i] += (xx[i] @ ad[0][w].double().T) @ ad[1][w].double().T
        return y

    # the prompts, all at once
    which = [1, -1, 0]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    m = sum(prompt)
    x = torch.cat([x_all[i, :n] for i, n in enumerate(prompt)]).contiguous()
    rs = 40 + 10 * torch.rand(m, device="cuda")
    first, adapter = i32(np.concatenate(([0], np.cumsum(prompt))).tolist()), i32(which)
    seq, pos = i32([i for i, n in enumerate(prompt) for _ in range(n)]), i32([t for n in prompt for t in range(n)])
    bufs = buffers(m)
    layer(x, rs, first, adapter, seq, pos, None, bufs)
    want = exact_projection(x, rs, w_in, adapters[0], [which[i] for i in seq.tolist()])
    off = float((bufs[0].double() - want).abs().max() / want.abs().max())
    assert off < 1e-5, off
    # decoding
    length, dpos = i32(prompt), i32([0] * seqs)
    first1, rs1, x1, bufs1 = i32([0, 1, 2, 3]), torch.full((seqs,), 44.0, device="cuda"), torch.empty(seqs, hidden, dtype=torch.uint8, device="cuda"), buffers(seqs)
    step = lambda: layer(x1, rs1, first1, adapter, None, dpos, length, bufs1)  # noqa: E731
    if graph:
        x1.fill_(128)
        dpos.copy_(length)
        step()          # (everything loaded and planned; the row is written again by the first step)
        torch.cuda.synchronize()
        g, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(g, stream=stream):
            B.lib().bolt_b200_set_stream(C.c_void_p(torch.cuda.current_stream().cuda_stream))
            step()
            B.lib().bolt_b200_set_stream(None)
        step = g.replay
    for t in range(12):
        x1.copy_(x_all[:, 45 + t])
        dpos.copy_(length)
        length += 1
        step()
        torch.cuda.synchronize()
        qkv, q, ctx, ones, y = bufs1
        want = exact_projection(x1, rs1, w_in, adapters[0], which)
        assert float((qkv.double() - want).abs().max() / want.abs().max()) < 1e-5
        rotated = turned(qkv.cpu().numpy().reshape(seqs, heads + 2 * kv, dim), dpos.cpu().numpy(), cos.cpu().numpy(), sin.cpu().numpy(), dim, 0)
        same = np.array_equal(q.cpu().numpy().reshape(seqs, heads, dim), rotated[:, :heads])
        assert same
        check_attention(cache, q.view(seqs, heads, dim), table, length, ctx.view(seqs, heads, dim), None, out_scale=out_scale)
        want = exact_projection(ctx, ones, w_out, adapters[1], which)
        assert float((y.double() - want).abs().max() / want.abs().max()) < 1e-5
    assert status() == 0
