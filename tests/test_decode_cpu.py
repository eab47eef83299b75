"""Host side of the operators of a decoding step without a GPU: what calls refuse (fake_gpu.py), what they launch, and where
numbers that the device reads lead."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.dirname(__file__))
import bolt_b200 as B  # noqa: E402
import fake_gpu  # noqa: E402
from bolt_b200 import build  # noqa: E402

HERE = os.path.dirname(os.path.abspath(__file__))
BIG = np.zeros(1 << 16, np.uint8)
AT = (BIG.ctypes.data + 255) & ~255


@pytest.fixture(scope="module")
def harness(tmp_path_factory):
    so = str(tmp_path_factory.mktemp("native") / "decode_harness.so")
    cmd = [build._nvcc()] + build.NVCC_FLAGS + ["-shared", "-o", so, os.path.join(HERE, "native", "decode_harness.cu")]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    lib = C.CDLL(so)
    lib.harness_row.restype = lib.harness_scale.restype = C.c_longlong
    u, l = C.c_uint32, C.c_uint64
    lib.harness_row.argtypes = [C.c_void_p, l, u, u, u, u, u, l, l, l, u, u, u]
    lib.harness_scale.argtypes = [u] * 6
    lib.harness_tokens.argtypes = [C.c_int32, u, u, u, C.c_void_p]
    lib.harness_parts.argtypes, lib.harness_parts.restype = [u, u], u
    lib.harness_part_begin.argtypes, lib.harness_part_begin.restype = [u, u, u], u
    lib.harness_part_of.argtypes, lib.harness_part_of.restype = [u, u, u], u
    lib.harness_tiles.argtypes, lib.harness_tiles.restype = [u, u, u], u
    return lib


def test_rows_of_a_cache(harness):
    """every row inside the cache, each once; whatever leads outside is refused"""
    pages, ps, heads, dim = 5, 7, 3, 16
    table = np.array([[4, 0, 2], [1, 3, 99], [-1, 5, -2147483648]], np.int32)
    for strides in ((heads * ps * dim, dim, ps * dim), (ps * heads * dim, heads * dim, dim)):
        seen = set()
        for s in range(3):
            for position in list(range(0, 30)) + [0x7FFFFFFF, 0xFFFFFFFF]:
                for h in range(heads):
                    at = harness.harness_row(table.ctypes.data, s, 3, pages, ps, heads, dim, *strides, position, h, 2)
                    p = position // ps
                    good = p < 3 and 0 <= table[s, p] < pages
                    assert (at >= 0) == good
                    if good:
                        assert at % 32 == 0 and at + 32 <= 2 * pages * heads * ps * dim and at not in seen
                        seen.add(at)
        assert len(seen) == 5 * ps * heads
    # far into a large cache
    t = np.array([(1 << 31) - 1], np.int32)
    assert harness.harness_row(t.ctypes.data, 0, 1, (1 << 31) - 1, 64, 8, 256, 1 << 17, 256, 1 << 14, 0, 0, 2) == -1
    assert harness.harness_row(t.ctypes.data, 0, 1, 1 << 31, 64, 8, 256, 1 << 17, 256, 1 << 14, 63, 7, 2) == 2 * (((1 << 31) - 1) * (1 << 17) + 63 * 256 + (7 << 14))
    assert harness.harness_scale(1 << 31, 64, 8, (1 << 31) - 1, 63, 7) == (((1 << 31) - 1) * 8 + 7) * 64 + 63


def test_tokens_of_a_sequence(harness):
    r = (C.c_uint32 * 2)()
    for length, pages, page, window, good, begin, end in (
            (0, 3, 16, 0, 1, 0, 0), (48, 3, 16, 0, 1, 0, 48), (49, 3, 16, 0, 0, 0, 48), (-1, 3, 16, 5, 0, 0, 0), (40, 3, 16, 5, 1, 35, 40), (4, 3, 16, 5, 1, 0, 4),
            (5, 3, 16, 5, 1, 0, 5), (0x7FFFFFFF, 1 << 20, 1 << 20, 7, 1, 0x7FFFFFF8, 0x7FFFFFFF), (-2147483648, 1, 1, 0, 0, 0, 0), (0x7FFFFFFF, 2, 1, 1, 0, 1, 2)):
        assert harness.harness_tokens(length, pages, page, window, r) == good and list(r) == [begin, end]


def test_parts_cover_the_row_once(harness):
    """every place of the row is in one part, no part is empty, they differ by one place at most, and a part is found from a place"""
    assert harness.harness_parts(0, 148) == 0
    for total in (1, 2, 3, 147, 148, 149, 1000, 12345, (1 << 31) + 5, (1 << 32) - 1):
        for most in (1, 2, 147, 148, 1184):
            parts = harness.harness_parts(total, most)
            assert parts == min(total, most)
            borders = [harness.harness_part_begin(i, total, most) for i in range(parts + 1)]
            assert borders[0] == 0 and borders[-1] == total
            sizes = {b - a for a, b in zip(borders, borders[1:])}
            assert min(sizes) >= 1 and max(sizes) - min(sizes) <= 1
            for place in sorted({0, total - 1, total // 2, *borders[:-1], *[b - 1 for b in borders[1:]]}):
                i = harness.harness_part_of(place, total, most)
                assert borders[i] <= place < borders[i + 1], (total, most, place, i)
    for begin, end, shift, n in ((0, 0, 7, 0), (5, 5, 7, 0), (0, 1, 7, 1), (0, 128, 7, 1), (0, 129, 7, 2), (127, 129, 7, 2), (128, 129, 7, 1),
                                 (130, 700, 7, 5), (0, 0x7FFFFFFF, 8, 1 << 23)):
        assert harness.harness_tiles(begin, end, shift) == n


def cache(**kw):
    a = dict(dt=B.DT_F16, pages=4, page_size=16, kv_heads=2, dim=64, page_stride=2048, token_stride=64, head_stride=1024, k=AT, v=AT, k_scale=None,
             v_scale=None)
    a.update(kw)
    return B.KvCache(**a)


I8 = dict(dt=B.DT_I8, k_scale=AT, v_scale=AT)


def append(**kw):
    a = dict(tokens=3, heads=4, dt=B.DT_F32, q_out_dt=B.DT_F32, q=AT, k=AT, v=AT, q_out=AT, q_stride=512, k_stride=512, v_stride=512, q_out_stride=256,
             sequence=AT, position=AT, table=AT, sequences=3, table_pages=2, rotary_dim=64, interleaved=0, rotary_positions=32, cos=AT, sin=AT)
    a.update(kw)
    return B.KvAppend(**a)


def attention(**kw):
    a = dict(sequences=3, heads=4, q_dt=B.DT_F32, out_dt=B.DT_F32, q=AT, out=AT, lse=AT, q_stride=256, out_stride=256, table=AT, length=AT, table_pages=2,
             window=0, scale=0.125, out_scale=1.0)
    a.update(kw)
    return B.PagedAttention(**a)


def lora(**kw):
    a = dict(rows=5, N=64, K=64, rank=16, adapters=2, segments=2, x_dt=B.DT_F32, x=AT, y=AT, x_stride=64, y_stride=64, a=AT, b=AT, a_stride=64, scale=AT,
             first_row=AT, adapter=AT, sA=1.0, d_sA=None, row_scale=None)
    a.update(kw)
    return B.Lora(**a)


OK, NULL, MISMATCH, UNSUPPORTED = B.SUCCESS, B.NULL_POINTER, B.NOT_MATCH, B.NOT_SUPPORTED
CACHES = [
    (dict(k=None), NULL), (dict(v=None), NULL), (dict(dt=B.DT_F32), UNSUPPORTED), (dict(dt=B.DT_U8_Q), UNSUPPORTED), (dict(dt=B.DT_I8), NULL),
    (dict(I8, v_scale=None), NULL), (dict(I8, k_scale=AT + 2), UNSUPPORTED), (dict(pages=0), MISMATCH), (dict(page_size=0), MISMATCH), (dict(kv_heads=0), MISMATCH),
    (dict(dim=0), MISMATCH), (dict(dim=264, token_stride=264, page_stride=1 << 15, head_stride=1 << 14), UNSUPPORTED), (dict(dim=60), UNSUPPORTED),
    (dict(I8, dim=56), UNSUPPORTED), (dict(k=AT + 8), UNSUPPORTED), (dict(v=AT + 2), UNSUPPORTED), (dict(token_stride=68), UNSUPPORTED),
    (dict(token_stride=32), MISMATCH), (dict(head_stride=0), MISMATCH), (dict(page_stride=8), MISMATCH), (dict(page_stride=1 << 50), UNSUPPORTED),
    (dict(pages=1 << 31), UNSUPPORTED)]


@pytest.mark.parametrize("change,code", CACHES)
def test_caches_that_are_refused(change, code):
    lib = fake_gpu.load()
    n = C.c_uint32()
    tmp = C.c_void_p(AT)
    assert lib.bolt_b200_kv_append(cache(**change), append()) == code
    assert lib.bolt_b200_paged_attention(cache(**change), attention(), 1 << 30, tmp) == code
    assert lib.bolt_b200_paged_attention_tmp_bytes(cache(**change), attention(), C.byref(n)) == code
    assert fake_gpu.launches(lib) == [] and lib.fake_last_error() == 0


@pytest.mark.parametrize("change,code", [
    ({}, OK), (dict(tokens=0), OK), (dict(q=None), NULL), (dict(q_out=None), NULL), (dict(heads=0, q=None, q_out=None), OK), (dict(k=None), NULL), (dict(v=None), NULL),
    (dict(position=None), NULL), (dict(table=None), NULL), (dict(cos=None), NULL), (dict(rotary_dim=0, cos=None, sin=None), OK), (dict(dt=B.DT_I8), UNSUPPORTED),
    (dict(q_out_dt=B.DT_U8_Q), UNSUPPORTED), (dict(q_out_dt=B.DT_F16), OK), (dict(rotary_dim=65), MISMATCH), (dict(rotary_dim=66), MISMATCH),
    (dict(rotary_dim=6), OK), (dict(sequence=None), OK), (dict(sequence=None, tokens=4), MISMATCH), (dict(sequences=0), MISMATCH), (dict(table_pages=0), MISMATCH),
    (dict(q_stride=255), MISMATCH), (dict(k_stride=127), MISMATCH), (dict(v_stride=0), MISMATCH), (dict(q_out_stride=8), MISMATCH),
    (dict(tokens=1, q_stride=0, k_stride=0, v_stride=0, q_out_stride=0), OK), (dict(k_stride=1 << 40), UNSUPPORTED), (dict(q=AT + 2), UNSUPPORTED),
    (dict(dt=B.DT_F16, k=AT + 2), OK), (dict(dt=B.DT_F16, v=AT + 1), UNSUPPORTED), (dict(position=AT + 2), UNSUPPORTED), (dict(cos=AT + 1), UNSUPPORTED),
    (dict(tokens=0xFFFFFFFF), UNSUPPORTED), (dict(heads=70000, q_stride=1 << 24, q_out_stride=1 << 24), UNSUPPORTED)])
def test_appends(change, code):
    lib = fake_gpu.load()
    for c in (cache(), cache(**I8)):
        lib.fake_forget_launches()
        before = lib.bolt_b200_launch_count()
        assert lib.bolt_b200_kv_append(c, append(**change)) == code
        n = 1 if code == OK and change.get("tokens") != 0 else 0
        assert len(fake_gpu.launches(lib)) == n == lib.bolt_b200_launch_count() - before
        assert lib.fake_last_error() == 0
    assert lib.bolt_b200_kv_append(None, append()) == NULL and lib.bolt_b200_kv_append(cache(), None) == NULL


@pytest.mark.parametrize("change,code", [
    ({}, OK), (dict(sequences=0), OK), (dict(q=None), NULL), (dict(out=None), NULL), (dict(lse=None), OK), (dict(table=None), NULL), (dict(length=None), NULL),
    (dict(heads=0), MISMATCH), (dict(heads=5, q_stride=320, out_stride=320), MISMATCH), (dict(table_pages=0), MISMATCH), (dict(q_dt=B.DT_U8_Q), UNSUPPORTED),
    (dict(out_dt=B.DT_I8), UNSUPPORTED), (dict(out_dt=B.DT_U8_Q), OK), (dict(q_stride=100), MISMATCH), (dict(out_stride=255), MISMATCH),
    (dict(sequences=1, q_stride=0, out_stride=0), OK), (dict(q_stride=1 << 40), UNSUPPORTED), (dict(q=AT + 2), UNSUPPORTED), (dict(q_dt=B.DT_F16, q=AT + 2), OK),
    (dict(out=AT + 2), UNSUPPORTED), (dict(out_dt=B.DT_U8_Q, out=AT + 1), OK), (dict(lse=AT + 1), UNSUPPORTED), (dict(length=AT + 2), UNSUPPORTED),
    (dict(sequences=70000), UNSUPPORTED), (dict(sequences=60000, table_pages=1 << 14), OK), (dict(sequences=60000, table_pages=1 << 18), UNSUPPORTED)])
def test_attentions(change, code):
    lib = fake_gpu.load()
    n = C.c_uint32(0)
    for c in (cache(), cache(**I8)):
        call = attention(**change)
        early = change.get("sequences") == 0
        if code == OK:
            assert lib.bolt_b200_paged_attention_tmp_bytes(c, call, C.byref(n)) == OK
            if n.value and not early:
                assert lib.bolt_b200_paged_attention(c, call, n.value - 1, C.c_void_p(AT)) == MISMATCH
                assert lib.bolt_b200_paged_attention(c, call, n.value, None) == NULL
                assert lib.bolt_b200_paged_attention(c, call, n.value, C.c_void_p(AT + 8)) == UNSUPPORTED
        lib.fake_forget_launches()
        before = lib.bolt_b200_launch_count()
        assert lib.bolt_b200_paged_attention(c, call, 1 << 30, C.c_void_p(AT)) == code
        assert (len(fake_gpu.launches(lib)) != 0) == (code == OK and not early)
        assert len(fake_gpu.launches(lib)) == lib.bolt_b200_launch_count() - before and lib.fake_last_error() == 0
    assert lib.bolt_b200_paged_attention(None, attention(), 0, None) == NULL and lib.bolt_b200_paged_attention(cache(), None, 0, None) == NULL
    assert lib.bolt_b200_paged_attention_tmp_bytes(cache(), attention(), None) == NULL


@pytest.mark.parametrize("change,code", [
    ({}, OK), (dict(rows=0), OK), (dict(segments=0), OK), (dict(x=None), NULL), (dict(y=None), NULL), (dict(a=None), NULL), (dict(b=None), NULL),
    (dict(first_row=None), NULL), (dict(adapter=None), NULL), (dict(scale=None), OK), (dict(x_dt=B.DT_F16), UNSUPPORTED), (dict(x_dt=B.DT_U8_Q), OK),
    (dict(x_dt=B.DT_U8_Q, x=AT + 1, row_scale=AT, d_sA=AT), OK), (dict(K=0), MISMATCH), (dict(N=0), MISMATCH), (dict(adapters=0), MISMATCH), (dict(a_stride=56), MISMATCH),
    (dict(a_stride=68), UNSUPPORTED), (dict(rank=0), UNSUPPORTED), (dict(rank=12), UNSUPPORTED), (dict(rank=136), UNSUPPORTED), (dict(rank=128), OK),
    (dict(x_stride=63), MISMATCH), (dict(y_stride=63), MISMATCH), (dict(rows=1, x_stride=0, y_stride=0), OK), (dict(x_stride=1 << 40), UNSUPPORTED),
    (dict(x=AT + 2), UNSUPPORTED), (dict(y=AT + 1), UNSUPPORTED), (dict(a=AT + 8), UNSUPPORTED), (dict(b=AT + 2), UNSUPPORTED), (dict(scale=AT + 2), UNSUPPORTED),
    (dict(adapter=AT + 1), UNSUPPORTED), (dict(K=63), OK), (dict(N=61), OK), (dict(rows=1 << 23), UNSUPPORTED), (dict(segments=1 << 21), UNSUPPORTED)])
def test_adapters(change, code):
    lib = fake_gpu.load()
    n = C.c_uint32(0)
    call = lora(**change)
    early = change.get("rows") == 0 or change.get("segments") == 0
    if code == OK:
        assert lib.bolt_b200_lora_tmp_bytes(call, C.byref(n)) == OK
        if not early:
            assert lib.bolt_b200_lora(call, n.value - 1, C.c_void_p(AT)) == MISMATCH
            assert lib.bolt_b200_lora(call, n.value, None) == NULL
            assert lib.bolt_b200_lora(call, n.value, C.c_void_p(AT + 8)) == UNSUPPORTED
    lib.fake_forget_launches()
    before = lib.bolt_b200_launch_count()
    assert lib.bolt_b200_lora(call, 1 << 30, C.c_void_p(AT)) == code
    assert (len(fake_gpu.launches(lib)) != 0) == (code == OK and not early)
    assert len(fake_gpu.launches(lib)) == lib.bolt_b200_launch_count() - before and lib.fake_last_error() == 0
    assert lib.bolt_b200_lora(None, 0, None) == NULL and lib.bolt_b200_lora_tmp_bytes(call, None) == NULL
