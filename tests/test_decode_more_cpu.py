"""Host side of the operators of a decoding step, continued: sizes and strides whose products leave 64 bits."""
import ctypes as C
import os
import sys

import pytest

sys.path.insert(0, os.path.dirname(__file__))
import fake_gpu  # noqa: E402
from test_decode_cpu import AT, I8, OK, UNSUPPORTED, append, attention, cache, lora  # noqa: E402

MOST = (1 << 31) - 1
FAR = 1 << 36       # the largest stride of a cache


@pytest.mark.parametrize("change,code", [
    (dict(pages=MOST, page_stride=1 << 30), OK), (dict(pages=MOST, page_stride=FAR), UNSUPPORTED), (dict(pages=1 << 24, page_stride=FAR), OK),
    (dict(page_size=MOST, token_stride=FAR), UNSUPPORTED), (dict(page_size=MOST, token_stride=1 << 28), OK), (dict(kv_heads=65535, head_stride=FAR), OK),
    (dict(pages=MOST, page_size=MOST, page_stride=1 << 29, token_stride=1 << 29), OK),
    (dict(pages=MOST, page_size=MOST, page_stride=1 << 30, token_stride=1 << 30), UNSUPPORTED),
    (dict(I8, pages=MOST, page_stride=1 << 31), OK), (dict(I8, pages=MOST, page_size=MOST), UNSUPPORTED),
    (dict(I8, pages=1 << 20, page_size=1 << 20, kv_heads=1 << 15), OK), (dict(I8, pages=1 << 25, page_size=1 << 20, kv_heads=1 << 15), OK),
    (dict(I8, pages=1 << 26, page_size=1 << 20, kv_heads=1 << 15), UNSUPPORTED)])
def test_caches_beyond_64_bits(change, code):
    lib = fake_gpu.load()
    n = C.c_uint32()
    c, tmp = cache(**change), C.c_void_p(AT)
    wide = 64 * change.get("kv_heads", 2)
    heads = dict(heads=change.get("kv_heads", 2), q_stride=wide, out_stride=wide, sequences=1, table_pages=1 << 10 if change.get("page_size", 16) < 1 << 16 else 1)
    assert lib.bolt_b200_kv_append(c, append(tokens=1, k_stride=wide, v_stride=wide)) == code
    assert lib.bolt_b200_paged_attention_tmp_bytes(c, attention(**heads), C.byref(n)) == code
    assert lib.bolt_b200_paged_attention(c, attention(**heads), 1 << 30, tmp) == code
    assert (fake_gpu.launches(lib) == []) == (code != OK) and lib.fake_last_error() == 0


def test_tables_and_adapters_beyond_64_bits():
    lib = fake_gpu.load()
    n = C.c_uint32()
    for sequences, pages, code in ((1 << 31, 1 << 29, OK), (1 << 31, 1 << 30, UNSUPPORTED), (0xFFFFFFFF, 0xFFFFFFFF, UNSUPPORTED)):
        assert lib.bolt_b200_kv_append(cache(), append(sequences=sequences, table_pages=pages)) == code
    for adapters, rank, stride, code in ((MOST, 16, 1 << 26, OK), (MOST, 16, 1 << 27, UNSUPPORTED), (MOST, 128, 1 << 30, UNSUPPORTED), (1 << 22, 128, 1 << 30, OK)):
        call = lora(adapters=adapters, rank=rank, a_stride=stride)
        assert lib.bolt_b200_lora_tmp_bytes(call, C.byref(n)) == code
        assert lib.bolt_b200_lora(call, 1 << 30, C.c_void_p(AT)) == code
