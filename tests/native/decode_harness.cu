// The arithmetic of decode.cuh on numbers that a device reads, on the host (test_decode_cpu.py).
#include "decode.cuh"

using namespace b200;

extern "C" {

// byte offset of the row in a cache of `size`-byte elements, or -1
long long harness_row(const int32_t *table, uint64_t sequence, uint32_t table_pages, uint32_t pages, uint32_t page_size, uint32_t kv_heads,
    uint32_t dim, uint64_t page_stride, uint64_t token_stride, uint64_t head_stride, uint32_t position, uint32_t head, uint32_t size)
{
    const CacheView c{pages, page_size, kv_heads, dim, page_stride, token_stride, head_stride};
    uint32_t page, at;
    if (!page_of(table, sequence, table_pages, pages, page_size, position, &page, &at)) {
        return -1;
    }
    return (long long)(row_element(c, page, at, head) * size);
}
long long harness_scale(uint32_t pages, uint32_t page_size, uint32_t kv_heads, uint32_t page, uint32_t at, uint32_t head)
{
    const CacheView c{pages, page_size, kv_heads, 64, 0, 0, 0};
    return (long long)scale_element(c, page, at, head);
}

int harness_tokens(int32_t length, uint32_t table_pages, uint32_t page_size, uint32_t window, uint32_t *range)
{
    return live_tokens(length, table_pages, page_size, window, range, range + 1);
}
// parts that are made; their borders; the part that holds a place
uint32_t harness_parts(uint32_t total, uint32_t most)
{
    return Parts(total, most).n;
}
uint32_t harness_part_begin(uint32_t i, uint32_t total, uint32_t most)
{
    return Parts(total, most).begin(i);
}
uint32_t harness_part_of(uint32_t place, uint32_t total, uint32_t most)
{
    return Parts(total, most).of(place);
}
uint32_t harness_tiles(uint32_t begin, uint32_t end, uint32_t shift)
{
    return tiles_of(begin, end, shift);
}

}  // extern "C"
