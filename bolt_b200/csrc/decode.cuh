// decode.cuh -- what the operators of a decoding step (kv_append.cu, paged_attention.cu, lora.cu) share: where rows of a
// paged cache are, and the checks of their pointers.  The arithmetic on numbers that the device reads is __host__
// __device__, so that what happens to wrong ones can be seen without a GPU.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace b200 {

enum DecodeStatus { BAD_APPEND = 51, BAD_ATTENTION = 52, BAD_LORA = 53 };   // what the device status word says

struct CacheView {
    uint32_t pages, page_size, kv_heads, dim;
    uint64_t page_stride, token_stride, head_stride;   // elements
};

// The page of a position, or false: nothing there may be touched.
__host__ __device__ inline bool page_of(const int32_t *table, uint64_t sequence, uint32_t table_pages, uint32_t pages, uint32_t page_size,
    uint32_t position, uint32_t *page, uint32_t *at)
{
    const uint32_t p = position / page_size;
    if (p >= table_pages) {
        return false;
    }
    const int32_t t = table[sequence * table_pages + p];
    *page = (uint32_t)t;
    *at = position - p * page_size;
    return t >= 0 && (uint32_t)t < pages;
}
__host__ __device__ inline uint64_t row_element(const CacheView &c, uint32_t page, uint32_t at, uint32_t head)
{
    return page * c.page_stride + at * c.token_stride + head * c.head_stride;
}
__host__ __device__ inline uint64_t scale_element(const CacheView &c, uint32_t page, uint32_t at, uint32_t head)
{
    return ((uint64_t)page * c.kv_heads + head) * c.page_size + at;
}

// [begin, end) of a sequence's tokens: the last `window` (if any) of those that its table has room for.  False: the length is none.
__host__ __device__ inline bool live_tokens(int32_t length, uint32_t table_pages, uint32_t page_size, uint32_t window, uint32_t *begin, uint32_t *end)
{
    const uint64_t room = (uint64_t)table_pages * page_size;
    const bool good = length >= 0 && (uint64_t)length <= room;
    *end = good ? (uint32_t)length : (length < 0 ? 0u : (uint32_t)room);
    *begin = window != 0 && *end > window ? *end - window : 0;
    return good;
}
// Work that stands in a row, cut into n contiguous parts, none empty, of equal length but for one.  (32 bits: a 64-bit
// division takes ten times as long.)
struct Parts {
    uint32_t each, longer, n;   // the first `longer` parts have each + 1
    __host__ __device__ Parts(uint32_t total, uint32_t most)
    {
        n = total < most ? total : most;
        each = n == 0 ? 0 : total / n;
        longer = total - each * n;
    }
    __host__ __device__ uint32_t begin(uint32_t i) const
    {
        return i * each + (i < longer ? i : longer);
    }
    // the part that holds a place
    __host__ __device__ uint32_t of(uint32_t place) const
    {
        const uint32_t border = (each + 1) * longer;
        return place < border ? place / (each + 1) : (place - border) / each + longer;
    }
};
// tiles of 2^shift tokens, on a grid that starts at token 0
__host__ __device__ inline uint32_t tiles_of(uint32_t begin, uint32_t end, uint32_t shift)
{
    return end <= begin ? 0 : ((end - 1) >> shift) - (begin >> shift) + 1;
}

inline bool aligned(const void *p, size_t n)
{
    return reinterpret_cast<uintptr_t>(p) % n == 0;
}
// Strides are described by the caller.  With the first limit 2^32 rows of a call's own stay within 64 bits; what has more than
// that to an index (pages, adapters, tables) is held below the second.
constexpr uint64_t MAX_STRIDE = 1ull << 30, MAX_BYTES = 1ull << 62;

// memory of the GPU that the calling thread's calls run on
bool on_this_device(const void *p);
// everything about a cache that the host can see
EE check_cache(const bolt_b200_kv_cache *cache);
inline CacheView view_of(const bolt_b200_kv_cache &c)
{
    return CacheView{c.pages, c.page_size, c.kv_heads, c.dim, c.page_stride, c.token_stride, c.head_stride};
}

#ifdef __CUDACC__
// A launch judged by its own status, not by the thread's last error: that may be an earlier call's.
template <typename... P, typename... A>
EE launch_kernel(dim3 grid, uint32_t block, size_t smem, cudaStream_t st, void (*kernel)(P...), const A &...args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    B200_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    count_launch();
    return SUCCESS;
}
__device__ __forceinline__ void load4(const float *p, float (&x)[4])
{
    const float4 v = *reinterpret_cast<const float4 *>(p);
    x[0] = v.x;
    x[1] = v.y;
    x[2] = v.z;
    x[3] = v.w;
}
__device__ __forceinline__ void load4(const __half *p, float (&x)[4])
{
    const uint2 v = *reinterpret_cast<const uint2 *>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
    x[0] = a.x;
    x[1] = a.y;
    x[2] = b.x;
    x[3] = b.y;
}
__device__ __forceinline__ void load2(const float *p, float &x, float &y)
{
    const float2 v = *reinterpret_cast<const float2 *>(p);
    x = v.x;
    y = v.y;
}
__device__ __forceinline__ void load2(const __half *p, float &x, float &y)
{
    const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(p));
    x = v.x;
    y = v.y;
}
__device__ __forceinline__ float load1(const float *p)
{
    return *p;
}
__device__ __forceinline__ float load1(const __half *p)
{
    return __half2float(*p);
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
#endif

}  // namespace b200
