// lora.cu -- low-rank adapters of many requests beside a shared projection: y += s (x A^T) B^T for every segment of rows.
//
// HBM bound: with a few rows the adapters' own bytes, with many the result's (read and written once).  Two kernels: the
// inner sums t = x A^T (rows x rank) into the workspace, K split over CTAs and warps, then y += t B^T; where K is short, the
// second alone makes its inner sums, too.  Both work on blocks of 16 rows of one segment, which one instruction of the tensor
// pipe takes at once; with one row to a request 15 of the 16 stand idle, but the weights are streamed all the same.  Operands
// go from global memory straight into the fragments: the order of K inside an instruction is free, so a lane loads 16
// neighbouring bytes of a row of A or B.
//
// Bytes of x become binary16 exactly.  Binary32 x enters as two tf32 numbers (23 bits; tf32 has binary32's range), t as two
// binary16 numbers of rows brought to a common power of two.  The accumulation of the matrix instructions truncates, which adds
// up: what the first number of a pair leaves goes first, while the sum is small, and sums go on in binary32 registers, over K after
// two instructions for the first numbers, over the rank after 64 of it.  Sums of positive products of binary32 numbers come out
// 0.7 to 1.5 2^-23 too small on the average (5 to 14 with all of K that is in flight in one chain), those of any sign are as near
// as binary32 throughout (1.1 to 1.7 2^-23 of the result, in root mean square).
//
// 2048 rows, 8192 -> 28672, rank 16, six requests: 75 to 92 us, 5.1 to 6.3 TB/s of the 470 MB of the result, read and written.  Every 16
// rows read all of A and B, from L2: rank 64 118 us, rank 128 202.  16 rows with an adapter each: 13.3 us, two kernels of dependent
// loads over 23 MB.
#include "decode.cuh"

namespace b200 {
namespace {

struct LoraParams {
    uint32_t rows, N, K, rank, adapters, segments;
    const void *x;
    float *y;
    uint64_t x_stride, y_stride, a_stride;
    const __half *a, *b;
    const float *scale;
    const int32_t *first_row, *adapter;
    float sA;
    const float *d_sA, *row_scale;
    int u8, x_vectors, y_width;   // whether rows of x can be read 8 bytes / 4 numbers at a time; numbers of y: 4, 2 or 1
    bool alone;                           // one kernel does it all
    uint32_t units, splits, outer_ctas;   // blocks of 16 rows at most, parts of K, CTAs of the second kernel
    float *t;   // [splits][rows][rank]
    int *status;
};

constexpr uint32_t MAX_SEGMENTS = 65535;

// ---- blocks of rows -----------------------------------------------------------------------------------------------
struct Unit {
    uint32_t row, rows;   // 0: there is none
    int32_t adapter;
};
// Segment s, given the largest bound in front of it: false if it is left out.
__device__ __forceinline__ bool segment(const LoraParams &p, uint32_t s, int32_t top, int32_t *from, int32_t *to, int32_t *adapter)
{
    *from = p.first_row[s];
    *to = p.first_row[s + 1];
    *adapter = p.adapter[s];
    return *from >= top && *to >= *from && (uint32_t)*to <= p.rows && *adapter < (int32_t)p.adapters;
}
// By 256 threads that share the counting: how many units there are, and which is which.
class Units {
public:
    __device__ __forceinline__ Units(const LoraParams &params, bool report) : p(params)
    {
        __shared__ int32_t tops[8];
        __shared__ uint32_t counts[8];
        const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, per = (p.segments + 255) / 256;
        s0 = min(threadIdx.x * per, p.segments);
        s1 = min(s0 + per, p.segments);
        // the largest bound in front of the thread's first segment
        int32_t upto = 0;
        for (uint32_t s = s0; s < s1; ++s) {
            upto = max(upto, p.first_row[s]);
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int32_t v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
            upto = lane >= o ? max(upto, v) : upto;
        }
        if (lane == 31) {
            tops[warp] = upto;
        }
        __syncthreads();
        top = __shfl_up_sync(0xFFFFFFFFu, upto, 1);
        top = lane == 0 ? 0 : top;
        for (uint32_t w = 0; w < warp; ++w) {
            top = max(top, tops[w]);
        }
        mine = 0;
        walk(report, [&](uint32_t, uint32_t n, int32_t) { mine += (n + 15) / 16; });
        uint32_t sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, sum, o);
            sum += lane >= o ? v : 0;
        }
        if (lane == 31) {
            counts[warp] = sum;
        }
        __syncthreads();
        first = sum - mine;
        total = 0;
        for (uint32_t w = 0; w < 8; ++w) {
            first += w < warp ? counts[w] : 0;
            total += counts[w];
        }
    }
    __device__ __forceinline__ uint32_t count() const
    {
        return total;
    }
    __device__ __forceinline__ Unit get(uint32_t want) const
    {
        __shared__ Unit found;
        if (threadIdx.x == 0) {
            found = Unit{0, 0, 0};
        }
        __syncthreads();
        if (want >= first && want < first + mine) {
            uint32_t before = first;
            walk(false, [&](uint32_t row, uint32_t n, int32_t adapter) {
                const uint32_t blocks = (n + 15) / 16, b = want - before;
                if (want >= before && b < blocks) {
                    found = Unit{row + 16 * b, min(16u, n - 16 * b), adapter};
                }
                before += blocks;
            });
        }
        __syncthreads();
        return found;
    }

private:
    // the thread's segments
    template <typename F>
    __device__ __forceinline__ void walk(bool report, F each) const
    {
        int32_t t = top;
        for (uint32_t s = s0; s < s1; ++s) {
            int32_t from, to, adapter;
            const bool good = segment(p, s, t, &from, &to, &adapter);
            if (!good && report) {
                atomicExch(p.status, BAD_LORA);
            }
            t = max(t, from);
            if (good && adapter >= 0) {
                each((uint32_t)from, (uint32_t)(to - from), adapter);
            }
        }
    }
    const LoraParams &p;
    uint32_t s0, s1, mine, first, total;
    int32_t top;
};

// ---- instructions -----------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)   // c = a b
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f), "f"(0.f), "f"(0.f), "f"(0.f));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)   // c = a b
{
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f), "f"(0.f), "f"(0.f), "f"(0.f));
}
__device__ __forceinline__ void matrices(uint32_t (&r)[4], const void *at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"((uint32_t)__cvta_generic_to_shared(at))
                 : "memory");
}
// two neighbouring bytes u (0: the lower two of a word, 1: the upper two) as u - 128 in binary16: 0x6400 | u is 1024 + u
template <int UPPER>
__device__ __forceinline__ uint32_t centred(uint32_t x)
{
    const uint32_t y = __byte_perm(x, 0x64646464u, UPPER ? 0x4342 : 0x4140), k = 0x64806480u;
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&y), *reinterpret_cast<const __half2 *>(&k));
    return *reinterpret_cast<const uint32_t *>(&h);
}
// A number as the sum of two that the tensor pipe sees whole (tf32: eleven bits), each the nearest: what is left out is 2^-23 of
// it at most.  (What would round to infinity, infinities and NaN are cut off as they stand.)
__device__ __forceinline__ void tf32_pair(float x, uint32_t &hi, uint32_t &lo)
{
    const uint32_t b = __float_as_uint(x), half = (b & 0x7FFFFFFFu) < 0x7F7FF000u ? 0x1000u : 0u;
    hi = (b + half) & 0xFFFFE000u;
    lo = (__float_as_uint(x - __uint_as_float(hi)) + half) & 0xFFFFE000u;
}

__device__ __forceinline__ void add(float (&sum)[4], const float (&c)[4])
{
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        sum[e] += c[e];
    }
}

// ---- inner sums ---------------------------------------------------------------------------------------------------
// eight neighbours of a row of x from k on, zeros (after centring) behind K or for a row that does not exist
template <bool U8>
struct Eight;
template <>
struct Eight<true> {
    uint32_t h[4];   // pairs of binary16
    __device__ __forceinline__ void load(const LoraParams &p, uint64_t row, uint32_t k, bool on)
    {
        uint32_t w[2] = {0x80808080u, 0x80808080u};
        const uint8_t *x = reinterpret_cast<const uint8_t *>(p.x) + row * p.x_stride + k;
        if (on && p.x_vectors && k + 8 <= p.K) {
            const uint2 v = *reinterpret_cast<const uint2 *>(x);
            w[0] = v.x;
            w[1] = v.y;
        } else if (on && k + 8 <= p.K) {
            // the aligned words that hold a byte of the eight, shifted into place
            const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(x) & 3);
            const uint32_t *words = reinterpret_cast<const uint32_t *>(x - off);
            const uint32_t a = words[0], b = words[1], c = off != 0 ? words[2] : 0;
            w[0] = __funnelshift_r(a, b, 8 * off);
            w[1] = __funnelshift_r(b, c, 8 * off);
        } else if (on) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (k + i < p.K) {
                    w[i / 4] = (w[i / 4] & ~(0xFFu << (i % 4 * 8))) | (uint32_t)x[i] << (i % 4 * 8);
                }
            }
        }
        h[0] = w[0];
        h[1] = w[1];
    }
    __device__ __forceinline__ void convert()
    {
        const uint32_t a = h[0], b = h[1];
        h[0] = centred<0>(a);
        h[1] = centred<1>(a);
        h[2] = centred<0>(b);
        h[3] = centred<1>(b);
    }
};
template <>
struct Eight<false> {
    float f[8];
    __device__ __forceinline__ void load(const LoraParams &p, uint64_t row, uint32_t k, bool on)
    {
        const float *x = reinterpret_cast<const float *>(p.x) + row * p.x_stride + k;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            f[i] = 0.f;
        }
        if (on && p.x_vectors && k + 8 <= p.K) {
            const float4 u = *reinterpret_cast<const float4 *>(x), v = reinterpret_cast<const float4 *>(x)[1];
            f[0] = u.x;
            f[1] = u.y;
            f[2] = u.z;
            f[3] = u.w;
            f[4] = v.x;
            f[5] = v.y;
            f[6] = v.z;
            f[7] = v.w;
        } else if (on) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (k + i < p.K) {
                    f[i] = x[i];
                }
            }
        }
    }
};

// sum += sixteen rows x eight neighbours of rows of A (each lane's)
template <int NT>
__device__ __forceinline__ void add_products(Eight<true> &x0, Eight<true> &x1, const uint4 (&a)[NT], float (&sum)[NT][4])
{
    x0.convert();
    x1.convert();
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float c[4];
        mma_f16_first(c, x0.h[0], x1.h[0], x0.h[1], x1.h[1], a[n].x, a[n].y);
        mma_f16(c, x0.h[2], x1.h[2], x0.h[3], x1.h[3], a[n].z, a[n].w);
        add(sum[n], c);
    }
}
template <int NT>
__device__ __forceinline__ void add_products(const Eight<false> &x0, const Eight<false> &x1, const uint4 (&a)[NT], float (&sum)[NT][4])
{
#pragma unroll
    for (int e = 0; e < 8; e += 4) {     // two instructions' worth: first what the first parts leave, while the sum is small
        uint32_t hi[2][4], lo[2][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            tf32_pair(x0.f[e + i], hi[i / 2][i % 2 * 2], lo[i / 2][i % 2 * 2]);
            tf32_pair(x1.f[e + i], hi[i / 2][i % 2 * 2 + 1], lo[i / 2][i % 2 * 2 + 1]);
        }
        constexpr int GROUP = NT < 8 ? NT : 8;    // instructions that do not wait for one another
#pragma unroll
        for (int n0 = 0; n0 < NT; n0 += GROUP) {
            float c[GROUP][4];
            auto multiply = [&](const uint32_t (&x)[4], int n, int i, bool first) {
                const uint4 &w = a[n0 + n];
                const uint32_t h = e == 0 ? (i == 0 ? w.x : w.y) : (i == 0 ? w.z : w.w);
                const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&h));
                if (first) {
                    mma_tf32_first(c[n], x[0], x[1], x[2], x[3], __float_as_uint(b.x), __float_as_uint(b.y));
                } else {
                    mma_tf32(c[n], x[0], x[1], x[2], x[3], __float_as_uint(b.x), __float_as_uint(b.y));
                }
            };
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int n = 0; n < GROUP; ++n) {
                    multiply(i < 2 ? lo[i] : hi[i - 2], n, i % 2, i == 0);
                }
            }
#pragma unroll
            for (int n = 0; n < GROUP; ++n) {
                add(sum[n0 + n], c[n]);
            }
        }
    }
}

// By the 256 threads of a CTA: the sums over blocks from .. to - 1 of 32 of K for the rows of a unit, times their scales, in warp 0: sum
// [n][0, 1] for row g and columns 8 n + 2 c4 and the next, [2, 3] for row g + 8.  NT: blocks of eight of the rank, rounded up.
template <bool U8, int NT>
__device__ __forceinline__ void inner_sums(const LoraParams &p, const Unit &u, uint32_t from, uint32_t to, float (*merge)[NT * 4 * 32], float (&sum)[NT][4])
{
    constexpr int AT_ONCE = NT <= 2 ? 4 : (NT <= 4 ? 2 : 1);   // blocks of 32 of K whose loads a warp has in flight (divide() knows)
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, c4 = lane % 4;
    const __half *a = p.a + (uint64_t)u.adapter * p.rank * p.a_stride + g * p.a_stride + 8 * c4;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        sum[n][0] = sum[n][1] = sum[n][2] = sum[n][3] = 0.f;
    }
#pragma unroll 1
    for (uint32_t kb = from + warp; kb < to; kb += 8 * AT_ONCE) {
        uint4 w[AT_ONCE][NT];
        Eight<U8> x[AT_ONCE][2];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const uint32_t b = kb + 8 * i, k = 32 * b + 8 * c4;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                w[i][n] = make_uint4(0, 0, 0, 0);
                if (b < to && n * 8 < p.rank && k < p.K) {
                    w[i][n] = *reinterpret_cast<const uint4 *>(a + n * 8 * p.a_stride + 32 * b);
                }
            }
            x[i][0].load(p, u.row + g, k, b < to && k < p.K && g < u.rows);
            x[i][1].load(p, u.row + g + 8, k, b < to && k < p.K && g + 8 < u.rows);
        }
        __syncwarp();       // (matrix instructions take a warp as a whole, and come behind branches that some lanes have taken)
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const uint32_t k = 32 * (kb + 8 * i) + 8 * c4;
            if (k + 8 > p.K) {   // what lies behind K in a row of A is nobody's
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    uint32_t h[4] = {w[i][n].x, w[i][n].y, w[i][n].z, w[i][n].w};
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        if (k + e >= p.K) {
                            h[e / 2] &= e % 2 ? 0x0000FFFFu : 0xFFFF0000u;
                        }
                    }
                    w[i][n] = make_uint4(h[0], h[1], h[2], h[3]);
                }
            }
            add_products(x[i][0], x[i][1], w[i], sum);
        }
    }
    // the warps' shares, the upper half's added to the lower half's, and so on
#pragma unroll 1
    for (uint32_t half = 4; half != 0; half /= 2) {
        if (warp >= half && warp < 2 * half) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    merge[warp - half][(4 * n + e) * 32 + lane] = sum[n][e];
                }
            }
        }
        __syncthreads();
        if (warp < half) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sum[n][e] += merge[warp][(4 * n + e) * 32 + lane];
                }
            }
        }
        __syncthreads();
    }
    if (warp == 0) {
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            if (g + 8 * r < u.rows) {
                const uint32_t row = u.row + g + 8 * r;
                float factor = p.scale != nullptr ? p.scale[u.adapter] : 1.f;
                if (U8) {
                    factor = __fdiv_rn(factor, p.row_scale != nullptr ? p.row_scale[row] : (p.d_sA != nullptr ? *p.d_sA : p.sA));
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    sum[n][2 * r] *= factor;
                    sum[n][2 * r + 1] *= factor;
                }
            }
        }
    }
}
// (Binary32 x with ranks of 17 to 64: a few registers above half of them all without the bound; 2048 rows of rank 64 130 us, 149
// without.)
template <bool U8, int NT>
__global__ void __launch_bounds__(256, !U8 && (NT == 4 || NT == 8) ? 2 : 0) lora_inner_kernel(const __grid_constant__ LoraParams p)
{
    __shared__ float merge[4][NT * 4 * 32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // (what was in front of this kernel is over)
    const Units units(p, blockIdx.x == 0 && blockIdx.y == 0);
    if (blockIdx.x >= units.count()) {
        return;
    }
    const Unit u = units.get(blockIdx.x);
    const uint32_t blocks = (p.K + 31) / 32;
    float sum[NT][4];
    inner_sums<U8, NT>(p, u, (uint32_t)((uint64_t)blocks * blockIdx.y / p.splits), (uint32_t)((uint64_t)blocks * (blockIdx.y + 1) / p.splits), merge, sum);
    if (threadIdx.x >= 32) {
        return;
    }
    const uint32_t g = threadIdx.x / 4, c4 = threadIdx.x % 4;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        if (g + 8 * r < u.rows) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (n * 8 < p.rank) {
                    *reinterpret_cast<float2 *>(p.t + ((uint64_t)blockIdx.y * p.rows + u.row + g + 8 * r) * p.rank + n * 8 + 2 * c4) =
                        make_float2(sum[n][2 * r], sum[n][2 * r + 1]);
                }
            }
        }
    }
}

// ---- the result -----------------------------------------------------------------------------------------------------
// The rank in blocks of 32, then 16, then 8: a lane loads 8, 4 or 2 neighbours of a row of B, and t stands in shared memory in
// the order in which the instruction then meets them.
__device__ __forceinline__ uint32_t place_of(uint32_t r, uint32_t rank)
{
    const uint32_t b = r & ~31u, left = rank - b, i = r - b;
    if (left >= 32) {
        return b + i % 8 / 4 * 16 + i / 8 * 2 + i % 2 + i % 4 / 2 * 8;
    }
    if (left >= 16 && i < 16) {
        return b + i / 4 * 2 + i % 2 + i % 4 / 2 * 8;
    }
    return r;
}
// Columns go in steps of 256 (32 to a warp); the steps of all units stand in one row, of which every CTA takes an equal part.
constexpr uint32_t STEP = 256;
// KS: blocks of 16 of the rank, rounded up.  ALONE: there is no lora_inner_kernel in front, every CTA makes the inner sums of its
// rows by itself (divide() says when); binary32 x takes all registers of one CTA for that.
enum Alone { NOT_ALONE, ALONE_F32, ALONE_U8 };
template <int KS, Alone ALONE>
__global__ void __launch_bounds__(256, ALONE ? (ALONE == ALONE_U8 ? 2 : 1) : (KS <= 1 ? 4 : (KS <= 2 ? 3 : 2))) lora_outer_kernel(const __grid_constant__ LoraParams p)
{
    constexpr int PITCH = KS * 16 + 8, TILES = 4;   // columns of a warp at a time: 4 x 8
    constexpr int AT_ONCE = KS <= 2 ? 8 : 4;        // parts of K whose inner sums are asked for at a time
    __shared__ __align__(16) __half hi[16][PITCH], lo[16][PITCH];
    __shared__ float down[16];
    __shared__ float merge[ALONE ? 4 : 1][ALONE ? KS * 2 * 4 * 32 : 1], inner[ALONE ? 16 : 1][ALONE ? KS * 16 + 2 : 1];
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, c4 = lane % 4;
    for (uint32_t i = threadIdx.x; i < 16 * PITCH; i += 256) {
        (&hi[0][0])[i] = (&lo[0][0])[i] = __float2half_rn(0.f);
    }
    if (ALONE) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
    }
    // (nothing that lora_inner_kernel, in front of this one, writes is read here: it writes the inner sums only, and has seen
    // the end of what was in front of it)
    const Units units(p, ALONE && blockIdx.x == 0);
    const uint32_t steps = (p.N + STEP - 1) / STEP;
    const Parts parts(units.count() * steps, gridDim.x);
    const bool some = blockIdx.x < parts.n;
    uint32_t at = some ? parts.begin(blockIdx.x) : 0;
    const uint32_t stop = some ? parts.begin(blockIdx.x + 1) : 0;

    Unit u = {0, 0, 0};
    uint32_t w[TILES][KS][2];
    float v[2][TILES / 2][4];
    // The order of the columns inside an instruction is free, too: those of two tiles are dealt out so that a lane has four
    // neighbours of the result (and rows g / 2 * 4 + g % 2 of B, and the one two further on, and so on).
    uint32_t step = 0, n0 = 0;      // of the unit; the warp's first column of the step
    float *y0 = nullptr, *y1 = nullptr;
    const __half *b = nullptr;
    bool on0 = false, on1 = false;
    auto enter = [&]() {
        u = units.get(at / steps);
        step = at % steps;
        n0 = step * STEP + warp * 8 * TILES;
        y0 = p.y + (uint64_t)(u.row + g) * p.y_stride + n0 + 4 * c4;
        y1 = y0 + 8 * p.y_stride;
        b = p.b + ((uint64_t)u.adapter * p.N + n0 + g / 2 * 4 + g % 2) * p.rank;
        on0 = g < u.rows;
        on1 = g + 8 < u.rows;
    };
    auto advance = [&]() {
        ++step;
        n0 += STEP;
        y0 += STEP;
        y1 += STEP;
        b += (uint64_t)STEP * p.rank;
    };
    auto whole = [&]() { return n0 + 8 * TILES <= p.N; };    // no column to look after
    // four neighbours of a row of y
    auto load_y = [&](const float *y, float (&x)[4]) {
        if (p.y_width == 4) {
            const float4 a = __ldcs(reinterpret_cast<const float4 *>(y));
            x[0] = a.x;
            x[1] = a.y;
            x[2] = a.z;
            x[3] = a.w;
        } else if (p.y_width == 2) {
            const float2 a = __ldcs(reinterpret_cast<const float2 *>(y)), b = __ldcs(reinterpret_cast<const float2 *>(y) + 1);
            x[0] = a.x;
            x[1] = a.y;
            x[2] = b.x;
            x[3] = b.y;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = __ldcs(y + e);
            }
        }
    };
    auto store_y = [&](float *y, const float (&x)[4]) {
        if (p.y_width == 4) {
            __stcs(reinterpret_cast<float4 *>(y), make_float4(x[0], x[1], x[2], x[3]));
        } else if (p.y_width == 2) {
            __stcs(reinterpret_cast<float2 *>(y), make_float2(x[0], x[1]));
            __stcs(reinterpret_cast<float2 *>(y) + 1, make_float2(x[2], x[3]));
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                __stcs(y + e, x[e]);
            }
        }
    };
    // (Where this kernel starts behind lora_inner_kernel nothing that may write B still runs.  Alone it starts beside the end of what is
    // in front of it: memory is no read-only memory then.  As plain loads, which stay behind the stores of the step before,
    // 2048 rows of rank 128 take 246 us, not 213.)
    auto weights = [](const auto *at) {
        if constexpr (ALONE) {
            return *at;
        } else {
            return __ldg(at);
        }
    };
    auto fetch_row = [&](int t, const __half *row, bool on) {
        if (KS == 1 && on && p.rank == 16) {
            const uint2 x = weights(reinterpret_cast<const uint2 *>(row + 4 * c4));
            w[t][0][0] = x.x;
            w[t][0][1] = x.y;
            return;
        }
#pragma unroll
        for (int s = 0; s < KS; s += 2) {
            uint32_t q[4] = {0, 0, 0, 0};
            const uint32_t left = p.rank - 16 * s;
            if (on && 16 * s < p.rank) {
                if (KS > 1 && left >= 32) {
                    const uint4 x = weights(reinterpret_cast<const uint4 *>(row + 16 * s + 8 * c4));
                    q[0] = x.x;
                    q[1] = x.y;
                    q[2] = x.z;
                    q[3] = x.w;
                } else {
                    uint32_t r = 16 * s;
                    if (left >= 16) {
                        const uint2 x = weights(reinterpret_cast<const uint2 *>(row + r + 4 * c4));
                        q[0] = x.x;
                        q[1] = x.y;
                        r += 16;
                    }
                    if (left % 16 == 8) {
                        const uint32_t x = weights(reinterpret_cast<const uint32_t *>(row + r + 2 * c4));
                        q[left >= 16 ? 2 : 0] = x;
                    }
                }
            }
            w[t][s][0] = q[0];
            w[t][s][1] = q[1];
            if (s + 1 < KS) {
                w[t][s + 1][0] = q[2];
                w[t][s + 1][1] = q[3];
            }
        }
    };
    auto fetch = [&]() {
        if (whole()) {
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                fetch_row(t, b + (t / 2 * 16 + t % 2 * 2) * p.rank, true);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
                for (int t = 0; t < TILES / 2; ++t) {
                    v[r][t][0] = v[r][t][1] = v[r][t][2] = v[r][t][3] = 0.f;
                    if (r == 0 ? on0 : on1) {
                        load_y((r == 0 ? y0 : y1) + 16 * t, v[r][t]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                const uint32_t further = t / 2 * 16 + t % 2 * 2;
                fetch_row(t, b + further * p.rank, n0 + g / 2 * 4 + g % 2 + further < p.N);
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
                for (int t = 0; t < TILES / 2; ++t) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t further = 16 * t + e;
                        v[r][t][e] = (r == 0 ? on0 : on1) && n0 + 4 * c4 + further < p.N ? (r == 0 ? y0 : y1)[further] : 0.f;
                    }
                }
            }
        }
    };
    if (at < stop) {
        enter();
        fetch();    // on its way while the inner sums are still being made
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (!ALONE) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
    }
#pragma unroll 1
    while (at < stop) {
        if constexpr (ALONE) {
            float sum[KS * 2][4];
            inner_sums<ALONE == ALONE_U8, KS * 2>(p, u, 0, (p.K + 31) / 32, merge, sum);
            if (warp == 0) {
#pragma unroll
                for (int n = 0; n < KS * 2; ++n) {
                    *reinterpret_cast<float2 *>(&inner[g][n * 8 + 2 * c4]) = make_float2(sum[n][0], sum[n][1]);
                    *reinterpret_cast<float2 *>(&inner[g + 8][n * 8 + 2 * c4]) = make_float2(sum[n][2], sum[n][3]);
                }
            }
        }
        __syncthreads();    // everybody is through with the unit before (and the zeros are there)
        {
            // sixteen threads to a row
            const uint32_t row = threadIdx.x / 16, l = threadIdx.x % 16;
            float x[KS];
            int top = 0;
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                x[i] = 0.f;
            }
            if (ALONE) {
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    x[i] = l + 16 * i < p.rank ? inner[row][l + 16 * i] : 0.f;
                }
            } else if (row < u.rows) {
                const float *t = p.t + (uint64_t)(u.row + row) * p.rank;
                const uint64_t split = (uint64_t)p.rows * p.rank;
#pragma unroll 1
                for (uint32_t s = 0; s < p.splits; s += AT_ONCE) {
                    float part[AT_ONCE][KS];
#pragma unroll
                    for (int j = 0; j < AT_ONCE; ++j) {
#pragma unroll
                        for (int i = 0; i < KS; ++i) {
                            part[j][i] = s + j < p.splits && l + 16 * i < p.rank ? __ldcg(t + (s + j) * split + l + 16 * i) : 0.f;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < AT_ONCE; ++j) {
#pragma unroll
                        for (int i = 0; i < KS; ++i) {
                            x[i] += part[j][i];
                        }
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                top = max(top, magnitude(x[i]));
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) {
                top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
            }
            const int e = max(top >> 23, 20);   // to 2^13 .. 2^14
            const float up = __int_as_float((267 - e) << 23);
            if (l == 0) {
                down[row] = __int_as_float((e - 13) << 23);
            }
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                const uint32_t r = l + 16 * i;
                if (r < p.rank) {
                    const uint32_t to = place_of(r, p.rank);
                    const float scaled = x[i] * up;
                    const __half h = __float2half_rn(scaled);
                    hi[row][to] = h;
                    lo[row][to] = __float2half_rn(scaled - __half2float(h));
                }
            }
        }
        __syncthreads();
        // t's fragments: in registers, or (larger ranks) read again for every step
        constexpr bool KEPT = KS <= 2;
        uint32_t th[KEPT ? KS : 1][4], tl[KEPT ? KS : 1][4];
        auto fragment = [&](uint32_t (&r)[4], const __half (&of)[16][PITCH], int s) { matrices(r, &of[lane % 16][16 * s + lane / 16 * 8]); };
        if constexpr (KEPT) {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                fragment(th[s], hi, s);
                fragment(tl[s], lo, s);
            }
        }
        const float down0 = down[g], down1 = down[g + 8];
#pragma unroll 1
        for (;;) {
            __syncwarp();
            // The instruction's own accumulation truncates: what binary16 has cut off of t goes first, while the sums are small, and
            // every 16 * FOLD of the rank the sums go on in binary32.
            constexpr int FOLD = KS < 4 ? KS : 4;
#pragma unroll
            for (int s0 = 0; s0 < KS; s0 += FOLD) {
                float c[TILES][4];
#pragma unroll
                for (int i = 0; i < 2 * FOLD; ++i) {
                    const int s = s0 + i % FOLD;
                    uint32_t a[4];
                    if constexpr (KEPT) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            a[e] = i < FOLD ? tl[s][e] : th[s][e];
                        }
                    } else {
                        fragment(a, i < FOLD ? lo : hi, s);
                    }
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        if (i == 0) {
                            mma_f16_first(c[t], a[0], a[1], a[2], a[3], w[t][s][0], w[t][s][1]);
                        } else {
                            mma_f16(c[t], a[0], a[1], a[2], a[3], w[t][s][0], w[t][s][1]);
                        }
                    }
                }
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        v[0][t / 2][t % 2 * 2 + e] = fmaf(c[t][e], down0, v[0][t / 2][t % 2 * 2 + e]);
                        v[1][t / 2][t % 2 * 2 + e] = fmaf(c[t][2 + e], down1, v[1][t / 2][t % 2 * 2 + e]);
                    }
                }
            }
            const bool all = whole();
#pragma unroll
            for (int r = 0; r < 2; ++r) {
#pragma unroll
                for (int t = 0; t < TILES / 2; ++t) {
                    if (!(r == 0 ? on0 : on1)) {
                        continue;
                    }
                    float *y = (r == 0 ? y0 : y1) + 16 * t;
                    if (all) {
                        store_y(y, v[r][t]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (n0 + 4 * c4 + 16 * t + e < p.N) {
                                y[e] = v[r][t][e];
                            }
                        }
                    }
                }
            }
            advance();
            if (++at == stop || step == steps) {
                break;
            }
            fetch();
        }
        if (at < stop) {
            enter();
            fetch();
        }
    }
}

// How the work is divided: from what the host knows, the rows and the number of segments.
void divide(LoraParams *p, const DeviceCtx *c)
{
    const uint32_t most = p->rows / 16 + p->segments, sms = (uint32_t)c->sm_count;
    p->units = most < p->rows ? most : p->rows;
    // K in as many parts as give every SM four CTAs (2048 rows of 8192: 86.5 us, with two 87.0, with eight 88.3), each at least
    // as long as what a CTA asks for at a time, and sixteen at most, which the second kernel asks for in two goes.
    // 16 rows of 8192 with adapters of rank 16: 13.3 us in 8 parts of 1024, 14.5 in 16, 18.9 in 32, 13.6 in 4; one row of 28672: 8.1
    // in 16 parts, 9.4 in 8; 16 rows with one adapter of rank 128: 23.5 and 30.5.
    const uint32_t at_a_time = p->rank <= 16 ? 1024 : (p->rank <= 32 ? 512 : 256);
    const uint32_t want = p->units == 0 ? 1 : 4 * sms / p->units, at_most = (p->K - 1) / at_a_time + 1;
    p->splits = want < 1 ? 1 : (want < at_most ? want : at_most);
    p->splits = p->splits < 16 ? p->splits : 16;
    const uint64_t steps = (uint64_t)p->units * ((p->N + STEP - 1) / STEP), by_itself = (uint64_t)sms * (p->u8 ? 2 : 1);
    // One kernel, in which every CTA makes its rows' inner sums, where they take no more than one go and few CTAs meet a second
    // unit: 16 rows of 768 -> 768 6.3 us in place of 7.4 (binary32), 5.5 in place of 6.5 (bytes).  With four goes 16 rows of
    // 4096 -> 4096 take 12.6 in place of 8.0, and 1024 rows of 768 -> 2304 with eight adapters 13.0 in place of 12.7.
    p->alone = p->rank <= 32 && p->K <= at_a_time && steps <= 2 * by_itself;
    // as many CTAs as run at a time, and no more than there are steps
    const uint64_t ctas = p->alone ? by_itself : (uint64_t)sms * (p->rank <= 16 ? 4 : (p->rank <= 32 ? 3 : 2));
    p->outer_ctas = (uint32_t)(steps < ctas ? steps : ctas);
}
EE check(const bolt_b200_lora_call *a, LoraParams *p, DeviceCtx **c)
{
    if (a == nullptr) {
        return NULL_POINTER;
    }
    *c = ctx();
    if (*c == nullptr) {
        return UNKNOWN;
    }
    if (a->x_dt != DT_F32 && a->x_dt != DT_U8_Q) {
        return NOT_SUPPORTED;
    }
    if (a->K == 0 || a->N == 0 || a->adapters == 0 || a->a_stride < a->K) {
        return NOT_MATCH;
    }
    if (a->rank == 0 || a->rank % 8 != 0 || a->rank > 128 || a->a_stride % 8 != 0) {
        return NOT_SUPPORTED;
    }
    if (a->rows > 1 && (a->x_stride < a->K || a->y_stride < a->N)) {
        return NOT_MATCH;
    }
    if (a->x_stride > MAX_STRIDE || a->y_stride > MAX_STRIDE || a->a_stride > MAX_STRIDE || a->rows > (1u << 22) || a->N > (1u << 23) ||
        a->adapters > 0x7FFFFFFFu || a->segments > MAX_SEGMENTS || (unsigned __int128)a->adapters * a->rank * a->a_stride * 2 > MAX_BYTES) {
        return NOT_SUPPORTED;
    }
    p->rows = a->rows;
    p->N = a->N;
    p->K = a->K;
    p->rank = a->rank;
    p->adapters = a->adapters;
    p->segments = a->segments;
    p->x = a->x;
    p->y = a->y;
    p->x_stride = a->x_stride;
    p->y_stride = a->y_stride;
    p->a_stride = a->a_stride;
    p->a = reinterpret_cast<const __half *>(a->a);
    p->b = reinterpret_cast<const __half *>(a->b);
    p->scale = a->scale;
    p->first_row = a->first_row;
    p->adapter = a->adapter;
    p->sA = a->sA;
    p->d_sA = a->d_sA;
    p->row_scale = a->row_scale;
    p->u8 = a->x_dt == DT_U8_Q;
    p->x_vectors = p->u8 ? aligned(a->x, 8) && a->x_stride % 8 == 0 : aligned(a->x, 16) && a->x_stride % 4 == 0;
    p->y_width = aligned(a->y, 16) && a->y_stride % 4 == 0 ? 4 : (aligned(a->y, 8) && a->y_stride % 2 == 0 ? 2 : 1);
    p->status = (*c)->d_status;
    divide(p, *c);
    if ((uint64_t)p->splits * p->rows * p->rank > 0x3FFFFFFFull || (uint64_t)p->units * ((p->N + STEP - 1) / STEP) > 0xFFFFFFFFull) {
        return NOT_SUPPORTED;    // the workspace and the steps are counted in 32 bits
    }
    return SUCCESS;
}
U32 workspace_bytes(const LoraParams &p)
{
    return p.splits * p.rows * p.rank * 4;
}
template <typename K>
EE launch(K kernel, dim3 grid, const LoraParams &p, cudaStream_t st)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    B200_CUDA(launch_programmatic(cfg, kernel, p));
    count_launch();
    return SUCCESS;
}
template <bool U8>
EE launch_inner(const LoraParams &p, cudaStream_t st)
{
    const dim3 grid(p.units, p.splits);
    if (p.rank <= 16) {
        return launch(lora_inner_kernel<U8, 2>, grid, p, st);
    }
    if (p.rank <= 32) {
        return launch(lora_inner_kernel<U8, 4>, grid, p, st);
    }
    return p.rank <= 64 ? launch(lora_inner_kernel<U8, 8>, grid, p, st) : launch(lora_inner_kernel<U8, 16>, grid, p, st);
}
template <Alone ALONE>
EE launch_outer(const LoraParams &p, cudaStream_t st)
{
    const dim3 grid(p.outer_ctas);
    if (p.rank <= 16) {
        return launch(lora_outer_kernel<1, ALONE>, grid, p, st);
    }
    if (ALONE || p.rank <= 32) {
        return launch(lora_outer_kernel<2, ALONE>, grid, p, st);
    }
    if constexpr (ALONE == NOT_ALONE) {
        return p.rank <= 64 ? launch(lora_outer_kernel<4, ALONE>, grid, p, st) : launch(lora_outer_kernel<8, ALONE>, grid, p, st);
    }
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

EE bolt_b200_lora_tmp_bytes(const bolt_b200_lora_call *call, U32 *bytes)
{
    if (bytes == nullptr) {
        return NULL_POINTER;
    }
    LoraParams p;
    DeviceCtx *c = nullptr;
    B200_EE(check(call, &p, &c));
    *bytes = workspace_bytes(p);
    return SUCCESS;
}

EE bolt_b200_lora(const bolt_b200_lora_call *call, U32 tmpBytes, void *tmp)
{
    LoraParams p;
    DeviceCtx *c = nullptr;
    B200_EE(check(call, &p, &c));
    if (p.rows == 0 || p.segments == 0) {
        return SUCCESS;
    }
    if (p.x == nullptr || p.y == nullptr || p.a == nullptr || p.b == nullptr || p.first_row == nullptr || p.adapter == nullptr || tmp == nullptr) {
        return NULL_POINTER;
    }
    if (tmpBytes < workspace_bytes(p)) {
        return NOT_MATCH;
    }
    if (!aligned(p.x, p.u8 ? 1 : 4) || !aligned(p.y, 4) || !aligned(p.a, 16) || !aligned(p.b, 16) || !aligned(p.scale, 4) || !aligned(p.first_row, 4) ||
        !aligned(p.adapter, 4) || !aligned(p.d_sA, 4) || !aligned(p.row_scale, 4) || !aligned(tmp, 16)) {
        return NOT_SUPPORTED;
    }
    if (!on_this_device(p.x) || !on_this_device(p.y) || !on_this_device(p.a) || !on_this_device(p.b) || !on_this_device(p.first_row) ||
        !on_this_device(p.adapter) || !on_this_device(tmp) || (p.scale != nullptr && !on_this_device(p.scale)) ||
        (p.d_sA != nullptr && !on_this_device(p.d_sA)) || (p.row_scale != nullptr && !on_this_device(p.row_scale))) {
        return NOT_MATCH;
    }
    p.t = reinterpret_cast<float *>(tmp);
    const cudaStream_t st = tls().stream;
    if (p.alone) {
        return p.u8 ? launch_outer<ALONE_U8>(p, st) : launch_outer<ALONE_F32>(p, st);
    }
    B200_EE(p.u8 ? launch_inner<true>(p, st) : launch_inner<false>(p, st));
    return launch_outer<NOT_ALONE>(p, st);
}

}  // extern "C"
