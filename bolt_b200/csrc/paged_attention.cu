// paged_attention.cu -- attention of one new token per sequence over a paged cache.
//
// out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m), s_t = scale q . k_t, in one pass over the tokens with a running maximum
// m: when it rises, what has been summed so far is scaled down.  Shares of a sequence are joined the same way.
//
// HBM bound: keys and values are read once, whatever the number of query heads, and everything else is small beside them.
// One CTA per SM takes an equal part of all tokens of the batch (which the host does not know), cut where it may be; a
// second kernel joins the units that were cut.  Inside a CTA every warp streams tokens of its own through a private
// ring of asynchronous copies and keeps its own maximum, total and sums, so that warps meet only at the end of a unit.
// The products run on mma.m16n8k16: eight query heads that share a key head are half a tile's rows, and the other half
// holds what binary16 has cut off of them, so that one instruction per operand tile multiplies 22-bit queries (and
// probabilities) with the cache's binary16; bytes become binary16 in registers, two instructions for two of them.
#include <type_traits>

#include "decode.cuh"

namespace b200 {
namespace {

struct AttentionParams {
    CacheView cache;
    const void *k, *v;
    const float *k_scale, *v_scale;
    const void *q;
    void *out;
    float *lse;
    uint64_t q_stride, out_stride;
    const int32_t *table, *length;
    uint32_t sequences, heads, group, head_blocks, table_pages, window;
    float scale, out_scale;
    int i8, q_f16, out_kind;   // 0 binary32, 1 binary16, 2 u8
    float *parts;   // workspace: two partial results for every CTA
    int *status;
};

__device__ __forceinline__ bool live_tokens(const AttentionParams &p, uint32_t sequence, uint32_t *begin, uint32_t *end)
{
    return b200::live_tokens(p.length[sequence], p.table_pages, p.cache.page_size, p.window, begin, end);
}

__device__ __forceinline__ void store_out(const AttentionParams &p, uint64_t at, float x)
{
    if (p.out_kind == 0) {
        reinterpret_cast<float *>(p.out)[at] = x;
    } else if (p.out_kind == 1) {
        reinterpret_cast<__half *>(p.out)[at] = __float2half_rn(x);
    } else {
        // as quantize_cuda_b200, F32 -> U8_Q
        reinterpret_cast<uint8_t *>(p.out)[at] = (uint8_t)min(255, max(1, cvt_rne_x86(__fadd_rn(__fmul_rn(x, p.out_scale), 128.0f))));
    }
}

// ---- how the work is divided -----------------------------------------------------------------------------------
// A unit is one sequence, key head and block of query heads; it has tiles of WARPS x STEP tokens on a grid that starts at
// token 0.  All units' tiles stand in one row, in which every CTA takes an equal, contiguous part.
// By all THREADS threads of a CTA: the row's length, and the sequence that holds a place of it (place_of(length), if that is
// within the row) with that sequence's own first place.  sums[32] and *found are shared memory.
struct Found {
    uint32_t sequence;
    uint64_t first;
};
template <int THREADS, typename F>
__device__ __forceinline__ uint64_t locate(const AttentionParams &p, uint32_t units, uint32_t tile_tokens, bool report, uint64_t *sums, Found *found, F place_of)
{
    const uint32_t per = (p.sequences + THREADS - 1) / THREADS;
    const uint32_t s0 = min(threadIdx.x * per, p.sequences), s1 = min(s0 + per, p.sequences);
    uint64_t own = 0;
    for (uint32_t s = s0; s < s1; ++s) {
        uint32_t begin, end;
        if (!live_tokens(p, s, &begin, &end) && report) {
            atomicExch(p.status, BAD_ATTENTION);
        }
        own += tiles_of(begin, end, tile_tokens);
    }
    own *= units;
    uint64_t upto = own;
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        upto += lane >= o ? v : 0;
    }
    if (lane == 31) {
        sums[warp] = upto;
    }
    if (threadIdx.x == 0) {   // (always something inside the arrays, even if lengths change under the call)
        found->sequence = 0;
        found->first = 0;
    }
    __syncthreads();
    uint64_t total = 0;
    for (uint32_t w = 0; w < THREADS / 32; ++w) {
        upto += w < warp ? sums[w] : 0;
        total += sums[w];
    }
    const uint64_t place = total != 0 ? place_of(total) : 0;
    uint64_t first = upto - own;
    if (place >= first && place < upto) {
        for (uint32_t s = s0; s < s1; ++s) {
            uint32_t begin, end;
            live_tokens(p, s, &begin, &end);
            const uint64_t n = (uint64_t)tiles_of(begin, end, tile_tokens) * units;
            if (place < first + n) {
                found->sequence = s;
                found->first = first;
                break;
            }
            first += n;
        }
    }
    __syncthreads();
    return total;
}
// By a warp: the first sequence behind `sequence` that has a token (there is one).
__device__ __forceinline__ uint32_t next_sequence(const AttentionParams &p, uint32_t sequence)
{
    for (uint32_t s = sequence + 1;; s += 32) {
        const uint32_t mine = s + threadIdx.x % 32;
        uint32_t begin = 0, end = 0;
        if (mine < p.sequences) {
            live_tokens(p, mine, &begin, &end);
        }
        const uint32_t some = __ballot_sync(0xFFFFFFFFu, end != 0);
        if (some != 0) {
            return s + __ffs(some) - 1;
        }
        if (s >= p.sequences) {
            return p.sequences - 1;    // (lengths that change under the call: anything inside the arrays)
        }
    }
}

// ---- instructions -------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_at(const void *p)
{
    return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, uint32_t bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void *src, uint32_t bytes)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void matrices(uint32_t (&r)[4], uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void matrices_t(uint32_t (&r)[4], uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float reciprocal(float x)    // within 2^-23
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Bytes 0 and 2 (shift 0) or 1 and 3 (shift 8) of a word, as signed numbers, in binary16: 0x6400 is 1024, whose last ten bits
// count ones, so 0x6400 | (byte ^ 0x80) is 1152 + byte.
template <int SHIFT>
__device__ __forceinline__ uint32_t bytes_to_half2(uint32_t x)
{
    const uint32_t y = ((x >> SHIFT) & 0x00FF00FFu) ^ 0x64806480u, k = 0x64806480u;
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&y), *reinterpret_cast<const __half2 *>(&k));
    return *reinterpret_cast<const uint32_t *>(&h);
}
// a pair of numbers as the sum of two pairs of binary16: 22 bits
__device__ __forceinline__ void split_pair(float x, float y, uint32_t &hi, uint32_t &lo)
{
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t *>(&h);
    lo = half2_bits(x - f.x, y - f.y);
}

constexpr int WARPS = 8, MAX_PARTS = 256;
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// DP: elements of a row, rounded up; HB: blocks of eight query heads
template <int DP, bool I8, int HB>
struct Shape {
    static constexpr int SIZE = I8 ? 1 : 2, ROW = DP * SIZE, PITCH = ROW + 16;   // an odd number of 16-byte pieces: ldmatrix meets every bank once
    static constexpr int STEP = ROW <= 128 ? 32 : 16;                            // tokens that a warp takes at a time
    static constexpr uint32_t ALL = STEP == 32 ? 0xFFFFFFFFu : 0xFFFFu;
    static constexpr int SLOT = STEP * PITCH + (I8 ? STEP * 4 : 0);
    static constexpr int HEADS = 8 * HB, COLS = 64 / HB;
    static constexpr int Q_PITCH = DP * 2 + 16, Q_BYTES = 2 * HEADS * Q_PITCH;
    static constexpr int MERGE = WARPS * HEADS * (COLS + 4) * 4;
    static constexpr int FIXED = Q_BYTES + MERGE + 4096;
    static constexpr int FIT = (232448 - FIXED) / (WARPS * SLOT);
    static constexpr int SLOTS = FIT > 6 ? 6 : FIT;                              // ring of a warp: K, V, K, V ...
    static constexpr int SMEM = FIXED + WARPS * SLOTS * SLOT;
    static constexpr int PART = HEADS * (DP + 2);                                // floats of a partial result: sums, then maxima, then totals
    static constexpr bool Q_IN_REGISTERS = HB == 1 && DP <= 128;
    static_assert(SLOTS >= 2, "a ring needs two slots");
};

// What a warp loads next.  It runs ahead of what the warp computes, across the borders of units.
template <typename S>
struct Loader {
    uint64_t left;                         // tiles of the CTA's part, this one included
    uint32_t sequence, unit, tile, tile_end, begin, end;
    uint32_t page_index, at;               // of the lane's token
    uint32_t page;                         // table entry, asked for one tile ahead
    uint64_t row;                          // element of the lane's row in the tile at hand
    uint64_t scale_row;
    uint32_t mask;                         // its tokens that count
};

template <int DP, bool I8, int HB>
__global__ void __launch_bounds__(32 * WARPS, 1) paged_attention_kernel(const __grid_constant__ AttentionParams p)
{
    using S = Shape<DP, I8, HB>;
    extern __shared__ __align__(16) char smem[];
    char *const q_smem = smem;
    float *const merge = reinterpret_cast<float *>(smem + S::Q_BYTES);
    char *const small = smem + S::Q_BYTES + S::MERGE;
    uint64_t *const sums = reinterpret_cast<uint64_t *>(small);                 // 32
    Found *const found = reinterpret_cast<Found *>(small + 256);
    float *const factor = reinterpret_cast<float *>(small + 512);               // [16]
    float *const warp_m = factor + 16, *const warp_l = warp_m + WARPS * 16;     // [WARPS][16]
    uint32_t *const masks = reinterpret_cast<uint32_t *>(warp_l + WARPS * 16);  // [WARPS][SLOTS]
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, c4 = lane % 4;
    char *const ring = smem + S::FIXED + warp * S::SLOTS * S::SLOT;
    const uint32_t dim = p.cache.dim, pieces = dim * S::SIZE / 16, units = p.cache.kv_heads * p.head_blocks;
    constexpr uint32_t TILE = WARPS * S::STEP;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (dim < DP) {   // what no copy fills counts as zeros
        for (uint32_t i = lane; i < S::SLOTS * S::SLOT / 16; i += 32) {
            reinterpret_cast<uint4 *>(ring)[i] = make_uint4(0, 0, 0, 0);
        }
    }
    const uint64_t total = locate<32 * WARPS>(p, units, TILE, blockIdx.x == 0, sums, found,
        [&](uint64_t n) { return part_begin(blockIdx.x, n, gridDim.x); });
    if (total == 0) {
        return;
    }
    uint64_t place = part_begin(blockIdx.x, total, gridDim.x);
    const uint64_t stop = part_begin(blockIdx.x + 1, total, gridDim.x);
    if (place == stop) {
        return;
    }
    uint32_t sequence = found->sequence, begin, end;
    live_tokens(p, sequence, &begin, &end);
    uint32_t tiles = max(tiles_of(begin, end, TILE), 1u);
    uint32_t unit = min((uint32_t)((place - found->first) / tiles), units - 1), tile = (uint32_t)((place - found->first) % tiles);

    // ---- the copies ----
    const uint32_t page_size = p.cache.page_size;
    const bool one_page = page_size % S::STEP == 0;    // a step's tokens are neighbours in one page
    const uint32_t lane_token = lane % S::STEP, step_pages = TILE / page_size, step_at = TILE % page_size;
    Loader<S> ld;
    auto token0 = [&]() { return (ld.begin / TILE + ld.tile) * TILE + warp * S::STEP; };
    auto look_up = [&]() {
        const uint32_t t = token0() + (one_page ? 0 : lane_token);
        ld.page = t < ld.end && ld.page_index < p.table_pages ? (uint32_t)__ldg(p.table + (uint64_t)ld.sequence * p.table_pages + ld.page_index) : 0xFFFFFFFFu;
    };
    auto enter = [&]() {
        const uint32_t t = token0() + (one_page ? 0 : lane_token);
        ld.page_index = t / page_size;
        ld.at = t - ld.page_index * page_size;
        look_up();
    };
    ld.left = stop - place;
    ld.sequence = sequence;
    ld.unit = unit;
    ld.tile = tile;
    ld.tile_end = tiles;
    ld.begin = begin;
    ld.end = end;
    ld.mask = 0;
    ld.row = ld.scale_row = 0;
    enter();
    uint32_t fill_slot = 0;    // items: K, V, K, V ...
    const uint32_t copy_row = lane / (S::ROW / 16), copy_piece = lane % (S::ROW / 16);   // of the first piece that the lane copies
    const uint64_t token_bytes = p.cache.token_stride * S::SIZE, lane_bytes = copy_row * token_bytes + copy_piece * 16;
    const uint32_t ring_at = smem_at(ring), lane_at = ring_at + copy_row * S::PITCH + copy_piece * 16;
    auto issue = [&](bool values) {
        const uint32_t slot = fill_slot;
        fill_slot = fill_slot + 1 == S::SLOTS ? 0 : fill_slot + 1;
        if (!values) {
            ld.mask = 0;
            if (ld.left != 0) {
                const uint32_t head = ld.unit / p.head_blocks, t = token0() + lane_token;
                const bool inside = t >= ld.begin && t < ld.end, good = ld.page < p.cache.pages;
                if (inside && !good) {
                    atomicExch(p.status, BAD_ATTENTION);
                }
                ld.mask = __ballot_sync(0xFFFFFFFFu, inside && good);
                if (S::STEP == 16) {
                    ld.mask &= 0xFFFFu;
                }
                ld.row = good ? row_element(p.cache, ld.page, ld.at, head) : 0;
                ld.scale_row = I8 && good ? scale_element(p.cache, ld.page, ld.at, head) + (one_page ? lane_token : 0) : 0;
                // on to the next tile
                --ld.left;
                if (++ld.tile < ld.tile_end) {
                    ld.page_index += step_pages;
                    ld.at += step_at;
                    if (ld.at >= page_size) {
                        ld.at -= page_size;
                        ++ld.page_index;
                    }
                    look_up();
                } else if (ld.left != 0) {
                    ld.tile = 0;
                    if (++ld.unit == units) {
                        ld.unit = 0;
                        ld.sequence = next_sequence(p, ld.sequence);
                        live_tokens(p, ld.sequence, &ld.begin, &ld.end);
                        ld.tile_end = tiles_of(ld.begin, ld.end, TILE);
                    }
                    enter();
                }
            }
            if (lane == 0) {
                masks[warp * S::SLOTS + slot] = ld.mask;
            }
        }
        if (ld.mask != 0) {
            constexpr int ROWS = 32 / (S::ROW / 16);      // rows of one instruction
            const char *base = reinterpret_cast<const char *>(values ? p.v : p.k);
            uint32_t dst = lane_at + slot * S::SLOT;
            if (one_page && dim == DP && ld.mask == S::ALL) {
                const char *src = base + ld.row * S::SIZE + lane_bytes;
#pragma unroll
                for (int i = 0; i < S::STEP / ROWS; ++i) {
                    copy16(dst + i * ROWS * S::PITCH, src);
                    src += ROWS * token_bytes;
                }
            } else {
#pragma unroll 1
                for (int i = 0; i < S::STEP / ROWS; ++i) {
                    const uint32_t r = copy_row + i * ROWS;
                    const uint64_t row = one_page ? ld.row + r * p.cache.token_stride : __shfl_sync(0xFFFFFFFFu, ld.row, r);
                    if (copy_piece < pieces) {
                        const bool on = ld.mask >> r & 1;
                        copy16(dst + i * ROWS * S::PITCH, on ? base + row * S::SIZE + copy_piece * 16 : base, on ? 16 : 0);
                    }
                }
            }
            if (I8 && lane < S::STEP) {
                const float *s = values ? p.v_scale : p.k_scale;
                const bool on = ld.mask >> lane & 1;
                copy4(ring_at + slot * S::SLOT + S::STEP * S::PITCH + lane * 4, on ? s + ld.scale_row : s, on ? 4 : 0);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    __syncwarp();
#pragma unroll 1
    for (int i = 0; i < S::SLOTS - 1; ++i) {
        issue(i & 1);
    }
    uint32_t take_slot = 0;
    // the next item is there; the slot of the one before it is filled again
    auto next = [&](bool values) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S::SLOTS - 2) : "memory");
        __syncwarp();
        issue(values != (S::SLOTS % 2 == 0));    // item n + SLOTS - 1
        const uint32_t slot = take_slot;
        take_slot = take_slot + 1 == S::SLOTS ? 0 : take_slot + 1;
        return slot;
    };

    // ---- unit by unit ----
    constexpr int NT = S::STEP / 8, KS = DP / 16, TILES_D = DP / 8;
    while (place < stop) {
        const uint32_t head = unit / p.head_blocks, block = unit % p.head_blocks;
        const uint32_t heads_here = min((uint32_t)S::HEADS, p.group - block * S::HEADS), head0 = head * p.group + block * S::HEADS;
        const uint32_t count = (uint32_t)min((uint64_t)(tiles - tile), stop - place);
        // Queries: brought to 2^13 .. 2^14 by a power of two (which the factor of the scores takes back), then two binary16
        // numbers each, in rows (hi of every head, lo of every head) of the matrix instruction's left operand.  Bytes come
        // out of their words in the order 0, 2, 1, 3; the queries' elements stand in the same order.
        for (uint32_t h = warp; h < S::HEADS; h += WARPS) {
            float x[DP / 32];
            int top = 0;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                const uint32_t d = lane + 32 * i;
                x[i] = 0.f;
                if (h < heads_here && d < dim) {
                    const uint64_t e = sequence * p.q_stride + (uint64_t)(head0 + h) * dim + d;
                    x[i] = p.q_f16 ? load1(reinterpret_cast<const __half *>(p.q) + e) : load1(reinterpret_cast<const float *>(p.q) + e);
                }
                top = max(top, magnitude(x[i]));
            }
            top = __reduce_max_sync(0xFFFFFFFFu, top);
            const int e = max(top >> 23, 20);
            const float up = __int_as_float((127 + 13 + 127 - e) << 23);
            if (lane == 0) {
                factor[h] = __int_as_float((e - 13) << 23) * (p.scale * LOG2E);
            }
            const uint32_t hi_row = h, lo_row = S::HEADS + h;
#pragma unroll
            for (int i = 0; i < DP / 32; ++i) {
                const uint32_t d = lane + 32 * i, r = d % 4;
                const uint32_t k = I8 ? d / 16 * 16 + d % 16 / 4 * 2 + r / 2 + r % 2 * 8 : d;
                const float v = x[i] * up;
                const __half hi = __float2half_rn(v);
                *reinterpret_cast<__half *>(q_smem + hi_row * S::Q_PITCH + k * 2) = hi;
                *reinterpret_cast<__half *>(q_smem + lo_row * S::Q_PITCH + k * 2) = __float2half_rn(v - __half2float(hi));
            }
        }
        __syncthreads();
        uint32_t qa[S::Q_IN_REGISTERS ? KS : 1][4];
        const uint32_t q_at = smem_at(q_smem + (lane % 16) * S::Q_PITCH + lane / 16 * 16);
        if constexpr (S::Q_IN_REGISTERS) {
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                matrices(qa[s], q_at + s * 32);
            }
        }
        float fac[HB], m[HB], l[HB], acc[TILES_D][2 * HB], top_unit = 0.f;
#pragma unroll
        for (int b = 0; b < HB; ++b) {
            fac[b] = factor[g + 8 * b];
            m[b] = -INFINITY;
            l[b] = 0.f;
        }
#pragma unroll
        for (int n = 0; n < TILES_D; ++n) {
#pragma unroll
            for (int e = 0; e < 2 * HB; ++e) {
                acc[n][e] = 0.f;
            }
        }
#pragma unroll 1
        for (uint32_t i = 0; i < count; ++i) {
            // scores: [heads] x [tokens]
            const uint32_t ks = next(false);
            const char *const kt = ring + ks * S::SLOT;
            const uint32_t mask = masks[warp * S::SLOTS + ks];
            float sc[NT][4];
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
            }
            if (mask != 0) {
                uint32_t q_lo[4];
                auto multiply = [&](int s, int j, uint32_t b0, uint32_t b1) {
                    if constexpr (HB == 1) {
                        if constexpr (S::Q_IN_REGISTERS) {
                            mma(sc[j], qa[s], b0, b1);
                        } else {
                            mma(sc[j], qa[0], b0, b1);
                        }
                    } else {
                        mma(sc[j], qa[0], b0, b1);
                        mma(sc[j], q_lo, b0, b1);
                    }
                };
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    if constexpr (!S::Q_IN_REGISTERS) {
                        matrices(qa[0], q_at + s * 32);
                    }
                    if constexpr (HB == 2) {
                        matrices(q_lo, q_at + 16 * S::Q_PITCH + s * 32);
                    }
                    uint32_t r[4];
                    if constexpr (!I8) {
#pragma unroll
                        for (int j = 0; j < NT; j += 2) {
                            matrices(r, smem_at(kt + (8 * j + lane % 8 + lane / 16 * 8) * S::PITCH + s * 32 + lane / 8 % 2 * 16));
                            multiply(s, j, r[0], r[1]);
                            multiply(s, j + 1, r[2], r[3]);
                        }
                    } else if constexpr (S::STEP == 32) {
                        matrices(r, smem_at(kt + lane * S::PITCH + s * 16));
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            multiply(s, j, bytes_to_half2<0>(r[j]), bytes_to_half2<8>(r[j]));
                        }
                    } else {
                        matrices(r, smem_at(kt + lane % 16 * S::PITCH + s * 16));
                        multiply(s, 0, bytes_to_half2<0>(r[0]), bytes_to_half2<8>(r[0]));
                        multiply(s, 1, bytes_to_half2<0>(r[1]), bytes_to_half2<8>(r[1]));
                    }
                }
            }
            // weights: exp(s - m) times 2^14, which the division by their sum takes back
            float keep[HB], w[HB][NT][2];
            auto weights = [&](auto all) {
#pragma unroll
              for (int b = 0; b < HB; ++b) {
                float top = m[b];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float unit_k[2] = {1.f, 1.f};
                    if constexpr (I8) {
                        const float2 u = *reinterpret_cast<const float2 *>(kt + S::STEP * S::PITCH + (8 * j + 2 * c4) * 4);
                        unit_k[0] = reciprocal(u.x);
                        unit_k[1] = reciprocal(u.y);
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float s = HB == 1 ? sc[j][e] + sc[j][e + 2] : sc[j][e + 2 * b];
                        const bool on = all.value || (mask >> (8 * j + 2 * c4 + e) & 1);
                        w[b][j][e] = on ? s * (fac[b] * unit_k[e]) : -INFINITY;
                        top = fmaxf(top, w[b][j][e]);
                    }
                }
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                const float base = top == -INFINITY ? 0.f : top;
                keep[b] = exp2_fast(m[b] - base);
                m[b] = top;
                l[b] *= keep[b];
#pragma unroll
                for (int j = 0; j < NT; ++j) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        w[b][j][e] = exp2_fast(w[b][j][e] - (base - 14.f));
                        l[b] += w[b][j][e];
                    }
                }
              }
            };
            if (mask == S::ALL) {
                weights(std::true_type());
            } else {
                weights(std::false_type());
            }
            const uint32_t vs = next(true);
            if (mask == 0) {
                continue;
            }
            const char *const vt = ring + vs * S::SLOT;
            if constexpr (I8) {
                // Rows of bytes have units of their own.  They go into the weights, relative to the largest unit so far:
                // weights stay within binary16.
                float unit_v[NT][2], top = top_unit;
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    const float2 u = *reinterpret_cast<const float2 *>(vt + S::STEP * S::PITCH + (8 * j + 2 * c4) * 4);
                    unit_v[j][0] = mask >> (8 * j + 2 * c4) & 1 ? reciprocal(u.x) : 0.f;
                    unit_v[j][1] = mask >> (8 * j + 2 * c4 + 1) & 1 ? reciprocal(u.y) : 0.f;
                    top = fmaxf(top, fmaxf(unit_v[j][0], unit_v[j][1]));
                }
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                const float inv = top > 0.f ? reciprocal(top) : 0.f, change = top_unit * inv;
                top_unit = top;
#pragma unroll
                for (int b = 0; b < HB; ++b) {
                    keep[b] *= change;
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        w[b][j][0] *= unit_v[j][0] * inv;
                        w[b][j][1] *= unit_v[j][1] * inv;
                    }
                }
            }
            uint32_t pa[HB][NT / 2][4];    // HB 1: rows hi, lo; HB 2: [0] hi, [1] lo
#pragma unroll
            for (int t = 0; t < NT / 2; ++t) {
                if constexpr (HB == 1) {
                    split_pair(w[0][2 * t][0], w[0][2 * t][1], pa[0][t][0], pa[0][t][1]);
                    split_pair(w[0][2 * t + 1][0], w[0][2 * t + 1][1], pa[0][t][2], pa[0][t][3]);
                } else {
                    split_pair(w[0][2 * t][0], w[0][2 * t][1], pa[0][t][0], pa[HB - 1][t][0]);
                    split_pair(w[HB - 1][2 * t][0], w[HB - 1][2 * t][1], pa[0][t][1], pa[HB - 1][t][1]);
                    split_pair(w[0][2 * t + 1][0], w[0][2 * t + 1][1], pa[0][t][2], pa[HB - 1][t][2]);
                    split_pair(w[HB - 1][2 * t + 1][0], w[HB - 1][2 * t + 1][1], pa[0][t][3], pa[HB - 1][t][3]);
                }
            }
            // sums: the step's share is added to the running sum in binary32 (round to nearest: the matrix instruction's own
            // accumulation truncates, which adds up over thousands of steps)
            auto add = [&](int n, const float (&c)[4]) {
                if constexpr (HB == 1) {
                    acc[n][0] = fmaf(acc[n][0], keep[0], c[0] + c[2]);
                    acc[n][1] = fmaf(acc[n][1], keep[0], c[1] + c[3]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        acc[n][e % (2 * HB)] = fmaf(acc[n][e % (2 * HB)], keep[e / 2 % HB], c[e]);
                    }
                }
            };
            auto weigh = [&](float (&c)[4], int t, uint32_t b0, uint32_t b1) {
                mma(c, pa[0][t], b0, b1);
                if constexpr (HB == 2) {
                    mma(c, pa[HB - 1][t], b0, b1);
                }
            };
            if constexpr (!I8) {
#pragma unroll
                for (int n = 0; n < TILES_D; n += 2) {
                    float c0[4] = {0.f, 0.f, 0.f, 0.f}, c1[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int t = 0; t < NT / 2; ++t) {
                        uint32_t r[4];
                        matrices_t(r, smem_at(vt + (16 * t + lane % 16) * S::PITCH + n * 16 + lane / 16 * 16));
                        weigh(c0, t, r[0], r[1]);
                        weigh(c1, t, r[2], r[3]);
                    }
                    add(n, c0);
                    add(n + 1, c1);
                }
            } else {
#pragma unroll
                for (int n = 0; n < TILES_D; n += 4) {     // 32 bytes of a row: even and odd elements of two pieces
                    float c[4][4] = {};
#pragma unroll
                    for (int t = 0; t < NT / 2; ++t) {
                        uint32_t r[4];
                        matrices_t(r, smem_at(vt + (16 * t + lane % 16) * S::PITCH + n * 8 + lane / 16 * 16));
                        weigh(c[0], t, bytes_to_half2<0>(r[0]), bytes_to_half2<0>(r[1]));
                        weigh(c[1], t, bytes_to_half2<8>(r[0]), bytes_to_half2<8>(r[1]));
                        weigh(c[2], t, bytes_to_half2<0>(r[2]), bytes_to_half2<0>(r[3]));
                        weigh(c[3], t, bytes_to_half2<8>(r[2]), bytes_to_half2<8>(r[3]));
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        add(n + k, c[k]);
                    }
                }
            }
        }
        // ---- the warps' shares, and out ----
#pragma unroll
        for (int b = 0; b < HB; ++b) {
            l[b] += __shfl_xor_sync(0xFFFFFFFFu, l[b], 1);
            l[b] += __shfl_xor_sync(0xFFFFFFFFu, l[b], 2);
            if (c4 == 0) {
                warp_m[warp * 16 + g + 8 * b] = m[b];
                warp_l[warp * 16 + g + 8 * b] = l[b];
            }
        }
        __syncthreads();
        const bool whole = count == tiles;
        float *const part = p.parts + ((uint64_t)blockIdx.x * 2 + (tile != 0 ? 0 : 1)) * S::PART;
        float own[HB];
#pragma unroll
        for (int b = 0; b < HB; ++b) {
            float top = -INFINITY;
            for (int w = 0; w < WARPS; ++w) {
                top = fmaxf(top, warp_m[w * 16 + g + 8 * b]);
            }
            own[b] = exp2_fast(m[b] - (top == -INFINITY ? 0.f : top)) * (I8 ? top_unit : 1.f);
        }
        for (int col = 0; col < DP; col += S::COLS) {
#pragma unroll
            for (int n = 0; n < TILES_D; ++n) {
#pragma unroll
                for (int e = 0; e < 2 * HB; ++e) {
                    // element of the row: pairs of neighbours, or (bytes) every second one
                    const uint32_t d = I8 ? n / 2 * 16 + 4 * c4 + e % 2 * 2 + n % 2 : 8 * n + 2 * c4 + e % 2;
                    const bool here = I8 ? n / 2 * 16 >= col && n / 2 * 16 < col + S::COLS : 8 * n >= col && 8 * n < col + S::COLS;
                    if (here) {
                        merge[(warp * S::HEADS + g + e / 2 * 8) * (S::COLS + 4) + d - col] = acc[n][e] * own[e / 2];
                    }
                }
            }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < S::HEADS * S::COLS; i += 32 * WARPS) {
                const uint32_t h = i / S::COLS, d = i % S::COLS;
                float top = -INFINITY, sum = 0.f, all = 0.f;
                for (int w = 0; w < WARPS; ++w) {
                    top = fmaxf(top, warp_m[w * 16 + h]);
                }
                const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) {
                    sum += merge[(w * S::HEADS + h) * (S::COLS + 4) + d];
                    all += warp_l[w * 16 + h] * exp2_fast(warp_m[w * 16 + h] - base);
                }
                if (whole) {
                    if (h < heads_here && col + d < dim) {
                        store_out(p, sequence * p.out_stride + (uint64_t)(head0 + h) * dim + col + d, all == 0.f ? 0.f : __fdiv_rn(sum, all));
                    }
                    if (p.lse != nullptr && h < heads_here && col + d == 0) {
                        p.lse[(uint64_t)sequence * p.heads + head0 + h] = (top + log2f(all) - 14.f) * LN2;
                    }
                } else {
                    part[h * DP + col + d] = sum;
                    if (col + d == 0) {
                        part[S::HEADS * DP + h] = top;
                        part[S::HEADS * (DP + 1) + h] = all;
                    }
                }
            }
            __syncthreads();
        }
        // ---- the next unit ----
        place += count;
        tile = 0;
        if (place < stop && ++unit == units) {
            unit = 0;
            sequence = next_sequence(p, sequence);
            live_tokens(p, sequence, &begin, &end);
            tiles = max(tiles_of(begin, end, TILE), 1u);
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// Units that several CTAs have worked on: one block for the border at which such a unit is cut first, and each head.
template <int DP, int HB>
__global__ void __launch_bounds__(128) paged_attention_join_kernel(const __grid_constant__ AttentionParams p, uint32_t tile_tokens, uint32_t parts)
{
    constexpr int HEADS = 8 * HB, PART = HEADS * (DP + 2);
    __shared__ uint64_t sums[32];
    __shared__ Found found[1];
    __shared__ float weight[MAX_PARTS], share[MAX_PARTS], warp_top[4];
    const uint32_t i = blockIdx.x, units = p.cache.kv_heads * p.head_blocks, h = blockIdx.y;
    // sequences without a token, which no part holds: every parts-th is this block column's
    for (uint32_t s0 = 0; s0 < p.sequences; s0 += 32 * parts) {
        const uint64_t mine = s0 + (uint64_t)(threadIdx.x % 32) * parts + i;
        uint32_t begin, end = 1;
        if (mine < p.sequences) {
            live_tokens(p, (uint32_t)mine, &begin, &end);
        }
        for (uint32_t none = __ballot_sync(0xFFFFFFFFu, end == 0); none != 0; none &= none - 1) {
            const uint32_t s = s0 + (__ffs(none) - 1) * parts + i;
            for (uint32_t hq = h; hq < p.heads; hq += gridDim.y) {
                for (uint32_t d = threadIdx.x; d < p.cache.dim; d += 128) {
                    store_out(p, s * p.out_stride + (uint64_t)hq * p.cache.dim + d, 0.f);
                }
                if (p.lse != nullptr && threadIdx.x == 0) {
                    p.lse[(uint64_t)s * p.heads + hq] = -INFINITY;
                }
            }
        }
    }
    const uint64_t total = locate<128>(p, units, tile_tokens, false, sums, found, [&](uint64_t n) {
        const uint64_t stop = part_begin(i + 1, n, parts);
        return stop != 0 ? stop - 1 : 0;
    });
    if (total == 0) {
        return;
    }
    const uint64_t from = part_begin(i, total, parts), stop = part_begin(i + 1, total, parts);
    if (from == stop || stop == total) {
        return;
    }
    // the unit that holds the part's last tile
    const uint32_t sequence = found->sequence;
    const uint64_t first = found->first;
    uint32_t begin, end;
    live_tokens(p, sequence, &begin, &end);
    const uint32_t tiles = max(tiles_of(begin, end, tile_tokens), 1u);
    const uint32_t unit = min((uint32_t)((stop - 1 - first) / tiles), units - 1);
    const uint64_t a = first + (uint64_t)unit * tiles;
    const uint32_t head = unit / p.head_blocks, block = unit % p.head_blocks;
    if (a < from || a + tiles <= stop || block * HEADS + h >= p.group) {
        return;    // cut before, or not here
    }
    const uint32_t n = part_of(a + tiles - 1, total, parts) - i + 1;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // part c of the unit is a share of CTA i + c: what it began (slot 1) in the first, what it went on with in the others
    auto part = [&](uint32_t c) { return p.parts + ((uint64_t)(i + c) * 2 + (c == 0 ? 1 : 0)) * PART; };
    float top = -INFINITY;
    for (uint32_t c = threadIdx.x; c < n; c += 128) {
        // (with fewer tiles than CTAs, some have none)
        const bool empty = total < parts && part_begin(i + c, total, parts) == part_begin(i + c + 1, total, parts);
        weight[c] = empty ? -INFINITY : part(c)[HEADS * DP + h];
        share[c] = empty ? 0.f : part(c)[HEADS * (DP + 1) + h];
        top = fmaxf(top, weight[c]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
    }
    if (threadIdx.x % 32 == 0) {
        warp_top[threadIdx.x / 32] = top;
    }
    __syncthreads();
    top = fmaxf(fmaxf(warp_top[0], warp_top[1]), fmaxf(warp_top[2], warp_top[3]));
    for (uint32_t c = threadIdx.x; c < n; c += 128) {
        weight[c] = exp2_fast(weight[c] - (top == -INFINITY ? 0.f : top));
    }
    __syncthreads();
    float all = 0.f, sum[(DP + 127) / 128] = {};
#pragma unroll 8
    for (uint32_t c = 0; c < n; ++c) {
        const float *q = part(c) + h * DP;
        const float w = weight[c];
        all = fmaf(share[c], w, all);
#pragma unroll
        for (int k = 0; k < (DP + 127) / 128; ++k) {
            const uint32_t d = threadIdx.x + 128 * k;
            const float x = d < DP && w != 0.f ? q[d] : 0.f;
            sum[k] = fmaf(x, w, sum[k]);
        }
    }
    const uint32_t hq = head * p.group + block * HEADS + h;
#pragma unroll
    for (int k = 0; k < (DP + 127) / 128; ++k) {
        const uint32_t d = threadIdx.x + 128 * k;
        if (d < p.cache.dim) {
            store_out(p, sequence * p.out_stride + (uint64_t)hq * p.cache.dim + d, all == 0.f ? 0.f : __fdiv_rn(sum[k], all));
        }
    }
    if (p.lse != nullptr && threadIdx.x == 0) {
        p.lse[(uint64_t)sequence * p.heads + hq] = (top + log2f(all) - 14.f) * LN2;
    }
}

uint32_t parts_of(const DeviceCtx *c)
{
    return c->sm_count < MAX_PARTS ? (uint32_t)c->sm_count : MAX_PARTS;
}
template <int DP, bool I8, int HB>
EE launch(DeviceCtx *c, AttentionParams &p, cudaStream_t st)
{
    using S = Shape<DP, I8, HB>;
    const void *kernel = reinterpret_cast<const void *>(paged_attention_kernel<DP, I8, HB>);
    B200_EE(raise_smem_limit(c, (KernelFamily)(KF_ATTENTION + (DP == 64 ? 0 : (DP == 128 ? 1 : 2)) + 3 * I8 + 6 * (HB - 1)), &kernel, 1, S::SMEM));
    const uint32_t parts = parts_of(c);
    B200_EE(launch_kernel(parts, 32 * WARPS, S::SMEM, st, paged_attention_kernel<DP, I8, HB>, p));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(parts, S::HEADS < (int)p.group ? S::HEADS : p.group);
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    B200_CUDA(launch_programmatic(cfg, paged_attention_join_kernel<DP, HB>, p, (uint32_t)(WARPS * S::STEP), parts));
    count_launch();
    return SUCCESS;
}
template <bool I8>
EE launch(DeviceCtx *c, AttentionParams &p, cudaStream_t st)
{
    const uint32_t dim = p.cache.dim;
    if (p.group <= 8) {
        return dim <= 64 ? launch<64, I8, 1>(c, p, st) : (dim <= 128 ? launch<128, I8, 1>(c, p, st) : launch<256, I8, 1>(c, p, st));
    }
    return dim <= 64 ? launch<64, I8, 2>(c, p, st) : (dim <= 128 ? launch<128, I8, 2>(c, p, st) : launch<256, I8, 2>(c, p, st));
}

// the checks of both entry points; *p is filled in
EE check(const bolt_b200_kv_cache *cache, const bolt_b200_paged_attention_call *a, AttentionParams *p, DeviceCtx **c)
{
    if (cache == nullptr || a == nullptr) {
        return NULL_POINTER;
    }
    *c = ctx();
    if (*c == nullptr) {
        return UNKNOWN;
    }
    B200_EE(check_cache(cache));
    if (a->heads == 0 || a->heads % cache->kv_heads != 0 || a->table_pages == 0) {
        return NOT_MATCH;
    }
    if ((a->q_dt != DT_F32 && a->q_dt != DT_F16) || (a->out_dt != DT_F32 && a->out_dt != DT_F16 && a->out_dt != DT_U8_Q) || a->heads > 65535u ||
        a->sequences > 65535u) {
        return NOT_SUPPORTED;
    }
    const uint64_t row = (uint64_t)a->heads * cache->dim;
    if (a->sequences > 1 && (a->q_stride < row || a->out_stride < row)) {
        return NOT_MATCH;
    }
    if (a->q_stride > MAX_STRIDE || a->out_stride > MAX_STRIDE) {
        return NOT_SUPPORTED;
    }
    p->cache = view_of(*cache);
    p->k = cache->k;
    p->v = cache->v;
    p->k_scale = cache->k_scale;
    p->v_scale = cache->v_scale;
    p->q = a->q;
    p->out = a->out;
    p->lse = a->lse;
    p->q_stride = a->q_stride;
    p->out_stride = a->out_stride;
    p->table = a->table;
    p->length = a->length;
    p->sequences = a->sequences;
    p->heads = a->heads;
    p->group = a->heads / cache->kv_heads;
    p->head_blocks = p->group <= 8 ? 1 : (p->group + 15) / 16;
    p->table_pages = a->table_pages;
    p->window = a->window;
    p->scale = a->scale;
    p->out_scale = a->out_scale;
    p->i8 = cache->dt == DT_I8;
    p->q_f16 = a->q_dt == DT_F16;
    p->out_kind = a->out_dt == DT_F32 ? 0 : (a->out_dt == DT_F16 ? 1 : 2);
    p->status = (*c)->d_status;
    return SUCCESS;
}
U32 workspace_bytes(const AttentionParams &p, const DeviceCtx *c)
{
    const U32 dp = p.cache.dim <= 64 ? 64 : (p.cache.dim <= 128 ? 128 : 256);
    return parts_of(c) * 2 * (p.group <= 8 ? 8 : 16) * (dp + 2) * 4;
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" {

EE bolt_b200_paged_attention_tmp_bytes(const bolt_b200_kv_cache *cache, const bolt_b200_paged_attention_call *call, U32 *bytes)
{
    if (bytes == nullptr) {
        return NULL_POINTER;
    }
    AttentionParams p;
    DeviceCtx *c = nullptr;
    B200_EE(check(cache, call, &p, &c));
    *bytes = workspace_bytes(p, c);
    return SUCCESS;
}

EE bolt_b200_paged_attention(const bolt_b200_kv_cache *cache, const bolt_b200_paged_attention_call *call, U32 tmpBytes, void *tmp)
{
    AttentionParams p;
    DeviceCtx *c = nullptr;
    B200_EE(check(cache, call, &p, &c));
    if (p.sequences == 0) {
        return SUCCESS;
    }
    if (p.q == nullptr || p.out == nullptr || p.table == nullptr || p.length == nullptr) {
        return NULL_POINTER;
    }
    const U32 need = workspace_bytes(p, c);
    if (tmpBytes < need) {
        return NOT_MATCH;
    }
    if (need != 0 && tmp == nullptr) {
        return NULL_POINTER;
    }
    const size_t out_size = p.out_kind == 0 ? 4 : (p.out_kind == 1 ? 2 : 1);
    if (!aligned(p.q, p.q_f16 ? 2 : 4) || !aligned(p.out, out_size) || !aligned(p.lse, 4) || !aligned(p.table, 4) || !aligned(p.length, 4) ||
        (need != 0 && !aligned(tmp, 16))) {
        return NOT_SUPPORTED;
    }
    if (!on_this_device(p.q) || !on_this_device(p.out) || !on_this_device(p.table) || !on_this_device(p.length) ||
        (p.lse != nullptr && !on_this_device(p.lse)) || (need != 0 && !on_this_device(tmp))) {
        return NOT_MATCH;
    }
    p.parts = reinterpret_cast<float *>(tmp);
    return p.i8 ? launch<true>(c, p, tls().stream) : launch<false>(c, p, tls().stream);
}

}  // extern "C"
