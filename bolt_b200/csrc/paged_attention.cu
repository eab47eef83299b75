// paged_attention.cu -- attention of one new token per sequence over a paged cache.
//
// out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m), s_t = scale q . k_t, in one pass over the tokens with a running maximum
// m: when it rises, what has been summed so far is scaled down.  Shares of a sequence are joined the same way.
//
// HBM bound: keys and values are read once for up to sixteen query heads of a key head (and once more for every sixteen beyond), and
// everything else is small beside them.
// Every team of warps takes an equal part of all tokens of the batch (whose lengths the host does not know), cut where it
// may be; a second kernel joins the units that were cut.  Inside a team every warp streams tokens of its own through a private
// ring of asynchronous copies and keeps its own maximum, total and sums, so that warps meet only at the end of a unit.
// The products run on mma.m16n8k16: eight query heads that share a key head are half a tile's rows, and the other half
// holds what binary16 has cut off of them, so that one instruction per operand tile multiplies 22-bit queries (and
// probabilities) with the cache's binary16; bytes become binary16 in registers, five instructions for four of them, unless
// mma.m16n8k32 takes them as they are (keys).
//
// Whole calls, 64 sequences of up to 8192 tokens, 8 key heads of 128: binary16 5.9 TB/s; bytes 4.6 TB/s in short bursts, bound by
// 924 instructions for a step of 32 tokens, and call after call, by the power that they take, 3.9 to 4.3 TB/s.  One sequence of
// 131072 tokens: 94 to 101 us, 5.3 to 5.7 TB/s.  One of 4000: 11.7 us, of which 8 are the chain length -> page -> keys -> values
// -> shares with the code that has to be fetched on the way, 4 the join.  Rows of 256 elements and groups of more than eight query
// heads keep 64 running sums a lane and run with eight warps: 2.6 TB/s in bytes with 16 heads, 4.7 in binary16.
#include <type_traits>

#include "decode.cuh"

namespace b200 {
namespace {

// a unit that a part has begun and others have gone on with
struct Cut {
    uint32_t parts;            // how many, 0: none
    uint32_t sequence, head0, heads;   // query heads
};
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
    uint32_t team, part_count, share_bytes;    // warps that share a unit; parts of the row; bytes of partial results
    uint32_t step_pages, step_at, run_tiles;   // tokens of a tile in pages and what is left; tiles of a run
    uint32_t page_magic;                       // 2^32 / page_size
    uint32_t even_bytes, to_1152;              // 0x00FF00FF, 0x64806480
    float *parts;                              // workspace: two partial results for every part,
    Cut *cuts;                                 // and what is to be joined
    int *status;
};

// position / page_size and the remainder: the multiplication is one too low at most
__device__ __forceinline__ void split_position(const AttentionParams &p, uint32_t position, uint32_t &page, uint32_t &at)
{
    page = __umulhi(position, p.page_magic);
    at = position - page * p.cache.page_size;
    if (at >= p.cache.page_size) {
        at -= p.cache.page_size;
        ++page;
    }
}
__device__ __forceinline__ bool live_tokens(const AttentionParams &p, uint32_t sequence, uint32_t *begin, uint32_t *end)
{
    return b200::live_tokens(p.length[sequence], p.table_pages, p.cache.page_size, p.window, begin, end);
}

// as quantize_cuda_b200, F32 -> U8_Q
__device__ __forceinline__ uint32_t to_u8(float x, float scale)
{
    return (uint32_t)min(255, max(1, cvt_rne_x86(__fadd_rn(__fmul_rn(x, scale), 128.0f))));
}
__device__ __forceinline__ void store_out(const AttentionParams &p, uint64_t at, float x)
{
    if (p.out_kind == 0) {
        reinterpret_cast<float *>(p.out)[at] = x;
    } else if (p.out_kind == 1) {
        reinterpret_cast<__half *>(p.out)[at] = __float2half_rn(x);
    } else {
        reinterpret_cast<uint8_t *>(p.out)[at] = (uint8_t)to_u8(x, p.out_scale);
    }
}

// ---- how the work is divided -----------------------------------------------------------------------------------
// A unit is one sequence, key head and block of query heads; it has tiles of team x STEP tokens on a grid that starts at
// token 0.  All units' tiles stand in one row, in which every team of warps takes an equal, contiguous part.
constexpr int MAX_WARPS = 16;
constexpr uint32_t MAX_SEQUENCES = 65535;
// Up to so many sequences every warp counts for itself, beyond, the CTA's warps share the counting and wait for one another
// (64 sequences of some 150 tokens, 12 heads of 64: 23.3 us and, shared, 24.0; 512: 112.3 and 110.7).
constexpr uint32_t BY_WARP = 256;
struct Found {
    uint32_t sequence, first;
};
struct Counting {     // shared memory
    uint32_t sums[MAX_WARPS];
    Found found[MAX_WARPS];
};
__device__ __forceinline__ uint32_t count_tiles(const AttentionParams &p, uint32_t s, uint32_t tile_shift)
{
    uint32_t begin, end;
    live_tokens(p, s, &begin, &end);
    return tiles_of(begin, end, tile_shift);
}
// By all warps of a CTA, for each its team's part: the row's length, and the sequence that holds the part's first tile with
// that sequence's own first place.
template <int WARPS>
__device__ __forceinline__ Parts locate(const AttentionParams &p, uint32_t units, uint32_t tile_shift, uint32_t team, Counting *c, Found *mine)
{
    const uint32_t lane = threadIdx.x % 32, warp = threadIdx.x / 32, teams = WARPS / team;
    const bool shared = p.sequences > BY_WARP;
    const uint32_t segment = shared ? (p.sequences + WARPS - 1) / WARPS : p.sequences;
    const uint32_t a = shared ? min(warp * segment, p.sequences) : 0, b = min(a + segment, p.sequences), per = (b - a + 31) / 32;
    const uint32_t s0 = min(a + lane * per, b), s1 = min(s0 + per, b);
    uint32_t own = 0;
#pragma unroll 1
    for (uint32_t s = s0; s < s1; ++s) {
        own += count_tiles(p, s, tile_shift);
    }
    own *= units;
    uint32_t upto = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        upto += lane >= o ? v : 0;
    }
    uint32_t total = __shfl_sync(0xFFFFFFFFu, upto, 31);
    if (shared) {
        if (lane == 0) {
            c->sums[warp] = total;
        }
        __syncthreads();
        total = 0;
        for (uint32_t w = 0; w < WARPS; ++w) {
            upto += w < warp ? c->sums[w] : 0;
            total += c->sums[w];
        }
    }
    const Parts parts(total, p.part_count);
    *mine = Found{0, 0};     // (always something inside the arrays, even if lengths change under the call)
#pragma unroll 1
    for (uint32_t t = shared ? 0 : warp / team; t < (shared ? teams : warp / team + 1); ++t) {
        const uint32_t part = blockIdx.x * teams + t;
        const uint32_t place = parts.begin(part);
        const uint32_t holder = __ballot_sync(0xFFFFFFFFu, part < parts.n && place >= upto - own && place < upto);
        if (holder == 0) {
            continue;
        }
        Found f = {s0, upto - own};
        if (holder >> lane & 1) {
#pragma unroll 1
            while (f.sequence < s1) {
                const uint32_t next = f.first + count_tiles(p, f.sequence, tile_shift) * units;
                if (place < next) {
                    break;
                }
                f.first = next;
                ++f.sequence;
            }
        }
        f.first = __shfl_sync(0xFFFFFFFFu, f.first, __ffs(holder) - 1);
        f.sequence = min(__shfl_sync(0xFFFFFFFFu, f.sequence, __ffs(holder) - 1), p.sequences - 1);
        if (shared) {
            c->found[t] = f;
        } else {
            *mine = f;
        }
    }
    if (shared) {
        __syncthreads();
        if (blockIdx.x * teams + warp / team < parts.n) {
            *mine = c->found[warp / team];
        }
    }
    return parts;
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
__device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)   // c = a b
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f), "f"(0.f), "f"(0.f), "f"(0.f));
}
__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float2 shared_pair(uint32_t at)
{
    float2 v;
    asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ float shared_number(uint32_t at)
{
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t shared_bits(uint32_t at)     // whether any of 16 bytes is set
{
    uint32_t a, b, c, d;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(at) : "memory");
    return a | b | c | d;
}
// two binary32 operations in one instruction: (x, y) = (x, y) * k + (a, b), and the sum of two pairs
__device__ __forceinline__ void fma_pair(float &x, float &y, float k, float a, float b)
{
    asm("{\n\t.reg .b64 u, v, w;\n\tmov.b64 u, {%0, %1};\n\tmov.b64 v, {%2, %2};\n\tmov.b64 w, {%3, %4};\n\tfma.rn.f32x2 u, u, v, w;\n\tmov.b64 {%0, %1}, u;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(k), "f"(a), "f"(b));
}
__device__ __forceinline__ void fma_pair(float &x, float &y, float k, float a, float b, float c, float d)   // (a, b) + (c, d)
{
    asm("{\n\t.reg .b64 u, v, w, z;\n\tmov.b64 u, {%0, %1};\n\tmov.b64 v, {%2, %2};\n\tmov.b64 w, {%3, %4};\n\tmov.b64 z, {%5, %6};\n\t"
        "add.rn.f32x2 w, w, z;\n\tfma.rn.f32x2 u, u, v, w;\n\tmov.b64 {%0, %1}, u;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(k), "f"(a), "f"(b), "f"(c), "f"(d));
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
// (The two constants come from the parameters: as immediates they take an instruction and a half more, since a three-way
// logic instruction has room for one.)
template <int SHIFT>
__device__ __forceinline__ uint32_t bytes_to_half2(const AttentionParams &p, uint32_t x)
{
    const uint32_t y = ((x >> SHIFT) & p.even_bytes) ^ p.to_1152, k = 0x64806480u;
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

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// Weights of rows of bytes are sums of two binary16 numbers in units of a power of two that puts the largest, ref or a little below,
// at 2^14 .. 2^15.  (From 2^-126 on, so that it and its reciprocal are normal numbers.)
__device__ __forceinline__ uint32_t weight_unit_bits(float ref)
{
    return max(__float_as_uint(ref) & 0x7F800000u, 15u << 23) - (14u << 23);
}

// DP: elements of a row, rounded up; HB: blocks of eight query heads
template <int DP, bool I8, int HB>
struct Shape {
    static constexpr int SIZE = I8 ? 1 : 2, ROW = DP * SIZE, PITCH = ROW + 16;   // an odd number of 16-byte pieces: ldmatrix meets every bank once
    static constexpr int STEP = ROW <= 128 ? 32 : 16;                            // tokens that a warp takes at a time
    static constexpr uint32_t ALL = STEP == 32 ? 0xFFFFFFFFu : 0xFFFFu;
    static constexpr int SLOT = STEP * PITCH + (I8 ? STEP * 4 : 0);
    static constexpr int HEADS = 8 * HB;
    static constexpr int NUMBERS = DP / 8 * 2 * HB;                              // running sums of a lane
    // Steps are chains of dependent instructions: sixteen warps (128 registers a lane) hide them where the running sums fit (64
    // sequences of up to 8192 tokens in bytes: 135 us, with eight warps and six slots 164; in binary16 202 and 227).
    static constexpr int WARPS = NUMBERS <= 32 && HB == 1 ? 16 : 8;
    // With one block of heads queries meet bytes as whole numbers, four digits of base 256 each, and keys need no conversion (64
    // sequences of up to 8192 tokens: 135 us, as binary16 137; rows of 256 elements 155 and 162; two blocks would have 64
    // running numbers more, which took 261 us in place of 242).
    static constexpr bool DIGITS = I8 && HB == 1;
    static constexpr float LIFT = I8 ? 0.f : 14.f;     // binary16: weights are exp(s - m) 2^14
    static constexpr int Q_PITCH = DP * (DIGITS ? 1 : 2) + 16, Q_ROWS = HEADS * (DIGITS ? 4 : 2), Q_BYTES = Q_ROWS * Q_PITCH;   // queries of a team
    static constexpr int TEAMS = 4 * Q_BYTES <= 20480 ? 4 : (2 * Q_BYTES <= 20480 ? 2 : 1);
    // Numbers of a lane that the warps exchange at a time, in the slot that each is through with: as many as there are, or as fit.
    static constexpr int GO = NUMBERS * 128 <= SLOT ? NUMBERS : (SLOT >= 4096 ? 32 : 16);
    static constexpr int SMALL = 1024 + WARPS * 320;
    static constexpr int FIXED = TEAMS * Q_BYTES + SMALL;
    static constexpr int FIT = (232448 - FIXED) / (WARPS * SLOT);
    // Ring of a warp: K, V, K, V ...  Two slots, three for two blocks of heads (eight warps with twice the products):
    // what shared memory does not take is L1, and more requests at a time do not help (64 sequences of up to 8192 tokens in
    // binary16: 202 us with two, 212 with three; 16 heads to a key head: 274, 253, and 257 with six).
    static constexpr int SLOTS = HB == 1 ? 2 : (FIT < 3 ? FIT : 3);
    static constexpr int SMEM = FIXED + WARPS * SLOTS * SLOT;
    static constexpr int PART = HEADS * (DP + 2);                                // floats of a partial result: sums, then maxima, then totals
    static_assert(SLOTS >= 2, "a ring needs two slots");
    static_assert(GO * 128 <= SLOT && NUMBERS % GO == 0, "the numbers have room in a slot");
};

// What a warp loads next: a run of tiles of one unit whose pages are at most 32 neighbours of the table, one in each lane.
struct Run {
    uint32_t head, begin, end;
    uint32_t left;                         // tiles
    uint32_t token;                        // first one of the warp's step
    uint32_t first_page;                   // of the table's row
};
// The run behind it, and where the one after that begins: in shared memory, for registers are short.  All lanes write the
// same; a barrier stands between what they read and the first write, and behind the last one, since nothing else keeps them
// together.
struct Ahead {
    Run run;
    uint32_t sequence, unit, tile, tiles, begin, end, left;
    uint32_t pages[32];
};

template <int DP, bool I8, int HB>
__global__ void __launch_bounds__(32 * Shape<DP, I8, HB>::WARPS, 1) paged_attention_kernel(const __grid_constant__ AttentionParams p)
{
    using S = Shape<DP, I8, HB>;
    constexpr int WARPS = S::WARPS;
    extern __shared__ __align__(16) char smem[];
    char *const small = smem + S::TEAMS * S::Q_BYTES;
    Counting *const counting = reinterpret_cast<Counting *>(small);             // 192 bytes
    float *const factors = reinterpret_cast<float *>(small + 512);              // [TEAMS][16]
    float *const warp_m = reinterpret_cast<float *>(small + 1024), *const warp_l = warp_m + WARPS * 16;     // [WARPS][16]
    uint32_t lane, warp = threadIdx.x / 32;
    asm volatile("mov.u32 %0, %%laneid;" : "=r"(lane));     // (kept in a register, not asked for again and again)
    asm volatile("mov.u32 %0, %0;" : "+r"(warp));
    const uint32_t g = lane / 4, c4 = lane % 4;
    static_assert(sizeof(Ahead) <= 192, "");
    Ahead &ahead = *reinterpret_cast<Ahead *>(small + 1024 + WARPS * 128 + warp * 192);
    char *const ring = smem + S::FIXED + warp * S::SLOTS * S::SLOT;
    const uint32_t dim = p.cache.dim, pieces = dim * S::SIZE / 16, units = p.cache.kv_heads * p.head_blocks;
    const uint32_t team = p.team, member = warp % team, teams = WARPS / team;
    const uint32_t tile_tokens = team * S::STEP, tile_shift = __ffs(tile_tokens) - 1;
    const uint32_t part = blockIdx.x * teams + warp / team;
    char *const q_smem = smem + warp / team * S::Q_BYTES;
    float *const factor = factors + warp / team * 16;

    if (dim < DP) {   // what no copy fills counts as zeros
        for (uint32_t i = lane; i < S::SLOTS * S::SLOT / 16; i += 32) {
            reinterpret_cast<uint4 *>(ring)[i] = make_uint4(0, 0, 0, 0);
        }
    }
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");    // nothing in front of this touches global memory
    Found found;
    const Parts parts = locate<WARPS>(p, units, tile_shift, team, counting, &found);
    uint32_t place = part < parts.n ? parts.begin(part) : 0;
    const uint32_t stop = part < parts.n ? parts.begin(part + 1) : 0;
    if (lane == 0 && member == 0) {
        p.cuts[part].parts = 0;
    }
    auto team_sync = [&]() {
        __syncwarp();       // (the barrier takes a warp as a whole, and comes behind branches that some lanes have taken)
        if (team == WARPS) {
            __syncthreads();
        } else {
            asm volatile("bar.sync %0, %1;" ::"r"(1 + warp / team), "r"(32 * team) : "memory");
        }
    };

    if (place < stop) {
        uint32_t sequence = found.sequence, begin, end;
        live_tokens(p, sequence, &begin, &end);
        uint32_t tiles = max(tiles_of(begin, end, tile_shift), 1u);
        const uint32_t units_before = (place - found.first) / tiles;
        uint32_t unit = min(units_before, units - 1), tile = place - found.first - units_before * tiles;

        // ---- the copies ----
        const uint32_t page_size = p.cache.page_size;
        const bool one_page = page_size % S::STEP == 0;    // a step's tokens are neighbours in one page
        const uint32_t lane_token = lane % S::STEP;
        Run run;
        uint32_t pages = 0;
        ahead.left = stop - place;
        ahead.sequence = sequence;
        ahead.unit = unit;
        ahead.tile = tile;
        ahead.tiles = tiles;
        ahead.begin = begin;
        ahead.end = end;
        __syncwarp();
        auto look_ahead = [&]() {
            Run next;
            uint32_t t = ahead.tile, tiles = ahead.tiles, left = ahead.left, unit_ahead = ahead.unit, sequence_ahead = ahead.sequence;
            next.begin = ahead.begin;
            next.end = ahead.end;
            __syncwarp();       // everybody has read the record, and (enter) the run in it
            next.left = min(min(p.run_tiles, tiles - t), left);
            if (next.left == 0) {
                ahead.run.left = 0;
                __syncwarp();
                return;
            }
            next.head = HB == 1 ? unit_ahead : unit_ahead / p.head_blocks;
            next.token = (((next.begin >> tile_shift) + t) << tile_shift) + member * S::STEP;
            uint32_t within;
            split_position(p, next.token, next.first_page, within);
            ahead.run = next;
            const uint64_t entry = (uint64_t)next.first_page + lane;
            const uint32_t page = entry < p.table_pages && entry * page_size < next.end ?
                (uint32_t)p.table[(uint64_t)sequence_ahead * p.table_pages + entry] : 0xFFFFFFFFu;
            left -= next.left;
            t += next.left;
            if (t == tiles && left != 0) {
                t = 0;
                if (++unit_ahead == units) {
                    unit_ahead = 0;
                    const uint32_t s = next_sequence(p, sequence_ahead);
                    uint32_t b, e;
                    live_tokens(p, s, &b, &e);
                    ahead.sequence = s;
                    ahead.begin = b;
                    ahead.end = e;
                    ahead.tiles = max(tiles_of(b, e, tile_shift), 1u);
                }
                ahead.unit = unit_ahead;
            }
            ahead.tile = t;
            ahead.left = left;
            __syncwarp();
            ahead.pages[lane] = page;       // (every lane's own: behind the barrier, which need not wait for the table)
        };
        uint32_t page_index = 0, at = 0;    // of the lane's token
        auto enter = [&]() {
            run = ahead.run;
            pages = ahead.pages[lane];
            split_position(p, run.token + (one_page ? 0 : lane_token), page_index, at);
            look_ahead();
        };
        look_ahead();
        enter();
        uint64_t row = 0, scale_row = 0;    // elements of the lane's row in the tile at hand
        uint32_t live = 0;                  // its tokens that count
        const uint32_t copy_row = lane / (S::ROW / 16), copy_piece = lane % (S::ROW / 16);   // of the first piece that the lane copies
        const uint64_t token_bytes = p.cache.token_stride * S::SIZE;
        const uint32_t ring_at = smem_at(ring), lane_at = copy_row * S::PITCH + copy_piece * 16;
        uint32_t coming[S::SLOTS / 2];      // `live` of the steps that have been asked for and not been used
        auto issue = [&](auto kind, uint32_t slot) {    // asks for K (and V) of the next step
            constexpr bool values = decltype(kind)::value;
            if constexpr (!values) {
                // (a run that has come to its end has no tokens inside)
                const uint32_t page = __shfl_sync(0xFFFFFFFFu, pages, page_index - run.first_page), t = run.token + lane_token;
                const bool inside = t >= run.begin && t < run.end, good = page < p.cache.pages;
                live = __ballot_sync(0xFFFFFFFFu, inside && good) & S::ALL;
                if (live != S::ALL && inside && !good) {
                    atomicExch(p.status, BAD_ATTENTION);
                }
                row = good ? row_element(p.cache, page, at, run.head) : 0;
                if (I8) {
                    scale_row = good ? scale_element(p.cache, page, at, run.head) + (one_page ? lane_token : 0) : 0;
                }
#pragma unroll
                for (int k = 0; k + 1 < S::SLOTS / 2; ++k) {
                    coming[k] = coming[k + 1];
                }
                coming[S::SLOTS / 2 - 1] = live;
                run.token += tile_tokens;
                page_index += p.step_pages;
                at += p.step_at;
                if (at >= page_size) {
                    at -= page_size;
                    ++page_index;
                }
                --run.left;
            }
            constexpr int ROWS = 32 / (S::ROW / 16);      // rows of one instruction
            const char *base = reinterpret_cast<const char *>(values ? p.v : p.k);
            const uint32_t dst = slot + lane_at;
            // (pages smaller than a step: every row's place comes from the lane that has looked it up)
            if (live == S::ALL) {
                if (one_page) {
                    const char *src = base + row * S::SIZE + copy_row * token_bytes + copy_piece * 16;
                    if (copy_piece < pieces) {
#pragma unroll
                        for (int i = 0; i < S::STEP / ROWS; ++i) {
                            copy16(dst + i * ROWS * S::PITCH, src);
                            src += ROWS * token_bytes;
                        }
                    }
                } else {
                    const uint64_t from = row * S::SIZE;
#pragma unroll
                    for (int i = 0; i < S::STEP / ROWS; ++i) {
                        const char *src = base + __shfl_sync(0xFFFFFFFFu, from, copy_row + i * ROWS) + copy_piece * 16;
                        if (copy_piece < pieces) {
                            copy16(dst + i * ROWS * S::PITCH, src);
                        }
                    }
                }
            } else if (live != 0) {
#pragma unroll 4
                for (int i = 0; i < S::STEP / ROWS; ++i) {
                    const uint32_t r = copy_row + i * ROWS;
                    const uint64_t from = one_page ? row + r * p.cache.token_stride : __shfl_sync(0xFFFFFFFFu, row, r);
                    if (copy_piece < pieces) {
                        const bool on = live >> r & 1;
                        copy16(dst + i * ROWS * S::PITCH, on ? base + from * S::SIZE + copy_piece * 16 : base, on ? 16 : 0);
                    }
                }
            }
            if constexpr (I8) {
                const bool on = live >> (lane % S::STEP) & 1;
                if (S::STEP == 32 || lane < S::STEP) {
                    const float *scales = values ? p.v_scale : p.k_scale;
                    copy4(slot + S::STEP * S::PITCH + lane * 4, on ? scales + scale_row : scales, on ? 4 : 0);
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            __syncwarp();       // (lanes that have copied nothing and those that have go on together)
            if (!values && run.left == 0) {
                if (ahead.run.left != 0) {
                    enter();
                } else {
                    run.end = 0;
                    run.left = 0xFFFFFFFFu;
                }
            }
        };
        __syncwarp();

        // ---- item by item (K, V, K, V ...) ----
        // In turn n the warp uses item n and asks for item n + SLOTS - 1, into the slot of item n - 1.  The first turns only
        // ask, so that the code, which a short call has to fetch before it can run, is there once.
        constexpr int NT = S::STEP / 8, KS = DP / 16, TILES_D = DP / 8;
        constexpr uint32_t RING = S::SLOTS * S::SLOT / 4;   // floats
        constexpr bool EVEN = S::SLOTS % 2 == 0;        // then a K turn asks for V, and a V turn for K
        uint32_t item = ring_at + S::SLOT, count = 0, done = 0;    // tiles of the unit, and how many of them are through
        uint32_t head0 = 0, heads_here = 0, mask = 0;
        float fac[HB], m[HB], l[HB], keep[HB], w[HB][NT][2], acc[TILES_D][2 * HB], ref[HB];
        const uint32_t q_at = smem_at(q_smem + (lane % 16) * S::Q_PITCH + lane / 16 * 16);
        int n = 1 - S::SLOTS;
        auto turn = [&](auto asks_for_values) {
            if (n >= 0) {
                // the item is there, and everybody is through with the one before it
                asm volatile("cp.async.wait_group %0;" ::"n"(S::SLOTS - 2) : "memory");
                __syncwarp();
            }
            issue(asks_for_values, item == ring_at ? ring_at + (S::SLOTS - 1) * S::SLOT : item - S::SLOT);
            return n >= 0;
        };
        auto turned = [&]() {
            ++n;
            item = item == ring_at + (S::SLOTS - 1) * S::SLOT ? ring_at : item + S::SLOT;
        };
#pragma unroll 1
        for (;;) {
            if (!EVEN || n != 1 - S::SLOTS) {
                mask = coming[0];
                if (n >= 0 && done == count) {
                    // ---- a unit begins ----
                    const uint32_t head = HB == 1 ? unit : unit / p.head_blocks, block = unit - head * (HB == 1 ? 1 : p.head_blocks);
                    heads_here = min((uint32_t)S::HEADS, p.group - block * S::HEADS);
                    head0 = head * p.group + block * S::HEADS;
                    count = min(tiles - tile, stop - place);
                    done = 0;
                    // Queries: brought to 2^13 .. 2^14 by a power of two (which the factor of the scores takes back), then two binary16
                    // numbers each, in the rows (hi of every head, lo of every head) of the matrix instruction's left operand.  Bytes come
                    // out of their words in the order 0, 2, 1, 3; the queries' elements stand in the same order.  As digits: brought to
                    // 2^29 .. 2^30 and rounded, then -128 .. 127 each, the highest first.
                    const uint64_t q_row = sequence * p.q_stride + (uint64_t)head0 * dim;
#pragma unroll 1
                    for (uint32_t h = member; h < S::HEADS; h += team) {
                        // (rows of heads that do not exist repeat the first: nobody reads their results)
                        const uint64_t from = q_row + (h < heads_here ? h : 0) * dim;
                        float x[DP / 32];
                        int top = 0;
#pragma unroll
                        for (int i = 0; i < DP / 32; ++i) {
                            const uint32_t d = lane + 32 * i;
                            x[i] = 0.f;
                            if (d < dim) {
                                x[i] = p.q_f16 ? load1(reinterpret_cast<const __half *>(p.q) + from + d) : load1(reinterpret_cast<const float *>(p.q) + from + d);
                            }
                            top = max(top, magnitude(x[i]));
                        }
                        constexpr int BITS = S::DIGITS ? 29 : 13, LEAST = S::DIGITS ? 30 : 20;    // (the factor stays a normal number)
                        const int highest = __reduce_max_sync(0xFFFFFFFFu, top) >> 23, e = max(highest, LEAST);
                        const float up = __int_as_float((127 + BITS + 127 - e) << 23);
                        if (lane == 0) {
                            // (whole numbers know no infinity: what is none goes on in the factor)
                            factor[h] = S::DIGITS && highest == 255 ? NAN : __int_as_float((e - BITS) << 23) * (p.scale * LOG2E);
                        }
#pragma unroll
                        for (int i = 0; i < DP / 32; ++i) {
                            const uint32_t d = lane + 32 * i;
                            const float v = x[i] * up;
                            if constexpr (S::DIGITS) {
                                int rest = __float2int_rn(v);
#pragma unroll
                                for (int digit = 3; digit >= 0; --digit) {
                                    q_smem[(digit * S::HEADS + h) * S::Q_PITCH + d] = (char)rest;
                                    rest = (rest - (signed char)rest) >> 8;
                                }
                            } else {
                                const uint32_t r = d % 4, k = I8 ? d / 16 * 16 + d % 16 / 4 * 2 + r / 2 + r % 2 * 8 : d;
                                const __half hi = __float2half_rn(v);
                                *reinterpret_cast<__half *>(q_smem + h * S::Q_PITCH + k * 2) = hi;
                                *reinterpret_cast<__half *>(q_smem + (S::HEADS + h) * S::Q_PITCH + k * 2) = __float2half_rn(v - __half2float(hi));
                            }
                        }
                    }
                    team_sync();
#pragma unroll
                    for (int b = 0; b < HB; ++b) {
                        fac[b] = factor[g + 8 * b];
                    }
#pragma unroll
                    for (int b = 0; b < HB; ++b) {
                        m[b] = -INFINITY;
                        l[b] = ref[b] = 0.f;
                    }
#pragma unroll
                    for (int n = 0; n < TILES_D; ++n) {
#pragma unroll
                        for (int e = 0; e < 2 * HB; ++e) {
                            acc[n][e] = 0.f;
                        }
                    }
                }
                if (turn(std::bool_constant<EVEN>())) {
                    // scores: [heads] x [tokens]
                    float score[HB][NT][2];
                    if constexpr (S::DIGITS) {
                        // The digits' products are whole numbers, two neighbouring digits' together below 2^31.  A tile has the rows of two
                        // digits of eight heads.
#pragma unroll
                        for (int j = 0; j < NT; j += 2) {
                            int c[2][2][4] = {};
#pragma unroll
                            for (int s = 0; s < DP / 32; ++s) {
                                uint32_t r[4], qa[4];
                                matrices(r, item + (lane % 8 + lane / 16 * 8) * S::PITCH + lane / 8 % 2 * 16 + 8 * j * S::PITCH + s * 32);
#pragma unroll
                                for (int k = 0; k < 2; ++k) {
                                    matrices(qa, q_at + 16 * k * S::Q_PITCH + s * 32);
                                    mma_s8(c[k][0], qa, r[0], r[1]);
                                    mma_s8(c[k][1], qa, r[2], r[3]);
                                }
                            }
#pragma unroll
                            for (int t = 0; t < 2; ++t) {
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    const int high = c[0][t][e] * 256 + c[0][t][e + 2], low = c[1][t][e] * 256 + c[1][t][e + 2];
                                    score[0][j + t][e] = fmaf((float)high, 65536.f, (float)low);
                                }
                            }
                        }
                    } else {
                        float sc[NT][4];
                        uint32_t qa[4], q_lo[4];
                        auto multiply = [&](int s, int j, uint32_t b0, uint32_t b1) {
                            if (s == 0) {
                                mma_first(sc[j], qa, b0, b1);
                            } else {
                                mma(sc[j], qa, b0, b1);
                            }
                            if constexpr (HB == 2) {
                                mma(sc[j], q_lo, b0, b1);
                            }
                        };
#pragma unroll
                        for (int s = 0; s < KS; ++s) {
                            matrices(qa, q_at + s * 32);
                            if constexpr (HB == 2) {
                                matrices(q_lo, q_at + 16 * S::Q_PITCH + s * 32);
                            }
                            uint32_t r[4];
                            if constexpr (!I8) {
#pragma unroll
                                for (int j = 0; j < NT; j += 2) {
                                    matrices(r, item + (lane % 8 + lane / 16 * 8) * S::PITCH + lane / 8 % 2 * 16 + 8 * j * S::PITCH + s * 32);
                                    multiply(s, j, r[0], r[1]);
                                    multiply(s, j + 1, r[2], r[3]);
                                }
                            } else if constexpr (S::STEP == 32) {
                                matrices(r, item + lane * S::PITCH + s * 16);
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    multiply(s, j, bytes_to_half2<0>(p, r[j]), bytes_to_half2<8>(p, r[j]));
                                }
                            } else {
                                matrices(r, item + lane % 16 * S::PITCH + s * 16);
                                multiply(s, 0, bytes_to_half2<0>(p, r[0]), bytes_to_half2<8>(p, r[0]));
                                multiply(s, 1, bytes_to_half2<0>(p, r[1]), bytes_to_half2<8>(p, r[1]));
                            }
                        }
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
#pragma unroll
                            for (int b = 0; b < HB; ++b) {
#pragma unroll
                                for (int e = 0; e < 2; ++e) {
                                    score[b][j][e] = HB == 1 ? sc[j][e] + sc[j][e + 2] : sc[j][e + 2 * b];
                                }
                            }
                        }
                    }
                    // weights: exp(s - m), in binary16 times 2^14, which the division by their sum takes back
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        float unit_k[2] = {1.f, 1.f};
                        if constexpr (I8) {
                            const float2 u = shared_pair(item + S::STEP * S::PITCH + (8 * j + 2 * c4) * 4);
                            unit_k[0] = reciprocal(u.x);
                            unit_k[1] = reciprocal(u.y);
                        }
#pragma unroll
                        for (int b = 0; b < HB; ++b) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                w[b][j][e] = score[b][j][e] * (fac[b] * unit_k[e]);
                            }
                        }
                    }
                    if (mask != S::ALL) {
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const bool on = mask >> (8 * j + 2 * c4 + e) & 1;
#pragma unroll
                                for (int b = 0; b < HB; ++b) {
                                    w[b][j][e] = on ? w[b][j][e] : -INFINITY;
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int b = 0; b < HB; ++b) {
                        float top = m[b];
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            top = fmaxf(top, fmaxf(w[b][j][0], w[b][j][1]));
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
                                w[b][j][e] = exp2_fast(w[b][j][e] - (base - S::LIFT));
                                l[b] += w[b][j][e];
                            }
                        }
                    }
                }
                turned();
            }
            if (turn(std::bool_constant<!EVEN>())) {
                if (mask != 0) {
                    if constexpr (I8) {
                        // Rows of bytes have units of their own, which go into the weights, and these are taken relative to the largest of
                        // a head so far (`ref`, as the sums relative to the running maximum of the scores): a row with a large unit that
                        // weighs little leaves the others their bits.  Rows of zeros, whose scale is 1 whatever the others' are, have no share.
                        const float own_scale = shared_number(item + S::STEP * S::PITCH + lane_token * 4);
                        uint32_t counts = mask;
#pragma unroll 1
                        for (uint32_t ones = __ballot_sync(0xFFFFFFFFu, own_scale == 1.f) & mask; ones != 0; ones &= ones - 1) {
                            const uint32_t r = __ffs(ones) - 1;
                            uint32_t bytes = 0;
                            if (lane < pieces) {
                                bytes = shared_bits(item + r * S::PITCH + lane * 16);
                            }
                            if (!__any_sync(0xFFFFFFFFu, bytes != 0)) {
                                counts &= ~(1u << r);
                            }
                        }
                        float unit_v[NT][2];
#pragma unroll
                        for (int j = 0; j < NT; ++j) {
                            const float2 u = shared_pair(item + S::STEP * S::PITCH + (8 * j + 2 * c4) * 4);
                            unit_v[j][0] = reciprocal(u.x);
                            unit_v[j][1] = reciprocal(u.y);
                        }
                        if (counts != S::ALL) {
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                unit_v[j][0] = counts >> (8 * j + 2 * c4) & 1 ? unit_v[j][0] : 0.f;
                                unit_v[j][1] = counts >> (8 * j + 2 * c4 + 1) & 1 ? unit_v[j][1] : 0.f;
                            }
                        }
#pragma unroll
                        for (int b = 0; b < HB; ++b) {
                            float top = 0.f;
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                w[b][j][0] *= unit_v[j][0];
                                w[b][j][1] *= unit_v[j][1];
                                top = fmaxf(top, fmaxf(w[b][j][0], w[b][j][1]));
                            }
                            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                            top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                            const float before = __uint_as_float(weight_unit_bits(ref[b]));
                            ref[b] = fmaxf(ref[b] * keep[b], top);
                            const float inv = __uint_as_float((254u << 23) - weight_unit_bits(ref[b]));
                            keep[b] = keep[b] * before * inv;
#pragma unroll
                            for (int j = 0; j < NT; ++j) {
                                w[b][j][0] *= inv;
                                w[b][j][1] *= inv;
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
                            fma_pair(acc[n][0], acc[n][1], keep[0], c[0], c[1], c[2], c[3]);
                        } else {
                            fma_pair(acc[n][0], acc[n][1], keep[0], c[0], c[1]);
                            fma_pair(acc[n][2 * HB - 2], acc[n][2 * HB - 1], keep[HB - 1], c[2], c[3]);
                        }
                    };
                    auto weigh = [&](float (&c)[4], int t, uint32_t b0, uint32_t b1) {
                        if (t == 0) {
                            mma_first(c, pa[0][t], b0, b1);
                        } else {
                            mma(c, pa[0][t], b0, b1);
                        }
                        if constexpr (HB == 2) {
                            mma(c, pa[HB - 1][t], b0, b1);
                        }
                    };
                    if constexpr (!I8) {
#pragma unroll
                        for (int n = 0; n < TILES_D; n += 2) {
                            float c0[4], c1[4];
#pragma unroll
                            for (int t = 0; t < NT / 2; ++t) {
                                uint32_t r[4];
                                matrices_t(r, item + lane % 16 * S::PITCH + lane / 16 * 16 + 16 * t * S::PITCH + n * 16);
                                weigh(c0, t, r[0], r[1]);
                                weigh(c1, t, r[2], r[3]);
                            }
                            add(n, c0);
                            add(n + 1, c1);
                        }
                    } else {
#pragma unroll
                        for (int n = 0; n < TILES_D; n += 4) {     // 32 bytes of a row: even and odd elements of two pieces
                            float c[4][4];
#pragma unroll
                            for (int t = 0; t < NT / 2; ++t) {
                                uint32_t r[4];
                                matrices_t(r, item + lane % 16 * S::PITCH + lane / 16 * 16 + 16 * t * S::PITCH + n * 8);
                                weigh(c[0], t, bytes_to_half2<0>(p, r[0]), bytes_to_half2<0>(p, r[1]));
                                weigh(c[1], t, bytes_to_half2<8>(p, r[0]), bytes_to_half2<8>(p, r[1]));
                                weigh(c[2], t, bytes_to_half2<0>(p, r[2]), bytes_to_half2<0>(p, r[3]));
                                weigh(c[3], t, bytes_to_half2<8>(p, r[2]), bytes_to_half2<8>(p, r[3]));
                            }
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                add(n + k, c[k]);
                            }
                        }
                    }
                }
                if (++done == count) {
                    // ---- the warps' shares, and out ----
                    const bool whole = count == tiles;
                    float *const share = p.parts + ((uint64_t)part * 2 + (tile != 0 ? 0 : 1)) * S::PART;
                    float own[HB];
                    const uint32_t warp0 = warp - member;
#pragma unroll
                    for (int b = 0; b < HB; ++b) {
                        l[b] += __shfl_xor_sync(0xFFFFFFFFu, l[b], 1);
                        l[b] += __shfl_xor_sync(0xFFFFFFFFu, l[b], 2);
                        if (c4 == 0) {
                            warp_m[warp * 16 + g + 8 * b] = m[b];
                            warp_l[warp * 16 + g + 8 * b] = l[b];
                        }
                    }
                    team_sync();
#pragma unroll
                    for (int b = 0; b < HB; ++b) {
                        // the four lanes of a head look at every fourth warp each
                        const uint32_t h = g + 8 * b;
                        float wm[WARPS / 4], top = -INFINITY, all = 0.f;
#pragma unroll
                        for (int k = 0; k < WARPS / 4; ++k) {
                            const uint32_t w = 4 * k + c4;
                            wm[k] = w < team ? warp_m[(warp0 + w) * 16 + h] : -INFINITY;
                            top = fmaxf(top, wm[k]);
                        }
                        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
                        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
                        for (int k = 0; k < WARPS / 4; ++k) {
                            const uint32_t w = 4 * k + c4;
                            all += w < team ? warp_l[(warp0 + w) * 16 + h] * exp2_fast(wm[k] - base) : 0.f;
                        }
                        all += __shfl_xor_sync(0xFFFFFFFFu, all, 1);
                        all += __shfl_xor_sync(0xFFFFFFFFu, all, 2);
                        own[b] = exp2_fast(m[b] - base) * (I8 ? __uint_as_float(weight_unit_bits(ref[b])) : 1.f);
                        if (whole) {
                            own[b] *= all == 0.f ? 0.f : __frcp_rn(all);
                        }
                        if (member == 0 && c4 == 0) {
                            if (!whole) {
                                share[S::HEADS * DP + h] = top;
                                share[S::HEADS * (DP + 1) + h] = all;
                            } else if (p.lse != nullptr && h < heads_here) {
                                p.lse[(uint64_t)sequence * p.heads + head0 + h] = (top + log2f(all) - S::LIFT) * LN2;
                            }
                        }
                    }
                    if (!whole && tile == 0 && member == 0 && lane == 0) {
                        p.cuts[part] = Cut{min(parts.of(place + tiles - 1), parts.n - 1) - part + 1, sequence, head0, heads_here};
                    }
                    // GO numbers of every lane of every warp at a time, in the values' slot (no copy goes there before the next turn); then
                    // each warp adds up some of them over its team, whose slots are at the same place of their rings.
                    float *const merge = reinterpret_cast<float *>(ring + (item - ring_at)) + lane, *const merge0 = merge - member * RING;
                    constexpr int NUMBERS = S::NUMBERS, GO = S::GO;
#pragma unroll
                    for (int x0 = 0; x0 < NUMBERS; x0 += GO) {
                        if (x0 != 0) {
                            team_sync();
                        }
#pragma unroll
                        for (int x = 0; x < GO; ++x) {
                            merge[x * 32] = acc[(x0 + x) / (2 * HB)][(x0 + x) % (2 * HB)] * own[(x0 + x) % (2 * HB) / 2];
                        }
                        team_sync();
#pragma unroll 1
                        for (uint32_t x = member; x < GO; x += team) {
                            float sum = 0.f;
#pragma unroll 4
                            for (uint32_t w = 0; w < team; ++w) {
                                sum += merge0[w * RING + x * 32];
                            }
                            const uint32_t t = (x0 + x) / (2 * HB), e = (x0 + x) % (2 * HB), h = g + e / 2 * 8;
                            const uint32_t d = I8 ? t / 2 * 16 + 4 * c4 + e % 2 * 2 + t % 2 : 8 * t + 2 * c4 + e % 2;
                            if (!whole) {
                                share[h * DP + d] = sum;
                            } else if (h < heads_here && d < dim) {
                                store_out(p, sequence * p.out_stride + (uint64_t)(head0 + h) * dim + d, sum);
                            }
                        }
                    }
                    team_sync();
                    if (dim < DP) {
                        for (uint32_t i = lane; i < S::SLOT / 16; i += 32) {
                            reinterpret_cast<uint4 *>(ring + (item - ring_at))[i] = make_uint4(0, 0, 0, 0);
                        }
                    }
                    // ---- the next unit ----
                    place += count;
                    tile = 0;
                    if (place >= stop) {
                        break;
                    }
                    if (++unit == units) {
                        unit = 0;
                        sequence = next_sequence(p, sequence);
                        live_tokens(p, sequence, &begin, &end);
                        tiles = max(tiles_of(begin, end, tile_shift), 1u);
                    }
                }
            }
            turned();
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    // sequences without a token, a warp each, and lengths that are none
    for (uint32_t s = blockIdx.x * WARPS + warp; s < p.sequences; s += gridDim.x * WARPS) {
        uint32_t begin, end;
        if (!live_tokens(p, s, &begin, &end) && lane == 0) {
            atomicExch(p.status, BAD_ATTENTION);
        }
        if (end == 0) {
            for (uint32_t i = lane; i < p.heads * dim; i += 32) {
                store_out(p, s * p.out_stride + i, 0.f);
            }
            for (uint32_t i = lane; p.lse != nullptr && i < p.heads; i += 32) {
                p.lse[(uint64_t)s * p.heads + i] = -INFINITY;
            }
        }
    }
}

// loads that are issued where they stand, all before the first result is needed
__device__ __forceinline__ float load_now(const float *p)
{
    float x;
    asm volatile("ld.global.cg.f32 %0, [%1];" : "=f"(x) : "l"(p) : "memory");
    return x;
}
__device__ __forceinline__ void load_now(const float *p, float &x, float &y)
{
    asm volatile("ld.global.cg.v2.f32 {%0, %1}, [%2];" : "=f"(x), "=f"(y) : "l"(p) : "memory");
}
// Units that several parts have worked on: a block for the part that has begun one, and for each eight query heads.  Shares
// are read eight at a time, and the warps of a head (two) take every second eight.
template <int DP, int HB>
__global__ void __launch_bounds__(512) paged_attention_join_kernel(const __grid_constant__ AttentionParams p)
{
    constexpr int HEADS = 8 * HB, PART = HEADS * (DP + 2), PER = DP / 32, AT_ONCE = PER <= 4 ? 8 : 4;
    __shared__ float other[8][DP + 2];
    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32, part = blockIdx.x, h = blockIdx.y * 8 + warp % 8, half = warp / 8;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Cut cut = p.cuts[part];
    if (cut.parts == 0) {
        return;
    }
    // share c: what the part began (slot 1), or the following ones went on with (slot 0)
    const float *const shares = p.parts + (uint64_t)part * 2 * PART + PART;
    auto share = [&](uint32_t c) { return shares + (c == 0 ? 0 : c * 2 * PART - PART); };
    float top = -INFINITY, all = 0.f, sum[PER] = {};
    // what stands relative to one maximum is brought to another
    auto factor = [](float from, float to) { return exp2_fast(from - (to == -INFINITY ? 0.f : to)); };
    for (uint32_t c0 = half * AT_ONCE; c0 < cut.parts; c0 += 2 * AT_ONCE) {
        float x[AT_ONCE][PER], m[AT_ONCE], l[AT_ONCE], higher = top;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const float *q = share(min(c0 + i, cut.parts - 1));
            m[i] = load_now(q + HEADS * DP + h);
            l[i] = load_now(q + HEADS * (DP + 1) + h);
#pragma unroll
            for (int k = 0; k < PER; k += 2) {
                load_now(q + h * DP + lane * PER + k, x[i][k], x[i][k + 1]);
            }
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            higher = fmaxf(higher, m[i]);    // (the last share counts again: it does not change the maximum)
        }
        const float keep = factor(top, higher);
        top = higher;
        all *= keep;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            sum[k] *= keep;
        }
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            const bool on = c0 + i < cut.parts;
            const float v = factor(m[i], top);
            all = on ? fmaf(l[i], v, all) : all;
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                sum[k] = on ? fmaf(x[i][k], v, sum[k]) : sum[k];
            }
        }
    }
    if (half == 1) {
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            other[warp % 8][lane * PER + k] = sum[k];
        }
        if (lane == 0) {
            other[warp % 8][DP] = all;
            other[warp % 8][DP + 1] = top;
        }
    }
    __syncthreads();
    if (half == 1 || h >= cut.heads) {
        return;
    }
    {
        const float theirs = other[warp][DP + 1], higher = fmaxf(top, theirs), a = factor(top, higher), b = factor(theirs, higher);
        top = higher;
        all = fmaf(all, a, other[warp][DP] * b);
#pragma unroll
        for (int k = 0; k < PER; ++k) {
            sum[k] = fmaf(sum[k], a, other[warp][lane * PER + k] * b);
        }
    }
    const uint32_t hq = cut.head0 + h;
    const float inv = all == 0.f ? 0.f : __frcp_rn(all);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const uint32_t d = lane * PER + k;
        if (d < p.cache.dim) {
            store_out(p, cut.sequence * p.out_stride + (uint64_t)hq * p.cache.dim + d, sum[k] * inv);
        }
    }
    if (p.lse != nullptr && lane == 0) {
        p.lse[(uint64_t)cut.sequence * p.heads + hq] = (top + log2f(all) - (p.i8 ? 0.f : 14.f)) * LN2;     // (Shape::LIFT)
    }
}

// The team: as many warps as leave a part for every unit, so that few units mean few shares to join (one sequence of 4000
// tokens: 11.7 us, with teams of four 15.8), and with many units no more warps than need be wait for others at a unit's end (64
// sequences of up to 8192 tokens in bytes: 135 us, with teams of sixteen 175).
template <int DP, bool I8, int HB>
EE plan(const DeviceCtx *c, AttentionParams *p, uint64_t units)
{
    using S = Shape<DP, I8, HB>;
    const uint32_t ctas = (uint32_t)c->sm_count;
    p->team = S::WARPS;
    while (p->team > S::WARPS / S::TEAMS && (uint64_t)ctas * S::WARPS / p->team < units) {
        p->team /= 2;
    }
    p->part_count = ctas * S::WARPS / p->team;
    p->share_bytes = p->part_count * 2 * S::PART * 4;
    const uint32_t tile = p->team * S::STEP, page = p->cache.page_size;
    p->step_pages = tile / page;
    p->step_at = tile % page;
    // tiles whose steps lie in 32 pages: (n - 1) tile + STEP tokens, beginning anywhere in a page
    const uint64_t room = 31ull * page, taken = (uint64_t)S::STEP + page - 2, tiles = room > taken ? (room - taken) / tile : 0;
    p->run_tiles = 1 + (uint32_t)(tiles < (1u << 20) ? tiles : (1u << 20));
    p->page_magic = page == 1 ? 0xFFFFFFFFu : (uint32_t)((1ull << 32) / page);
    return SUCCESS;
}
template <int DP, bool I8, int HB>
EE launch(DeviceCtx *c, const AttentionParams &p, cudaStream_t st)
{
    using S = Shape<DP, I8, HB>;
    const void *kernel = reinterpret_cast<const void *>(paged_attention_kernel<DP, I8, HB>);
    B200_EE(raise_smem_limit(c, (KernelFamily)(KF_ATTENTION + (DP == 64 ? 0 : (DP == 128 ? 1 : 2)) + 3 * I8 + 6 * (HB - 1)), &kernel, 1, S::SMEM));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((uint32_t)c->sm_count);
    cfg.blockDim = dim3(32 * S::WARPS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    B200_CUDA(launch_programmatic(cfg, paged_attention_kernel<DP, I8, HB>, p));
    count_launch();
    cfg.gridDim = dim3(p.part_count, HB);
    cfg.blockDim = dim3(512);
    cfg.dynamicSmemBytes = 0;
    B200_CUDA(launch_programmatic(cfg, paged_attention_join_kernel<DP, HB>, p));
    count_launch();
    return SUCCESS;
}
// f(std::integral_constant<int, DP>, std::bool_constant<I8>, std::integral_constant<int, HB>) for the call's kernel
template <bool I8, int HB, typename F>
EE by_dim(uint32_t dim, F f)
{
    using std::integral_constant;
    if (dim <= 64) {
        return f(integral_constant<int, 64>(), std::bool_constant<I8>(), integral_constant<int, HB>());
    }
    if (dim <= 128) {
        return f(integral_constant<int, 128>(), std::bool_constant<I8>(), integral_constant<int, HB>());
    }
    return f(integral_constant<int, 256>(), std::bool_constant<I8>(), integral_constant<int, HB>());
}
template <typename F>
EE by_shape(const AttentionParams &p, F f)
{
    if (p.i8) {
        return p.group <= 8 ? by_dim<true, 1>(p.cache.dim, f) : by_dim<true, 2>(p.cache.dim, f);
    }
    return p.group <= 8 ? by_dim<false, 1>(p.cache.dim, f) : by_dim<false, 2>(p.cache.dim, f);
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
        a->sequences > MAX_SEQUENCES) {
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
    p->even_bytes = 0x00FF00FFu;
    p->to_1152 = 0x64806480u;
    const uint64_t units = (uint64_t)a->sequences * cache->kv_heads * p->head_blocks;
    // tiles are counted in 32 bits (they hold 16 tokens or more)
    const uint64_t room = (uint64_t)a->table_pages * cache->page_size;
    if (units != 0 && room / 16 + 1 > 0xFFFFFFFFull / units) {
        return NOT_SUPPORTED;
    }
    return by_shape(*p, [&](auto dp, auto i8, auto hb) { return plan<dp.value, i8.value, hb.value>(*c, p, units); });
}
U32 workspace_bytes(const AttentionParams &p)
{
    return p.share_bytes + p.part_count * (U32)sizeof(Cut);
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
    *bytes = workspace_bytes(p);
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
    const U32 need = workspace_bytes(p);
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
    p.cuts = reinterpret_cast<Cut *>(reinterpret_cast<char *>(tmp) + p.share_bytes);
    return by_shape(p, [&](auto dp, auto i8, auto hb) { return launch<dp.value, i8.value, hb.value>(c, p, tls().stream); });
}

}  // extern "C"
