// kv_append.cu -- rows of new keys and values into a paged cache, rotated by position on the way; queries are rotated in
// the same launch.
//
// A pair (a, b) of a head turns by the angle of its position: a' = a cos - b sin, b' = b cos + a sin, each step one binary32
// operation, so that the rows are the same bits wherever they are computed.  HBM bound: every row is read once and written
// once, and the angles of a position are shared by the heads of a token.  16 or 32 lanes hold a row in registers, four
// neighbouring elements each: its largest magnitude (signed bytes) is a few shuffles away, and nobody reads a row twice
// except for the other halves of pairs, which come from L1.  4005 tokens of 64 + 16 heads of 128, binary32 into bytes: 47 us,
// 5.9 TB/s of the 277 MB; one token of 32 + 16 heads 2.5 us in a graph (start and three dependent loads).
#include "decode.cuh"

namespace b200 {

bool on_this_device(const void *p)
{
    if (p == nullptr) {
        return false;
    }
    if (tls().device_only) {
        return true;
    }
    cudaPointerAttributes a;
    if (cudaPointerGetAttributes(&a, p) != cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    if (a.type == cudaMemoryTypeManaged) {
        return true;
    }
    int dev = tls().device;
    if (a.type != cudaMemoryTypeDevice || (dev < 0 && cudaGetDevice(&dev) != cudaSuccess)) {
        return false;
    }
    return a.device == dev;
}

EE check_cache(const bolt_b200_kv_cache *c)
{
    if (c->k == nullptr || c->v == nullptr) {
        return NULL_POINTER;
    }
    if (c->dt != DT_F16 && c->dt != DT_I8) {
        return NOT_SUPPORTED;
    }
    const uint64_t size = c->dt == DT_F16 ? 2 : 1;
    if (c->pages == 0 || c->page_size == 0 || c->kv_heads == 0 || c->dim == 0) {
        return NOT_MATCH;
    }
    if (c->dim > 256 || c->dim * size % 16 != 0 || !aligned(c->k, 16) || !aligned(c->v, 16)) {
        return NOT_SUPPORTED;
    }
    const uint64_t strides[3] = {c->page_stride, c->token_stride, c->head_stride};
    const uint32_t counts[3] = {c->pages, c->page_size, c->kv_heads};
    for (int i = 0; i < 3; ++i) {
        if (counts[i] > 1 && strides[i] < c->dim) {
            return NOT_MATCH;
        }
        if (strides[i] > MAX_STRIDE * 64 || strides[i] * size % 16 != 0) {
            return NOT_SUPPORTED;
        }
    }
    // 2^62 bytes: more is no cache, and offsets stay within 64 bits
    if (c->pages > 0x7FFFFFFFu || c->page_size > 0x7FFFFFFFu || c->kv_heads > 65535u) {
        return NOT_SUPPORTED;
    }
    unsigned __int128 elements = c->dim;
    for (int i = 0; i < 3; ++i) {
        elements += (unsigned __int128)(counts[i] - 1) * strides[i];
    }
    if (elements * size > MAX_BYTES || (c->dt == DT_I8 && (unsigned __int128)c->pages * c->page_size * c->kv_heads * 4 > MAX_BYTES)) {
        return NOT_SUPPORTED;
    }
    if (c->dt == DT_I8) {
        if (c->k_scale == nullptr || c->v_scale == nullptr) {
            return NULL_POINTER;
        }
        if (!aligned(c->k_scale, 4) || !aligned(c->v_scale, 4)) {
            return NOT_SUPPORTED;
        }
        if (!on_this_device(c->k_scale) || !on_this_device(c->v_scale)) {
            return NOT_MATCH;
        }
    }
    return on_this_device(c->k) && on_this_device(c->v) ? SUCCESS : NOT_MATCH;
}

namespace {

struct AppendParams {
    CacheView cache;
    void *k_cache, *v_cache;
    float *k_scale, *v_scale;   // signed bytes
    const void *src[3];         // q, k, v
    uint64_t stride[3], q_out_stride;
    void *q_out;
    const int32_t *sequence, *position, *table;
    uint32_t tokens, heads, sequences, table_pages;
    uint32_t rotary, interleaved, rotary_positions;
    const float *cos, *sin;
    int i8, q_out_f16;
    int *status;
};

// ROWS neighbouring heads of a token, all queries, keys or values, by LANES lanes, VW neighbouring elements of a row at a
// time, PER times.  They share the position, the page, the angles and all but the last step of every address: with one row
// to a group of lanes 4005 tokens of 64 + 16 heads (277 MB) take 99 us, bound by the instructions.
//
// With more than a row to a group of lanes the CTAs are as many as run at a time, and each goes from task to task: the next
// one's position is asked for with this one's rows, and its rows go into L2 meanwhile (a task to a group and no more: 58.7 us, with
// binary16 rows 72.5; now 47 and 51).  Binary16 takes as many instructions a row as binary32, four elements at a time, and is bound
// by them: its bytes would take 22 us.
constexpr int RESIDENT = 4;
template <typename TIN, int VW, int LANES, int PER, int ROWS>
__global__ void __launch_bounds__(256, ROWS > 1 ? RESIDENT : 1) kv_append_kernel(const __grid_constant__ AppendParams p)
{
    const uint32_t q_groups = (p.heads + ROWS - 1) / ROWS, kv_groups = (p.cache.kv_heads + ROWS - 1) / ROWS, groups = q_groups + 2 * kv_groups;
    const uint32_t lane = threadIdx.x % LANES, dim = p.cache.dim;
    constexpr bool ON = ROWS > 1;
    const uint32_t stride = ON ? gridDim.x * (256 / LANES) : 0, further = stride / groups, further_of = stride - further * groups;
    // What a group of lanes works on: queries, keys or values (kind), so many heads from h0 on, of a token.
    struct Task {
        uint32_t token, of_token, h0, rows;
        int kind;
    };
    auto task = [&](uint32_t token, uint32_t of_token) {
        Task t = {token, of_token, 0, 0, of_token < q_groups ? 0 : (of_token < q_groups + kv_groups ? 1 : 2)};
        t.h0 = (of_token - (t.kind == 0 ? 0 : (t.kind == 1 ? q_groups : q_groups + kv_groups))) * ROWS;
        t.rows = token < p.tokens ? min((uint32_t)ROWS, (t.kind == 0 ? p.heads : p.cache.kv_heads) - t.h0) : 0;
        return t;
    };
    auto source = [&](const Task &t) { return reinterpret_cast<const TIN *>(p.src[t.kind]) + t.token * p.stride[t.kind] + (uint64_t)t.h0 * dim; };
    const uint32_t first = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    Task now = task(first / groups, first % groups);
    int32_t position = now.rows != 0 ? p.position[now.token] : -1;
    int64_t sequence = now.rows == 0 ? -1 : (p.sequence != nullptr ? p.sequence[now.token] : (int64_t)now.token);
    do {
        // Everything that does not hang on the position is asked for with it: the rows, and (y) the other halves of their pairs.
        const int kind = now.kind;
        const uint32_t token = now.token, h0 = now.h0, rows = now.rows;
        const uint32_t rotary = kind == 2 ? 0 : p.rotary, half = rotary / 2;
        const bool halves = VW == 4 && !p.interleaved;
        const TIN *const src = source(now);
        float x[ROWS][PER][VW], y[ROWS][PER][VW];
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t i = (lane + j * LANES) * VW;
            const TIN *from = src + i, *other = src + (i < half ? i + half : i - half);
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
#pragma unroll
                for (int e = 0; e < VW; ++e) {
                    x[r][j][e] = y[r][j][e] = 0.f;
                }
                if (r < rows && i < dim) {
                    if constexpr (VW == 4) {
                        load4(from, x[r][j]);
                        if (halves && i < rotary) {
                            load4(other, y[r][j]);
                        }
                    } else {
                        x[r][j][0] = load1(from);
                    }
                }
                from += dim;
                other += dim;
            }
        }
        // the next task: its position, and its rows on their way into L2
        int32_t next_position = -1;
        int64_t next_sequence = -1;
        if constexpr (ON) {
            const uint32_t of_token = now.of_token + further_of, over = of_token >= groups;
            now = task(token + further + over, over ? of_token - groups : of_token);
            if (now.rows != 0) {
                next_position = p.position[now.token];
                next_sequence = p.sequence != nullptr ? p.sequence[now.token] : (int64_t)now.token;
                if (lane * 128 < now.rows * dim * sizeof(TIN)) {
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(reinterpret_cast<const char *>(source(now)) + lane * 128));
                }
            }
        }
        // the page, asked for with the angles
        const bool turns = position >= 0 && (uint32_t)position < p.rotary_positions;
        uint32_t page = 0, at = 0;
        const bool live = position >= 0 && sequence >= 0 && sequence < (int64_t)p.sequences && (p.rotary == 0 || turns) &&
            page_of(p.table, (uint64_t)sequence, p.table_pages, p.cache.pages, p.cache.page_size, (uint32_t)position, &page, &at);
        const uint64_t angles = (uint64_t)(uint32_t)position * (p.rotary / 2);
        const float *cos = p.cos + angles, *sin = p.sin + angles;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const uint32_t i = (lane + j * LANES) * VW;
            if (!turns || i >= rotary) {
                continue;
            }
            if constexpr (VW == 4) {
                if (p.interleaved) {
                    const float c[2] = {cos[i / 2], cos[i / 2 + 1]}, s[2] = {sin[i / 2], sin[i / 2 + 1]};
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) {
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float a = x[r][j][2 * e], b = x[r][j][2 * e + 1];
                            x[r][j][2 * e] = __fsub_rn(__fmul_rn(a, c[e]), __fmul_rn(b, s[e]));
                            x[r][j][2 * e + 1] = __fadd_rn(__fmul_rn(b, c[e]), __fmul_rn(a, s[e]));
                        }
                    }
                } else {
                    float c[4], s[4];
                    load4(cos + (i < half ? i : i - half), c);
                    load4(sin + (i < half ? i : i - half), s);
                    // a' = a c + b (-s), b' = b c + a s: a sum with the negative is the difference, bit for bit
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[e] = i < half ? -s[e] : s[e];
                    }
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            x[r][j][e] = __fadd_rn(__fmul_rn(x[r][j][e], c[e]), __fmul_rn(y[r][j][e], s[e]));
                        }
                    }
                }
            } else {
                const bool first = p.interleaved ? (i & 1) == 0 : i < half;
                const uint32_t k = p.interleaved ? i / 2 : (first ? i : i - half), o = p.interleaved ? i ^ 1 : (first ? i + half : k);
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    if (r < rows) {
                        const float own = __fmul_rn(x[r][j][0], cos[k]), other = __fmul_rn(load1(src + r * dim + o), sin[k]);
                        x[r][j][0] = first ? __fsub_rn(own, other) : __fadd_rn(own, other);
                    }
                }
            }
        }
        if (position >= 0 && !live && lane == 0) {
            atomicExch(p.status, BAD_APPEND);
        }
        __syncwarp();   // q_out may be q: every lane has read its rows
        if (live) {     // (the same for all lanes of a group)
            // the rows, `step` elements apart from `to` on
            const uint64_t to = kind == 0 ? token * p.q_out_stride + (uint64_t)h0 * dim : row_element(p.cache, page, at, h0);
            const uint64_t step = kind == 0 ? dim : p.cache.head_stride;
            if (kind == 0 && !p.q_out_f16) {
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const uint32_t i = (lane + j * LANES) * VW;
                    float *d = reinterpret_cast<float *>(p.q_out) + to + i;
#pragma unroll
                    for (int r = 0; r < ROWS; ++r, d += step) {
                        if (r < rows && i < dim) {
                            if constexpr (VW == 4) {
                                *reinterpret_cast<float4 *>(d) = make_float4(x[r][j][0], x[r][j][1], x[r][j][2], x[r][j][3]);
                            } else {
                                *d = x[r][j][0];
                            }
                        }
                    }
                }
            } else if (kind == 0 || !p.i8) {
#pragma unroll
                for (int j = 0; j < PER; ++j) {
                    const uint32_t i = (lane + j * LANES) * VW;
                    __half *d = reinterpret_cast<__half *>(kind == 0 ? p.q_out : (kind == 1 ? p.k_cache : p.v_cache)) + to + i;
#pragma unroll
                    for (int r = 0; r < ROWS; ++r, d += step) {
                        if (r < rows && i < dim) {
                            if constexpr (VW == 4) {
                                *reinterpret_cast<uint2 *>(d) = make_uint2(half2_bits(x[r][j][0], x[r][j][1]), half2_bits(x[r][j][2], x[r][j][3]));
                            } else {
                                *d = __float2half_rn(x[r][j][0]);
                            }
                        }
                    }
                }
            } else {
                const unsigned mask = LANES == 32 ? 0xFFFFFFFFu : 0xFFFFu << (threadIdx.x & 16);
                uint8_t *d = reinterpret_cast<uint8_t *>(kind == 1 ? p.k_cache : p.v_cache) + to;
                float *scales = (kind == 1 ? p.k_scale : p.v_scale) + scale_element(p.cache, page, at, h0);
#pragma unroll
                for (int r = 0; r < ROWS; ++r, d += step, scales += p.cache.page_size) {
                    if (r >= rows) {
                        break;
                    }
                    int top = 0;
#pragma unroll
                    for (int j = 0; j < PER; ++j) {
#pragma unroll
                        for (int e = 0; e < VW; ++e) {
                            top = max(top, magnitude(x[r][j][e]));
                        }
                    }
#pragma unroll
                    for (int o = LANES / 2; o > 0; o >>= 1) {
                        top = max(top, __shfl_xor_sync(mask, top, o, LANES));
                    }
                    const float scale = top == 0 ? 1.0f : __fdiv_rn(127.0f, __int_as_float(top));
                    // rne, then the limits, as F32 -> I8 has it (the limits are whole numbers: their order does not matter; NaN: -127)
                    auto byte = [scale](float v) { return (uint32_t)__float2int_rn(fminf(fmaxf(__fmul_rn(v, scale), -127.f), 127.f)) & 0xFFu; };
#pragma unroll
                    for (int j = 0; j < PER; ++j) {
                        const uint32_t i = (lane + j * LANES) * VW;
                        if (i < dim) {
                            if constexpr (VW == 4) {
                                *reinterpret_cast<uint32_t *>(d + i) =
                                    byte(x[r][j][0]) | byte(x[r][j][1]) << 8 | byte(x[r][j][2]) << 16 | byte(x[r][j][3]) << 24;
                            } else {
                                d[i] = (uint8_t)byte(x[r][j][0]);
                            }
                        }
                    }
                    if (lane == 0) {
                        *scales = scale;
                    }
                }
            }
        }
        position = next_position;
        sequence = next_sequence;
    } while (ON && __any_sync(0xFFFFFFFFu, now.rows != 0));
}

template <typename TIN, int VW, int LANES, int PER, int ROWS>
EE launch_rows(const AppendParams &p, int sms, cudaStream_t st)
{
    const uint64_t groups = (uint64_t)p.tokens * ((p.heads + ROWS - 1) / ROWS + 2 * ((p.cache.kv_heads + ROWS - 1) / ROWS));
    const uint64_t ctas = (groups * LANES + 255) / 256, most = ROWS > 1 ? (uint64_t)sms * RESIDENT : ctas;
    return launch_kernel(dim3((uint32_t)(ctas < most ? ctas : most)), 256, 0, st, kv_append_kernel<TIN, VW, LANES, PER, ROWS>, p);
}
template <typename TIN>
EE launch(const AppendParams &p, bool vectors, int sms, cudaStream_t st)
{
    if (!vectors) {
        return launch_rows<TIN, 1, 32, 8, 1>(p, sms, st);
    }
    // One row to a group of lanes as long as every SM has at most 1280 of them, half of what it holds (64 tokens of 64 + 16 heads:
    // 3.5 us in a graph, 3.8 with four rows; 96 tokens: 4.7 and 3.9), two or four beyond.
    const uint64_t lanes = (uint64_t)p.tokens * (p.heads + 2 * p.cache.kv_heads) * (p.cache.dim <= 64 ? 16 : 32);
    const bool few = lanes <= (uint64_t)sms * 1280;
    if (p.cache.dim <= 64) {
        return few ? launch_rows<TIN, 4, 16, 1, 1>(p, sms, st) : launch_rows<TIN, 4, 16, 1, 4>(p, sms, st);
    }
    if (p.cache.dim <= 128) {
        return few ? launch_rows<TIN, 4, 32, 1, 1>(p, sms, st) : launch_rows<TIN, 4, 32, 1, 4>(p, sms, st);
    }
    return few ? launch_rows<TIN, 4, 32, 2, 1>(p, sms, st) : launch_rows<TIN, 4, 32, 2, 2>(p, sms, st);
}

}  // namespace
}  // namespace b200

using namespace b200;

extern "C" EE bolt_b200_kv_append(const bolt_b200_kv_cache *cache, const bolt_b200_kv_append_call *a)
{
    if (cache == nullptr || a == nullptr) {
        return NULL_POINTER;
    }
    DeviceCtx *c = ctx();
    if (c == nullptr) {
        return UNKNOWN;
    }
    B200_EE(check_cache(cache));
    if (a->tokens == 0) {
        return SUCCESS;
    }
    if (a->k == nullptr || a->v == nullptr || a->position == nullptr || a->table == nullptr || (a->heads != 0 && (a->q == nullptr || a->q_out == nullptr)) ||
        (a->rotary_dim != 0 && (a->cos == nullptr || a->sin == nullptr))) {
        return NULL_POINTER;
    }
    if ((a->dt != DT_F32 && a->dt != DT_F16) || (a->heads != 0 && a->q_out_dt != DT_F32 && a->q_out_dt != DT_F16)) {
        return NOT_SUPPORTED;
    }
    if (a->sequences == 0 || a->table_pages == 0 || (a->sequence == nullptr && a->tokens > a->sequences) || a->rotary_dim > cache->dim ||
        a->rotary_dim % 2 != 0) {
        return NOT_MATCH;
    }
    const uint64_t rows = (uint64_t)a->tokens * ((uint64_t)a->heads + 2ull * cache->kv_heads);
    if (a->heads > 65535u || rows > 0xFFFFFFFFull / 32 * 8 || (unsigned __int128)a->sequences * a->table_pages * 4 > MAX_BYTES) {
        return NOT_SUPPORTED;
    }
    const uint32_t size = a->dt == DT_F32 ? 4 : 2, q_size = a->q_out_dt == DT_F32 ? 4 : 2;
    const uint64_t q_row = (uint64_t)a->heads * cache->dim, kv_row = (uint64_t)cache->kv_heads * cache->dim;
    if (a->tokens > 1 && (a->k_stride < kv_row || a->v_stride < kv_row || (a->heads != 0 && (a->q_stride < q_row || a->q_out_stride < q_row)))) {
        return NOT_MATCH;
    }
    if (a->k_stride > MAX_STRIDE || a->v_stride > MAX_STRIDE || a->q_stride > MAX_STRIDE || a->q_out_stride > MAX_STRIDE) {
        return NOT_SUPPORTED;
    }
    if (!aligned(a->k, size) || !aligned(a->v, size) || !aligned(a->position, 4) || !aligned(a->table, 4) || !aligned(a->sequence, 4) ||
        (a->heads != 0 && (!aligned(a->q, size) || !aligned(a->q_out, q_size))) || (a->rotary_dim != 0 && (!aligned(a->cos, 4) || !aligned(a->sin, 4)))) {
        return NOT_SUPPORTED;
    }
    if (!on_this_device(a->k) || !on_this_device(a->v) || !on_this_device(a->position) || !on_this_device(a->table) ||
        (a->sequence != nullptr && !on_this_device(a->sequence)) || (a->heads != 0 && (!on_this_device(a->q) || !on_this_device(a->q_out))) ||
        (a->rotary_dim != 0 && (!on_this_device(a->cos) || !on_this_device(a->sin)))) {
        return NOT_MATCH;
    }
    AppendParams p;
    p.cache = view_of(*cache);
    p.k_cache = cache->k;
    p.v_cache = cache->v;
    p.k_scale = cache->k_scale;
    p.v_scale = cache->v_scale;
    p.src[0] = a->heads != 0 ? a->q : a->k;
    p.src[1] = a->k;
    p.src[2] = a->v;
    p.stride[0] = a->q_stride;
    p.stride[1] = a->k_stride;
    p.stride[2] = a->v_stride;
    p.q_out = a->q_out;
    p.q_out_stride = a->q_out_stride;
    p.sequence = a->sequence;
    p.position = a->position;
    p.table = a->table;
    p.tokens = a->tokens;
    p.heads = a->heads;
    p.sequences = a->sequences;
    p.table_pages = a->table_pages;
    p.rotary = a->rotary_dim;
    p.interleaved = a->interleaved != 0;
    p.rotary_positions = a->rotary_positions;
    p.cos = a->cos;
    p.sin = a->sin;
    p.i8 = cache->dt == DT_I8;
    p.q_out_f16 = a->q_out_dt == DT_F16;
    p.status = c->d_status;
    // Four elements at a time where rows and angles lie on their grid and no group of four holds rotated and other
    // elements, or both halves of its pairs; dim is a multiple of 8 (16-byte rows of the cache).
    const uint32_t q4 = size * 4;
    const bool vectors = aligned(a->k, q4) && aligned(a->v, q4) && a->k_stride % 4 == 0 && a->v_stride % 4 == 0 &&
        (a->heads == 0 || (aligned(a->q, q4) && a->q_stride % 4 == 0 && aligned(a->q_out, q_size * 4) && a->q_out_stride % 4 == 0)) &&
        (a->rotary_dim == 0 || (a->interleaved ? a->rotary_dim % 4 == 0 : a->rotary_dim % 8 == 0 && aligned(a->cos, 16) && aligned(a->sin, 16)));
    return a->dt == DT_F32 ? launch<float>(p, vectors, c->sm_count, tls().stream) : launch<__half>(p, vectors, c->sm_count, tls().stream);
}
