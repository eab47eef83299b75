// paged_attention.cu -- attention of one new token per sequence over a paged cache.
//
// out = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m), s_t = scale q . k_t: one pass over the tokens with a running maximum m;
// when it rises, what has been summed so far is scaled down.  One CTA per sequence and query head.
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
    uint32_t sequences, heads, group, table_pages, window;
    float scale, out_scale;
    int i8, q_f16, out_kind;   // 0 binary32, 1 binary16, 2 u8
    int *status;
};

// [begin, end) of a sequence's tokens
__host__ __device__ inline bool live_tokens(const AttentionParams &p, uint32_t sequence, uint32_t *begin, uint32_t *end)
{
    const int32_t n = p.length[sequence];
    const uint64_t room = (uint64_t)p.table_pages * p.cache.page_size;
    const bool good = n >= 0 && (uint64_t)n <= room;
    *end = good ? (uint32_t)n : (n < 0 ? 0u : (uint32_t)room);
    *begin = p.window != 0 && *end > p.window ? *end - p.window : 0;
    return good;
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

template <int I8>
__global__ void __launch_bounds__(128) paged_attention_kernel(const __grid_constant__ AttentionParams p)
{
    __shared__ float q[256], s[128];
    __shared__ uint64_t row[128];
    __shared__ float v_unit[128];
    __shared__ float red[2];
    const uint32_t h = blockIdx.x, b = blockIdx.y, dim = p.cache.dim, kv = h / p.group;
    for (uint32_t i = threadIdx.x; i < dim; i += 128) {
        const uint64_t at = b * p.q_stride + (uint64_t)h * dim + i;
        q[i] = p.q_f16 ? load1(reinterpret_cast<const __half *>(p.q) + at) : load1(reinterpret_cast<const float *>(p.q) + at);
    }
    uint32_t begin, end;
    if (!live_tokens(p, b, &begin, &end) && threadIdx.x == 0) {
        atomicExch(p.status, BAD_ATTENTION);
    }
    float m = -INFINITY, l = 0.f, acc[2] = {0.f, 0.f};
    for (uint32_t t0 = begin; t0 < end; t0 += 128) {
        const uint32_t t = t0 + threadIdx.x;
        float score = -INFINITY, unit = 0.f;
        uint64_t o = 0;
        uint32_t page, at;
        __syncthreads();
        if (t < end) {
            if (page_of(p.table, b, p.table_pages, p.cache.pages, p.cache.page_size, t, &page, &at)) {
                o = row_element(p.cache, page, at, kv);
                float sum = 0.f;
                for (uint32_t i = 0; i < dim; ++i) {
                    sum += q[i] * (I8 ? (float)reinterpret_cast<const int8_t *>(p.k)[o + i] : __half2float(reinterpret_cast<const __half *>(p.k)[o + i]));
                }
                unit = 1.f;
                if (I8) {
                    const uint64_t se = scale_element(p.cache, page, at, kv);
                    sum /= p.k_scale[se];
                    unit = 1.f / p.v_scale[se];
                }
                score = sum * p.scale;
            } else {
                atomicExch(p.status, BAD_ATTENTION);
                o = ~0ull;
            }
        }
        s[threadIdx.x] = score;
        row[threadIdx.x] = o;
        v_unit[threadIdx.x] = unit;
        __syncthreads();
        if (threadIdx.x == 0) {
            float mm = m;
            for (int i = 0; i < 128; ++i) {
                mm = fmaxf(mm, s[i]);
            }
            red[0] = mm;
        }
        __syncthreads();
        const float mm = red[0], base = mm == -INFINITY ? 0.f : mm, keep = expf(m - base);
        m = mm;
        l *= keep;
        acc[0] *= keep;
        acc[1] *= keep;
        const uint32_t n = min(128u, end - t0);
        for (uint32_t i = 0; i < n; ++i) {
            if (row[i] == ~0ull) {
                continue;
            }
            const float w = expf(s[i] - base);
            l += w;
            for (int j = 0; j < 2; ++j) {
                const uint32_t d = threadIdx.x + j * 128;
                if (d < dim) {
                    acc[j] += w * v_unit[i] *
                        (I8 ? (float)reinterpret_cast<const int8_t *>(p.v)[row[i] + d] : __half2float(reinterpret_cast<const __half *>(p.v)[row[i] + d]));
                }
            }
        }
    }
    for (int j = 0; j < 2; ++j) {
        const uint32_t d = threadIdx.x + j * 128;
        if (d < dim) {
            store_out(p, b * p.out_stride + (uint64_t)h * dim + d, l == 0.f ? 0.f : acc[j] / l);
        }
    }
    if (p.lse != nullptr && threadIdx.x == 0) {
        p.lse[(uint64_t)b * p.heads + h] = m + logf(l);
    }
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
U32 workspace_bytes(const AttentionParams &, const DeviceCtx *)
{
    return 0;
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
    const dim3 grid(p.heads, p.sequences);
    return p.i8 ? launch_kernel(grid, 128, 0, tls().stream, paged_attention_kernel<1>, p) : launch_kernel(grid, 128, 0, tls().stream, paged_attention_kernel<0>, p);
}

}  // extern "C"
