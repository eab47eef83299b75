// lora.cu -- low-rank adapters of many requests beside a shared projection: y += s (x A^T) B^T for every segment of rows.
//
// Two kernels: the inner sums t = x A^T into the workspace, then y.
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
    int u8;
    float *t;   // [rows][rank]
    int *status;
};

// adapter of a row, or -1
__device__ __forceinline__ int adapter_of(const LoraParams &p, uint32_t row)
{
    int32_t top = 0;
    for (uint32_t s = 0; s < p.segments; ++s) {
        const int32_t f = p.first_row[s], e = p.first_row[s + 1];
        top = max(top, f);
        if (f < top || e < f || (uint32_t)e > p.rows || p.adapter[s] >= (int32_t)p.adapters) {
            atomicExch(p.status, BAD_LORA);
            continue;
        }
        if (row >= (uint32_t)f && row < (uint32_t)e) {
            return p.adapter[s] < 0 ? -1 : p.adapter[s];
        }
    }
    return -1;
}

__global__ void __launch_bounds__(128) lora_inner_kernel(const __grid_constant__ LoraParams p)
{
    const uint32_t row = blockIdx.x, r = blockIdx.y * 4 + threadIdx.x / 32, lane = threadIdx.x % 32;
    const int ad = adapter_of(p, row);
    if (ad < 0) {
        return;
    }
    const __half *a = p.a + ((uint64_t)ad * p.rank + r) * p.a_stride;
    float sum = 0.f;
    for (uint32_t k = lane; k < p.K; k += 32) {
        const uint64_t at = row * p.x_stride + k;
        const float x = p.u8 ? (float)((int)reinterpret_cast<const uint8_t *>(p.x)[at] - 128) : reinterpret_cast<const float *>(p.x)[at];
        sum += x * __half2float(a[k]);
    }
    for (int s = 16; s > 0; s >>= 1) {
        sum += __shfl_xor_sync(0xFFFFFFFFu, sum, s);
    }
    if (lane == 0) {
        const float unit = !p.u8 ? 1.f : (p.row_scale != nullptr ? p.row_scale[row] : (p.d_sA != nullptr ? *p.d_sA : p.sA));
        p.t[(uint64_t)row * p.rank + r] = sum * (p.scale != nullptr ? p.scale[ad] : 1.f) / unit;
    }
}
__global__ void __launch_bounds__(128) lora_outer_kernel(const __grid_constant__ LoraParams p)
{
    const uint32_t row = blockIdx.x, n = blockIdx.y * 128 + threadIdx.x;
    const int ad = adapter_of(p, row);
    if (ad < 0 || n >= p.N) {
        return;
    }
    const __half *b = p.b + ((uint64_t)ad * p.N + n) * p.rank;
    float sum = 0.f;
    for (uint32_t r = 0; r < p.rank; ++r) {
        sum += p.t[(uint64_t)row * p.rank + r] * __half2float(b[r]);
    }
    p.y[row * p.y_stride + n] += sum;
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
        a->adapters > 0x7FFFFFFFu || a->segments > (1u << 20)) {
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
    p->status = (*c)->d_status;
    return SUCCESS;
}
U32 workspace_bytes(const LoraParams &p, const DeviceCtx *)
{
    return p.rows * p.rank * 4;
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
    *bytes = workspace_bytes(p, c);
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
    if (tmpBytes < workspace_bytes(p, c)) {
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
    B200_EE(launch_kernel(dim3(p.rows, p.rank / 4), 128, 0, st, lora_inner_kernel, p));
    return launch_kernel(dim3(p.rows, (p.N + 127) / 128), 128, 0, st, lora_outer_kernel, p);
}

}  // extern "C"
