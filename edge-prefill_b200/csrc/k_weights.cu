// k_weights.cu -- K7: softmax weights of a prompt's last rows over its cache.
//
// acc[h][j] = sum over the rows t and heads g of exp(x_tgj - lse_tg) with
// x = q . k * scale: first each row's lse over the keys it sees, then each
// key's sum over the rows that see it (one writer per key, fixed order).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "epsp_kernels.h"

namespace epsp {
namespace {

template <class T>
__device__ __forceinline__ float to_f(T x) {
    return static_cast<float>(x);
}

template <class T, int D>
__device__ __forceinline__ float dot_row(const WeightArgs& a, const float* qs, int j, int h) {
    bool bad = false;
    const int row = phys_row(a.paging, j, bad);
    if (bad) {
        report_error(a.err, kDevBadBlockTable, 0x92, j);
        return 0.f;
    }
    const T* kr = static_cast<const T*>(a.k) + ((int64_t)row * a.n_head_kv + h) * D;
    float x = 0.f;
    for (int i = 0; i < D; ++i) x += qs[i] * to_f(kr[i]);
    return x;
}

// One CTA per (query head, row).
template <class T, int D>
__global__ void __launch_bounds__(128) k7_stats_plain(const WeightArgs a, float* lse) {
    __shared__ float qs[D], rm[128], rl[128];
    const int hq = blockIdx.x, w = blockIdx.y, t = threadIdx.x;
    const int h = hq / (a.n_head / a.n_head_kv);
    const T* q = static_cast<const T*>(a.q) + ((int64_t)(a.row_begin + w) * a.n_head + hq) * D;
    for (int i = t; i < D; i += 128) qs[i] = to_f(q[i]) * a.kq_scale;
    __syncthreads();
    const int n = a.kv_len - a.n_tok + a.row_begin + w + 1;
    float m = -INFINITY, l = 0.f;
    for (int j = t; j < n; j += 128) {
        const float x = dot_row<T, D>(a, qs, j, h), m2 = fmaxf(m, x);
        const float ms = m2 == -INFINITY ? 0.f : m2;
        l = l * expf(m - ms) + expf(x - ms);
        m = m2;
    }
    rm[t] = m;
    rl[t] = l;
    __syncthreads();
    for (int k = 64; k > 0; k >>= 1) {
        if (t < k) {
            const float m2 = fmaxf(rm[t], rm[t + k]), ms = m2 == -INFINITY ? 0.f : m2;
            rl[t] = rl[t] * expf(rm[t] - ms) + rl[t + k] * expf(rm[t + k] - ms);
            rm[t] = m2;
        }
        __syncthreads();
    }
    if (t == 0) lse[(int64_t)w * a.n_head + hq] = rm[0] + logf(rl[0]);
}

// One thread per key of one KV head.
template <class T, int D>
__global__ void __launch_bounds__(128) k7_sums_plain(const WeightArgs a, const float* lse) {
    __shared__ float qs[D];
    const int h = blockIdx.y, j = blockIdx.x * 128 + threadIdx.x, G = a.n_head / a.n_head_kv;
    const int first = max(0, (int)(blockIdx.x * 128) - (a.kv_len - a.n_tok + a.row_begin));  // first row that sees the tile
    float sum = 0.f;
    for (int w = first; w < a.n_tok - a.row_begin; ++w)
        for (int g = 0; g < G; ++g) {
            const int hq = h * G + g;
            __syncthreads();
            for (int i = threadIdx.x; i < D; i += 128)
                qs[i] = to_f(static_cast<const T*>(a.q)[((int64_t)(a.row_begin + w) * a.n_head + hq) * D + i]) * a.kq_scale;
            __syncthreads();
            if (j <= a.kv_len - a.n_tok + a.row_begin + w)
                sum += expf(dot_row<T, D>(a, qs, j, h) - lse[(int64_t)w * a.n_head + hq]);
        }
    if (j < a.kv_len) {
        float* p = a.acc + (int64_t)h * a.acc_stride + j;
        *p = a.accumulate ? *p + sum : sum;
    }
}

template <class T, int D>
cudaError_t go(const WeightArgs& a, cudaStream_t s) {
    float* lse = static_cast<float*>(a.ws);
    const int rows = a.n_tok - a.row_begin;
    if (rows > 65535) return cudaErrorNotSupported;
    k7_stats_plain<T, D><<<dim3(a.n_head, rows), 128, 0, s>>>(a, lse);
    k7_sums_plain<T, D><<<dim3((a.kv_len + 127) / 128, a.n_head_kv), 128, 0, s>>>(a, lse);
    return cudaGetLastError();
}

}  // namespace

size_t weights_ws_bytes(int32_t, int32_t rows, int32_t n_head, int32_t) { return (size_t)rows * n_head * sizeof(float); }

cudaError_t launch_prompt_weights(const WeightArgs& a, cudaStream_t s) {
    const bool wide = a.head_dim == 128;
    switch (a.dtype) {
        case 0: return wide ? go<float, 128>(a, s) : go<float, 64>(a, s);
        case 1: return wide ? go<__half, 128>(a, s) : go<__half, 64>(a, s);
        default: return wide ? go<__nv_bfloat16, 128>(a, s) : go<__nv_bfloat16, 64>(a, s);
    }
}

}  // namespace epsp
