// k_decode.cu -- K6: attention of one new token per sequence over its cache.
//
// out = softmax(q . K^T * scale) V for each query head over the sequence's
// rows, in one pass over the cache with a running maximum and sum; the
// weights variant keeps the scores and adds exp(score - lse) to the rows'
// accumulated weights afterwards.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "epsp_kernels.h"

namespace epsp {
namespace {

constexpr int kTile = 128;

template <class T>
__device__ __forceinline__ float to_f(T x) {
    return static_cast<float>(x);
}

__device__ __forceinline__ void store_out(void* out, int32_t dtype, int64_t i, float x) {
    if (dtype == 0) static_cast<float*>(out)[i] = x;
    else if (dtype == 1) static_cast<__half*>(out)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(x);
}

// One CTA per (query head, sequence).
template <class T, int D>
__global__ void __launch_bounds__(kTile) k6_decode_plain(const DecodeArgs a, float* scores, float* lse, int stride) {
    __shared__ float qs[D], ps[kTile], red[kTile];
    __shared__ int rows[kTile];
    const int hq = blockIdx.x, s = blockIdx.y, t = threadIdx.x;
    const int G = a.n_head / a.n_head_kv, h = hq / G;
    const int n = batch_len(a.kv, s, a.err);
    const T* q = static_cast<const T*>(a.q) + ((int64_t)s * a.n_head + hq) * D;
    for (int i = t; i < D; i += kTile) qs[i] = to_f(q[i]) * a.kq_scale;
    __syncthreads();
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int j0 = 0; j0 < n; j0 += kTile) {
        const int j = j0 + t;
        float x = -INFINITY;
        if (j < n) {
            const int row = batch_row(a.kv, s, j, a.err);
            rows[t] = row;
            const bool fresh = a.k_new != nullptr && j == n - 1;
            x = 0.f;
            if (row >= 0) {
                const T* kr = fresh ? static_cast<const T*>(a.k_new) + ((int64_t)s * a.n_head_kv + h) * D
                                    : static_cast<const T*>(a.k) + ((int64_t)row * a.n_head_kv + h) * D;
                for (int i = 0; i < D; ++i) x += qs[i] * to_f(kr[i]);
                if (fresh && hq % G == 0) {
                    const T* vr = static_cast<const T*>(a.v_new) + ((int64_t)s * a.n_head_kv + h) * D;
                    for (int i = 0; i < D; ++i) {
                        static_cast<T*>(a.k)[((int64_t)row * a.n_head_kv + h) * D + i] = kr[i];
                        static_cast<T*>(a.v)[((int64_t)row * a.n_head_kv + h) * D + i] = vr[i];
                    }
                }
            }
            if (scores) scores[((int64_t)s * a.n_head + hq) * stride + j] = x;
        }
        red[t] = x;
        __syncthreads();
        for (int w = kTile / 2; w > 0; w >>= 1) {
            if (t < w) red[t] = fmaxf(red[t], red[t + w]);
            __syncthreads();
        }
        const float m2 = fmaxf(m, red[0]);
        const float ms = m2 == -INFINITY ? 0.f : m2;
        const float p = j < n ? expf(x - ms) : 0.f;
        const float alpha = expf(m - ms);
        __syncthreads();
        ps[t] = p;
        red[t] = p;
        __syncthreads();
        for (int w = kTile / 2; w > 0; w >>= 1) {
            if (t < w) red[t] += red[t + w];
            __syncthreads();
        }
        l = l * alpha + red[0];
        o *= alpha;
        if (t < D) {
            for (int i = 0; i < kTile && j0 + i < n; ++i) {
                if (rows[i] < 0) continue;
                const T* vr = a.v_new != nullptr && j0 + i == n - 1
                                  ? static_cast<const T*>(a.v_new) + ((int64_t)s * a.n_head_kv + h) * D
                                  : static_cast<const T*>(a.v) + ((int64_t)rows[i] * a.n_head_kv + h) * D;
                o += ps[i] * to_f(vr[t]);
            }
        }
        m = m2;
        __syncthreads();
    }
    if (t < D) store_out(a.out, a.out_dtype, ((int64_t)s * a.n_head + hq) * D + t, n > 0 ? o / l : 0.f);
    if (lse && t == 0) lse[(int64_t)s * a.n_head + hq] = m + logf(l);
}

__global__ void k6_add_weights(const DecodeArgs a, const float* scores, const float* lse, int stride) {
    const int h = blockIdx.y, s = blockIdx.z, j = blockIdx.x * blockDim.x + threadIdx.x;
    const int G = a.n_head / a.n_head_kv;
    if (j >= batch_len(a.kv, s, a.err)) return;
    float w = 0.f;
    for (int g = 0; g < G; ++g) {
        const int64_t i = (int64_t)s * a.n_head + h * G + g;
        w += expf(scores[i * stride + j] - lse[i]);
    }
    a.acc[((int64_t)s * a.n_head_kv + h) * a.acc_stride + j] += w;
}

}  // namespace

size_t decode_ws_bytes(int32_t n_seq, int32_t max_kv_len, int32_t n_head, int32_t, int32_t, bool weights) {
    if (!weights) return 16;
    const size_t stride = (size_t)(max_kv_len + 31) / 32 * 32;
    return ((size_t)n_seq * n_head * (stride + 1) + 16) * sizeof(float);
}

cudaError_t launch_decode(const DecodeArgs& a, cudaStream_t s) {
    float *scores = nullptr, *lse = nullptr;
    const int stride = (a.kv.max_kv_len + 31) / 32 * 32;
    if (a.acc) {
        scores = static_cast<float*>(a.ws);
        lse = scores + (size_t)a.kv.n_seq * a.n_head * stride;
    }
    const dim3 grid(a.n_head, a.kv.n_seq);
#define GO(T, D) k6_decode_plain<T, D><<<grid, kTile, 0, s>>>(a, scores, lse, stride)
    if (a.head_dim == 128) {
        if (a.dtype == 0) GO(float, 128);
        else if (a.dtype == 1) GO(__half, 128);
        else GO(__nv_bfloat16, 128);
    } else {
        if (a.dtype == 0) GO(float, 64);
        else if (a.dtype == 1) GO(__half, 64);
        else GO(__nv_bfloat16, 64);
    }
#undef GO
    cudaError_t e = cudaGetLastError();
    if (e == cudaSuccess && a.acc) {
        k6_add_weights<<<dim3((a.kv.max_kv_len + 255) / 256, a.n_head_kv, a.kv.n_seq), 256, 0, s>>>(a, scores, lse,
                                                                                                  stride);
        e = cudaGetLastError();
    }
    return e;
}

}  // namespace epsp
