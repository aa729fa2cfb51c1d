// k_evict.cu -- K8: eviction by accumulated weight.
//
// K8a picks, per sequence and KV head, the rows to keep: a radix selection
// finds the weight of the last row that stays (32-bit order-preserving keys,
// most significant digit first), then one pass in row order lists the rows
// above it and the first of those equal to it.  K8b moves the listed rows.
#include "epsp_kernels.h"

namespace epsp {
namespace {

constexpr int kThreads = 1024;

// Order-preserving key of a weight: larger weight, larger key; NaN as -inf;
// +0 and -0 alike.
__device__ __forceinline__ uint32_t weight_key(float x) {
    if (x != x) x = -INFINITY;
    x += 0.f;  // -0 -> +0
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct Plan {  // per sequence, in the workspace
    int32_t n, m;
};

// Inclusive sum over the CTA's threads.
__device__ int scan_cta(int x, int* warp_sums, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int v = x;
    for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += u;
    }
    if (lane == 31) warp_sums[warp] = v;
    __syncthreads();
    if (warp == 0) {
        int w = warp_sums[lane];
        for (int d = 1; d < 32; d <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, w, d);
            if (lane >= d) w += u;
        }
        warp_sums[lane] = w;
    }
    __syncthreads();
    if (warp > 0) v += warp_sums[warp - 1];
    total = warp_sums[31];
    __syncthreads();
    return v;
}

__global__ void __launch_bounds__(kThreads) k8a_select_rows(const EvictArgs a, int32_t* list, Plan* plan, int cap) {
    __shared__ int hist[256], warp_sums[32];
    __shared__ int s_digit, s_above;
    const int h = blockIdx.x, s = blockIdx.y, t = threadIdx.x;
    const int n = batch_len(a.src, s, a.err), m = min(n, a.n_keep);
    const int64_t sh = (int64_t)s * a.n_head_kv + h;
    const float* acc = a.acc + sh * a.acc_stride;
    int32_t* out = list + sh * cap;
    if (h == 0 && t == 0) plan[s] = {n, m};
    // the candidates are rows [lo, hi); `want` of them stay
    const int lo = n > m ? a.sink_rows : n, hi = n > m ? n - a.recent_rows : n;
    const int want = n > m ? m - a.sink_rows - a.recent_rows : 0;
    uint32_t key = 0;
    int ties = 0;
    if (want > 0 && want < hi - lo) {
        int left = want;
        for (int shift = 24; shift >= 0; shift -= 8) {
            for (int i = t; i < 256; i += kThreads) hist[i] = 0;
            __syncthreads();
            for (int r = lo + t; r < hi; r += kThreads) {
                const uint32_t k = weight_key(acc[r]);
                if (shift == 24 || (k >> (shift + 8)) == (key >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
            }
            __syncthreads();
            if (t == 0) {
                int above = 0, d = 255;
                while (above + hist[d] < left) above += hist[d--];
                s_digit = d;
                s_above = above;
            }
            __syncthreads();
            key |= (uint32_t)s_digit << shift;
            left -= s_above;
            __syncthreads();
        }
        ties = left;  // rows equal to `key` that stay, the first ones
    }
    const bool all = want >= hi - lo;
    int base = 0, seen = 0;  // rows listed, rows equal to key met
    for (int r0 = 0; r0 < n; r0 += kThreads) {
        const int r = r0 + t;
        const bool cand = r >= lo && r < hi;
        const uint32_t k = cand && !all && want > 0 ? weight_key(acc[r]) : 0;
        const bool equal = cand && !all && want > 0 && k == key;
        int n_eq = 0, n_keep = 0;
        const int rank = seen + scan_cta(equal, warp_sums, n_eq);
        const bool keep = r < n && (!cand || all || (want > 0 && (k > key || (equal && rank <= ties))));
        const int at = base + scan_cta(keep, warp_sums, n_keep) - 1;
        if (keep) out[at] = r;
        base += n_keep;
        seen += n_eq;
    }
    if (a.kept_rows) {
        __syncthreads();
        for (int i = t; i < a.n_keep; i += kThreads) a.kept_rows[sh * a.n_keep + i] = i < m ? out[i] : -1;
    }
}

// One CTA per (KV head, sequence) moves in row order, so that it can also
// compact in place: a kept row never moves up.
__global__ void __launch_bounds__(kThreads) k8b_move(const EvictArgs a, const int32_t* list, const Plan* plan, int cap) {
    const int h = blockIdx.x, s = blockIdx.y, t = threadIdx.x;
    const int m = plan[s].m;
    const int64_t sh = (int64_t)s * a.n_head_kv + h;
    const int32_t* rows = list + sh * cap;
    const int row_bytes = a.head_dim * a.elem_bytes, nv = row_bytes / 16;
    const int per = kThreads / nv;
    for (int i0 = 0; i0 < m; i0 += per) {
        const int i = i0 + t / nv, c = t % nv;
        uint4 kk, vv;
        int to = -1;
        if (i < m && t < per * nv) {
            const int from = batch_row(a.src, s, rows[i], a.err);
            to = batch_row(a.dst, s, i, a.err);
            if (from < 0) to = -1;
            if (to >= 0) {
                const int64_t f = ((int64_t)from * a.n_head_kv + h) * row_bytes + c * 16;
                kk = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.k) + f);
                vv = *reinterpret_cast<const uint4*>(static_cast<const char*>(a.v) + f);
            }
        }
        __syncthreads();
        if (to >= 0) {
            const int64_t f = ((int64_t)to * a.n_head_kv + h) * row_bytes + c * 16;
            *reinterpret_cast<uint4*>(static_cast<char*>(a.k_dst) + f) = kk;
            *reinterpret_cast<uint4*>(static_cast<char*>(a.v_dst) + f) = vv;
        }
        __syncthreads();
    }
    if (a.acc_dst) {
        for (int i0 = 0; i0 < a.acc_dst_stride; i0 += kThreads) {
            const int i = i0 + t;
            const float x = i < m ? a.acc[sh * a.acc_stride + rows[i]] : 0.f;
            __syncthreads();
            if (i < a.acc_dst_stride) a.acc_dst[sh * a.acc_dst_stride + i] = x;
            __syncthreads();
        }
    }
    if (a.new_lens && h == 0 && t == 0) a.new_lens[s] = m;
}

}  // namespace

size_t evict_ws_bytes(int32_t n_seq, int32_t max_kv_len, int32_t n_keep, int32_t n_head_kv) {
    const size_t cap = n_keep < max_kv_len ? n_keep : max_kv_len;
    return (size_t)n_seq * (sizeof(Plan) + n_head_kv * cap * sizeof(int32_t));
}

cudaError_t launch_evict(const EvictArgs& a, cudaStream_t s) {
    const int cap = a.n_keep < a.src.max_kv_len ? a.n_keep : a.src.max_kv_len;
    Plan* plan = static_cast<Plan*>(a.ws);
    int32_t* list = reinterpret_cast<int32_t*>(plan + a.src.n_seq);
    const dim3 grid(a.n_head_kv, a.src.n_seq);
    k8a_select_rows<<<grid, kThreads, 0, s>>>(a, list, plan, cap);
    k8b_move<<<grid, kThreads, 0, s>>>(a, list, plan, cap);
    return cudaGetLastError();
}

}  // namespace epsp
