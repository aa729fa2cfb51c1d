// k_evict.cu -- K8: eviction by accumulated weight.
//
// K8a picks, per sequence and KV head, the rows to keep.  A radix selection
// over 32-bit order-preserving keys (digits of 11, 11 and 10 bits, most
// significant first) finds the weight of the last row that stays; then every
// row above it, and the first of those equal to it, get their place by a
// prefix sum in row order.  The rows of one head are split over a cluster of
// up to 8 CTAs, which keep their slice of the weights in registers (one read
// of the weights) and add their histograms through distributed shared
// memory; only counts are exchanged, so the result is exact and has no order.
// Latency bounds it: a histogram round is one cluster barrier and a few block
// ones; the third, and often the second, is skipped when the whole bin stays.
//
// K8b moves the listed rows, which the bytes bound: a warp takes as many rows
// as fill its lanes with eight 16-byte loads each.  In place there is an order to
// keep (a row may only be written once every row read from it has been), and
// K8c gives each CTA a 32-byte column of one head, which it compacts from the
// first row to the last: a kept row never moves up, so a step's loads need
// only be done before its own stores.
#include <cooperative_groups.h>

#include "epsp_kernels.h"

namespace epsp {
namespace {

namespace cg = cooperative_groups;

// Slices of up to 2048 rows are held by 512 threads, 4 rows each (batches of
// short sequences: 14 against 16 us with 1024 threads), longer ones by 1024
// threads, 8 or 32 rows each (64 K rows: 26 against 28 us with 512).
constexpr int kSliceS = 2048, kSliceM = 8192, kSliceL = 32768;
constexpr int kBins = 2048;
constexpr int kMaxCluster = 8;
constexpr int kSms = 148;
// Order-preserving key of a weight: larger weight, larger key; NaN as -inf;
// +0 and -0 alike.
__device__ __forceinline__ uint32_t weight_key(float x) {
    if (x != x) x = -INFINITY;
    x += 0.f;  // -0 -> +0
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct EvictPlan {
    int32_t* kept;  // [n_seq] rows kept
    int32_t* list;  // [n_seq][Hkv][cap] kept rows, ascending
    int32_t cap;
    int32_t cluster;
    int32_t slice;  // rows that a CTA of K8a holds, at most; 0: the slices are too long, read again each time
};

// Inclusive sum over the CTA's threads.
template <int kWarps, class T>
__device__ __forceinline__ T scan_cta(T x, T* warp_sums, T& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const T u = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += u;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    T w = lane < kWarps ? warp_sums[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const T u = __shfl_up_sync(0xffffffffu, w, d);
        if (lane >= d) w += u;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const T before = __shfl_sync(0xffffffffu, w, warp > 0 ? warp - 1 : 0);
    __syncthreads();
    return warp > 0 ? x + before : x;
}

// Thread t holds the KPT rows r0 + t, r0 + kThreads + t, ... of its CTA's slice
// (KPT 0: any number of rows, read from memory each time).
template <int KPT, int kThreads>
__global__ void __launch_bounds__(kThreads, 1) k8a_select_rows(const EvictArgs a, const EvictPlan p) {
    constexpr int kWarps = kThreads / 32;
    // counts of up to 32 K rows share a word with their neighbour's: half the
    // bytes to read from the other CTAs
    constexpr bool kPairs = KPT > 0;
    __shared__ __align__(8) int hist[3][kPairs ? kBins / 2 : kBins];
    constexpr int kRuns = KPT > 0 ? KPT * kWarps : 1024;  // runs of 32 rows placed at a time
    constexpr int kRunsEach = (kRuns + kThreads - 1) / kThreads;
    __shared__ uint64_t warp_sums[32], counts[kRunsEach * kThreads], mine;
    __shared__ int s_len, s_digit, s_above, s_all, warp_counts[32];
    cg::cluster_group cluster = cg::this_cluster();
    const int C = p.cluster, rank = blockIdx.x % C, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int h = blockIdx.x / C % a.n_head_kv, s = blockIdx.x / C / a.n_head_kv;
    for (int i = t; i < (int)(sizeof(hist) / 8); i += kThreads) reinterpret_cast<int2*>(&hist[0][0])[i] = make_int2(0, 0);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    // one reading of the length for the whole cluster: its CTAs must take the
    // same turns
    int n;
    if (C > 1) {
        if (rank == 0 && t == 0) s_len = batch_len(a.src, s, a.err);
        cluster.sync();
        n = *cluster.map_shared_rank(&s_len, 0);
    } else {
        if (t == 0) s_len = batch_len(a.src, s, a.err);
        __syncthreads();
        n = s_len;
    }
    const int m = min(n, a.n_keep);
    const int64_t sh = (int64_t)s * a.n_head_kv + h;
    const float* acc = a.acc + sh * a.acc_stride;
    if (h == 0 && rank == 0 && t == 0) p.kept[s] = m;
    // rows [r0, r1) are this CTA's; [lo, hi) the candidates, of which `want` stay
    const int per = ((n + C - 1) / C + 31) & ~31;
    const int r0 = min(n, rank * per), r1 = min(n, r0 + per);
    const int lo = n > m ? a.sink_rows : n, hi = n > m ? n - a.recent_rows : n;
    const int want = n > m ? m - a.sink_rows - a.recent_rows : 0;
    const bool ranked = want > 0;  // else no candidate stays (or there is none)

    float w[KPT > 0 ? KPT : 1];
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
        const int r = r0 + i * kThreads + t;
        w[i] = r < r1 ? acc[r] : 0.f;
    }
    // f(row, weight) for this thread's rows
    auto each = [&](auto&& f) {
        if constexpr (KPT > 0) {
#pragma unroll
            for (int i = 0; i < KPT; ++i)
                if (r0 + i * kThreads + t < r1) f(r0 + i * kThreads + t, w[i]);
        } else {
            for (int r = r0 + t; r < r1; r += kThreads) f(r, acc[r]);
        }
    };
    __syncthreads();
    uint32_t key = 0;
    int ties = 0, known = 0;  // rows that share the key's bits from `known` on are equal
    auto sync_all = [&]() {
        if (C > 1) cluster.sync();
        else __syncthreads();
    };
    if (ranked) {  // the same in the whole cluster
        int left = want;
        const int shifts[3] = {21, 10, 0}, bits[3] = {11, 11, 10};
#pragma unroll
        for (int d = 0; d < 3; ++d) {
            const int shift = shifts[d], bins = 1 << bits[d];
            each([&](int r, float x) {
                if (r < lo || r >= hi) return;
                const uint32_t k = weight_key(x);
                if (d == 0 || (k >> (shift + bits[d])) == (key >> (shift + bits[d]))) {
                    const int b = (k >> shift) & (bins - 1);
                    if constexpr (kPairs) atomicAdd(&hist[d][b >> 1], b & 1 ? 65536 : 1);
                    else atomicAdd(&hist[d][b], 1);
                }
            });
            sync_all();
            // thread t has per_t pairs of bins, counted from the top
            constexpr int kMost = kBins / 2 / kThreads > 0 ? kBins / 2 / kThreads : 1;
            const int per_t = bins / 2 / kThreads > 0 ? bins / 2 / kThreads : 1;
            int c0[kMost], c1[kMost], sum = 0;  // upper and lower bin of each pair, over the cluster
#pragma unroll
            for (int q = 0; q < kMost; ++q) {
                const int b = bins - 1 - 2 * (t * per_t + q);
                int2 c[kMaxCluster];
#pragma unroll
                for (int k = 0; k < kMaxCluster; ++k) {
                    c[k] = make_int2(0, 0);
                    if (q >= per_t || b < 0 || k >= C) continue;
                    const int* other = cluster.map_shared_rank(&hist[d][0], k);
                    if constexpr (kPairs) c[k].x = other[b >> 1];
                    else c[k] = *reinterpret_cast<const int2*>(other + b - 1);
                }
                c0[q] = c1[q] = 0;
#pragma unroll
                for (int k = 0; k < kMaxCluster; ++k) {
                    c0[q] += kPairs ? (int)((uint32_t)c[k].x >> 16) : c[k].y;
                    c1[q] += kPairs ? c[k].x & 0xffff : c[k].x;
                }
                sum += c0[q] + c1[q];
            }
            int total;
            int above = scan_cta<kWarps>(sum, warp_counts, total) - sum;
#pragma unroll
            for (int q = 0; q < kMost; ++q) {
                const int b = bins - 1 - 2 * (t * per_t + q), upto = above + c0[q] + c1[q];
                if (above < left && left <= upto) {
                    const bool first = left <= above + c0[q];
                    s_digit = first ? b : b - 1;
                    s_above = first ? above : above + c0[q];
                    s_all = (first ? c0[q] : c1[q]) == left - s_above;
                }
                above = upto;
            }
            __syncthreads();
            key |= (uint32_t)s_digit << shift;
            left -= s_above;
            known = shift;
            const bool all = s_all;  // the whole bin stays: no need to look into it
            __syncthreads();
            if (all) break;
        }
        ties = left;  // rows equal to `key` that stay, the first ones
    }
    // a row stays whatever comes before it, or it equals `key`
    const uint32_t edge = key >> known;
    auto mark = [&](int r, float x, bool& hard, bool& eq) {
        const bool cand = r >= lo && r < hi;
        const uint32_t k = weight_key(x) >> known;
        hard = r < r1 && (!cand || (ranked && k > edge));
        eq = r < r1 && cand && ranked && k == edge;
    };
    int32_t* list = p.list + sh * p.cap;
    int32_t* kept_rows = a.kept_rows ? a.kept_rows + sh * a.n_keep : nullptr;
    float* acc_dst = a.acc_dst && (KPT > 0 || a.acc_dst != a.acc) ? a.acc_dst + sh * a.acc_dst_stride : nullptr;
    auto place = [&](int r, float x, bool hard, bool eq, uint64_t before) {
        const uint32_t all_hard = __ballot_sync(0xffffffffu, hard), all_eq = __ballot_sync(0xffffffffu, eq);
        const uint32_t below = (1u << lane) - 1;
        const int n_hard = (int)(before >> 32) + __popc(all_hard & below);
        const int n_eq = (int)(uint32_t)before + __popc(all_eq & below);
        if (hard || (eq && n_eq < ties)) {
            const int at = n_hard + min(n_eq, ties);
            list[at] = r;
            if (kept_rows) kept_rows[at] = r;
            if (acc_dst) acc_dst[at] = x;
        }
    };
    // rows of a warp's 32 that stay in any case (upper half) and that equal `key`
    auto count = [](bool hard, bool eq) {
        const int n_hard = __popc(__ballot_sync(0xffffffffu, hard)), n_eq = __popc(__ballot_sync(0xffffffffu, eq));
        return ((uint64_t)n_hard << 32) | (uint32_t)n_eq;
    };
    // the counts of the CTAs before this one
    auto base_of = [&](uint64_t total) {
        if (t == 0) mine = total;
        sync_all();
        uint64_t v[kMaxCluster], base = 0;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) v[k] = k < rank ? *cluster.map_shared_rank(&mine, k) : 0;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) base += v[k];
        return base;
    };
    uint64_t total;
    if constexpr (KPT > 0) {
        // rows in order are runs of 32, run i * 32 + warp
        static_assert(KPT <= 32, "a bit per row");
        uint32_t hards = 0, eqs = 0;  // bit i: this thread's row i
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            bool hard, eq;
            mark(r0 + i * kThreads + t, w[i], hard, eq);
            hards |= (uint32_t)hard << i;
            eqs |= (uint32_t)eq << i;
            const uint64_t c = count(hard, eq);
            if (lane == 0) counts[i * kWarps + warp] = c;
        }
        __syncthreads();
        uint64_t own[kRunsEach], sum = 0;
#pragma unroll
        for (int e = 0; e < kRunsEach; ++e) {
            own[e] = t * kRunsEach + e < kRuns ? counts[t * kRunsEach + e] : 0;
            sum += own[e];
        }
        uint64_t before = scan_cta<kWarps>(sum, warp_sums, total) - sum;
        before += base_of(total);
#pragma unroll
        for (int e = 0; e < kRunsEach; ++e) {
            counts[t * kRunsEach + e] = before;
            before += own[e];
        }
        cluster.barrier_arrive();  // `mine` of the others has been read
        __syncthreads();
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const int r = r0 + i * kThreads + t;
            place(r, w[i], hards >> i & 1, eqs >> i & 1, counts[i * kWarps + warp]);
        }
    } else {
        uint64_t sum = 0;
        each([&](int r, float x) {
            bool hard, eq;
            mark(r, x, hard, eq);
            sum += ((uint64_t)hard << 32) | (uint32_t)eq;
        });
        scan_cta<kWarps>(sum, warp_sums, total);
        uint64_t base = base_of(total);
        cluster.barrier_arrive();
        for (int c0 = r0; c0 < r1; c0 += kRuns * 32) {
            const int runs = min(kRuns, (r1 - c0 + 31) / 32);
            auto weight = [&](int r) { return r < r1 ? acc[r] : 0.f; };
            for (int g = warp; g < runs; g += kWarps) {
                const int r = c0 + g * 32 + lane;
                bool hard, eq;
                mark(r, weight(r), hard, eq);
                const uint64_t c = count(hard, eq);
                if (lane == 0) counts[g] = c;
            }
            __syncthreads();
            uint64_t own[kRunsEach], sum = 0;
#pragma unroll
            for (int e = 0; e < kRunsEach; ++e) {
                own[e] = t * kRunsEach + e < runs ? counts[t * kRunsEach + e] : 0;
                sum += own[e];
            }
            uint64_t before = base + scan_cta<kWarps>(sum, warp_sums, total) - sum;
#pragma unroll
            for (int e = 0; e < kRunsEach; ++e) {
                counts[t * kRunsEach + e] = before;
                before += own[e];
            }
            __syncthreads();
            for (int g = warp; g < runs; g += kWarps) {
                const int r = c0 + g * 32 + lane;
                const float x = weight(r);
                bool hard, eq;
                mark(r, x, hard, eq);
                place(r, x, hard, eq, counts[g]);
            }
            base += total;
            __syncthreads();
        }
    }
    if (kept_rows)
        for (int i = m + rank * kThreads + t; i < a.n_keep; i += C * kThreads) kept_rows[i] = -1;
    if (acc_dst)
        for (int i = m + rank * kThreads + t; i < a.acc_dst_stride; i += C * kThreads) acc_dst[i] = 0.f;
    cluster.barrier_wait();  // no CTA leaves while another reads its counts
}

constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 8;  // a thread's loads under way

// Kept rows a warp moves: a row of K and V is 2 NV 16-byte vectors.
constexpr int move_rows(int nv) { return 2 * nv > 32 ? kMoveUnroll / 2 : kMoveUnroll * (32 / (2 * nv)); }

// Grid (KV head, rows / (8 warps' rows), sequence): gathers into other rows
// than the source's.
template <int NV>  // 16-byte vectors of a row
__global__ void __launch_bounds__(kMoveThreads) k8b_move(const EvictArgs a, const EvictPlan p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr int kRows = move_rows(NV);
    constexpr int kTurns = 2 * NV > 32 ? 2 * NV / 32 : 1;
    constexpr int kAtOnce = 2 * NV > 32 ? 1 : 32 / (2 * NV);
    const int h = blockIdx.x, s = blockIdx.z, lane = threadIdx.x & 31;
    const int i0 = (blockIdx.y * (kMoveThreads / 32) + (threadIdx.x >> 5)) * kRows;
    const int i = i0 + lane;
    // (the list's capacity, not the count, bounds this load: both arrive together)
    const int row = lane < kRows && i < p.cap ? p.list[((int64_t)s * a.n_head_kv + h) * p.cap + i] : -1;
    const int m = p.kept[s];
    if (a.new_lens && h == 0 && blockIdx.y == 0 && threadIdx.x == 0) a.new_lens[s] = m;
    if (i0 >= m) return;
    int from = -1, to = -1;
    if (lane < kRows && i < m) {
        from = batch_row(a.src, s, row, a.err);
        to = batch_row(a.dst, s, i, a.err);
    }
    uint4 x[kRows / kAtOnce][kTurns];
    int dst[kRows / kAtOnce];
#pragma unroll
    for (int u = 0; u < kRows / kAtOnce; ++u) {
        const int j = u * kAtOnce + (kAtOnce > 1 ? lane / (2 * NV) : 0);
        const int f = __shfl_sync(0xffffffffu, from, j), d = __shfl_sync(0xffffffffu, to, j);
        dst[u] = f >= 0 ? d : -1;
#pragma unroll
        for (int v = 0; v < kTurns; ++v) {
            const int c = (lane + v * 32) % (2 * NV);
            const void* base = c < NV ? a.k : a.v;
            if (dst[u] >= 0) x[u][v] = *(static_cast<const uint4*>(base) + ((int64_t)f * a.n_head_kv + h) * NV + c % NV);
        }
    }
#pragma unroll
    for (int u = 0; u < kRows / kAtOnce; ++u)
#pragma unroll
        for (int v = 0; v < kTurns; ++v) {
            const int c = (lane + v * 32) % (2 * NV);
            void* base = c < NV ? a.k_dst : a.v_dst;
            if (dst[u] >= 0) *(static_cast<uint4*>(base) + ((int64_t)dst[u] * a.n_head_kv + h) * NV + c % NV) = x[u][v];
        }
}

constexpr int kPlaceThreads = 512;

// Grid (2 * row bytes / 32, KV head, sequence): compacts one 32-byte column of
// K or V where it is.
__global__ void __launch_bounds__(kPlaceThreads) k8c_compact(const EvictArgs a, const EvictPlan p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int nv = a.head_dim * a.elem_bytes / 16, cols = nv / 2;  // 16-byte vectors, 32-byte columns of a row
    const int h = blockIdx.y, s = blockIdx.z, t = threadIdx.x;
    const int m = p.kept[s];
    if (a.new_lens && h == 0 && blockIdx.x == 0 && t == 0) a.new_lens[s] = m;
    uint4* base = static_cast<uint4*>((int)blockIdx.x < cols ? a.k_dst : a.v_dst);
    const int vec = (blockIdx.x % cols) * 2 + (t & 1);
    const int32_t* list = p.list + ((int64_t)s * a.n_head_kv + h) * p.cap;
    constexpr int kUnroll = 4, kRows = kPlaceThreads / 2;
    for (int i0 = 0; i0 < m; i0 += kRows * kUnroll) {
        uint4 x[kUnroll];
        int64_t to[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
            const int i = i0 + u * kRows + (t >> 1);
            to[u] = -1;
            if (i >= m || list[i] == i) continue;
            const int from = batch_row(a.src, s, list[i], a.err), d = batch_row(a.src, s, i, a.err);
            if (from < 0 || d < 0) continue;
            to[u] = ((int64_t)d * a.n_head_kv + h) * nv + vec;
            x[u] = base[((int64_t)from * a.n_head_kv + h) * nv + vec];
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (to[u] >= 0) base[to[u]] = x[u];
    }
}

constexpr int kWeightThreads = 1024;

// Grid (KV head, sequence): the weights of slices too long for registers,
// compacted where they are.
__global__ void __launch_bounds__(kWeightThreads) k8d_compact_weights(const EvictArgs a, const EvictPlan p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int64_t sh = (int64_t)blockIdx.y * a.n_head_kv + blockIdx.x;
    const int m = p.kept[blockIdx.y];
    float* acc = a.acc_dst + sh * a.acc_dst_stride;
    for (int i0 = 0; i0 < a.acc_dst_stride; i0 += kWeightThreads) {
        const int i = i0 + threadIdx.x;
        const float x = i < m ? acc[p.list[sh * p.cap + i]] : 0.f;
        __syncthreads();
        if (i < a.acc_dst_stride) acc[i] = x;
    }
}

// ---------------------------------------------------------------- host side --
size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

size_t plan_of(int32_t n_seq, int32_t max_kv_len, int32_t n_keep, int32_t n_head_kv, char* ws, EvictPlan* p) {
    p->cap = n_keep < max_kv_len ? n_keep : max_kv_len;
    // One CTA per head when that fills the device; more for slices over 8 K
    // rows, and where few heads leave SMs idle, down to 2 K rows.  (64 heads of
    // 16 K rows: 67 us with clusters of 8, 35 with 4, 24 with 2.)
    const int64_t runs = (int64_t)n_seq * n_head_kv;
    auto slice = [&](int cluster) { return ((max_kv_len + cluster - 1) / cluster + 31) & ~31; };
    p->cluster = 1;
    while (p->cluster < kMaxCluster &&
           (slice(p->cluster) > kSliceM || (slice(p->cluster) > kSliceS && runs * p->cluster * 2 <= kSms)))
        p->cluster *= 2;
    const int each = slice(p->cluster);
    p->slice = each <= kSliceS ? kSliceS : each <= kSliceM ? kSliceM : each <= kSliceL ? kSliceL : 0;
    p->kept = reinterpret_cast<int32_t*>(ws);
    const size_t head = up16((size_t)n_seq * sizeof(int32_t));
    p->list = reinterpret_cast<int32_t*>(ws + head);
    return head + up16((size_t)n_seq * n_head_kv * p->cap * sizeof(int32_t));
}

template <class... P, class... A>
cudaError_t launch_after(void (*k)(P...), dim3 grid, int threads, cudaStream_t s, const A&... args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k, args...);
}

}  // namespace

size_t evict_ws_bytes(int32_t n_seq, int32_t max_kv_len, int32_t n_keep, int32_t n_head_kv) {
    EvictPlan p{};
    return plan_of(n_seq, max_kv_len, n_keep, n_head_kv, nullptr, &p);
}

cudaError_t launch_evict(const EvictArgs& a, cudaStream_t s) {
    EvictPlan p{};
    plan_of(a.src.n_seq, a.src.max_kv_len, a.n_keep, a.n_head_kv, static_cast<char*>(a.ws), &p);
    const int64_t ctas = (int64_t)a.src.n_seq * a.n_head_kv * p.cluster;
    if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(p.slice == kSliceS ? 512 : 1024);
    cfg.stream = s;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = p.cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    cudaError_t e = p.slice == kSliceS   ? cudaLaunchKernelEx(&cfg, k8a_select_rows<4, 512>, a, p)
                    : p.slice == kSliceM ? cudaLaunchKernelEx(&cfg, k8a_select_rows<8, 1024>, a, p)
                    : p.slice == kSliceL ? cudaLaunchKernelEx(&cfg, k8a_select_rows<32, 1024>, a, p)
                                         : cudaLaunchKernelEx(&cfg, k8a_select_rows<0, 1024>, a, p);
    if (e != cudaSuccess) return e;
    const int nv = a.head_dim * a.elem_bytes / 16;
    if (a.in_place) {
        e = launch_after(k8c_compact, dim3(nv, a.n_head_kv, a.src.n_seq), kPlaceThreads, s, a, p);
    } else {
        const int rows = move_rows(nv) * (kMoveThreads / 32);
        const dim3 grid(a.n_head_kv, (p.cap + rows - 1) / rows, a.src.n_seq);
        if (nv == 8) e = launch_after(k8b_move<8>, grid, kMoveThreads, s, a, p);
        else if (nv == 16) e = launch_after(k8b_move<16>, grid, kMoveThreads, s, a, p);
        else e = launch_after(k8b_move<32>, grid, kMoveThreads, s, a, p);
    }
    if (e == cudaSuccess && a.acc_dst == a.acc && p.slice == 0) {
        k8d_compact_weights<<<dim3(a.n_head_kv, a.src.n_seq), kWeightThreads, 0, s>>>(a, p);
        e = cudaGetLastError();
    }
    return e;
}

}  // namespace epsp
