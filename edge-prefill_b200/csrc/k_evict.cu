// k_evict.cu -- K8: eviction by accumulated weight.
//
// K8a picks, per sequence and KV head, the rows to keep.  A radix selection
// over 32-bit order-preserving keys (digits of 11, 11 and 10 bits, most
// significant first) finds the weight of the last row that stays; then every
// row above it, and the first of those equal to it, get their place by a
// prefix sum in row order.  The rows of one head are split over a cluster of
// up to 8 CTAs, which keep their slice of the weights in registers (one read
// of the weights), count in their own shared memory and add the bins that are
// not empty to every CTA's counts; only counts are exchanged, so the result is
// exact and has no order.  Latency bounds it: a histogram round is one cluster
// barrier and a few block ones; the third, and often the second, is skipped
// when the whole bin stays.  (Reading all bins of all CTAs instead: 64 K rows
// 24 us against 22; each CTA summing a share of the bins, two barriers: 23.)
//
// K8b moves the listed rows, which the bytes bound: a warp takes as many rows
// as fill its lanes with eight 16-byte loads each.  In place there is an order to
// keep (a row may only be written once every row read from it has been), and
// K8c gives each CTA a 32-byte column of one head, which it compacts from the
// first row to the last: a kept row never moves up, so a step's loads need
// only be done before its own stores.
#include <type_traits>

#include "epsp_kernels.h"
#include "tc100.cuh"

namespace epsp {
namespace {

// Slices of up to 2048 rows are held by 512 threads, 4 rows each (batches of
// short sequences: 11 against 14 us with 1024 threads), longer ones by 1024
// threads, 8 or 32 rows each (64 heads of 16 K rows: 20 against 22 us with 512).
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
    int32_t per;    // rows of a CTA of K8a
    int32_t slice;  // rows that it can hold; 0: they are too many, read again each time
};

// Inclusive sum over the CTA's threads.  `warp_sums` is this call's alone: no
// barrier comes after its last reading.
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
    return warp > 0 ? x + before : x;
}

struct Choice {
    int digit, above, all;
};

// Thread t holds the KPT rows from r0 + t KPT on of its CTA's slice (KPT 0:
// any number of rows, read from memory each time).
template <int KPT, int kThreads>
__global__ void __launch_bounds__(kThreads, 1) k8a_select_rows(const EvictArgs a, const EvictPlan p) {
    constexpr int kWarps = kThreads / 32;
    // counts of the cluster's rows per bin and digit; a cluster's CTAs count in
    // `own` first and then add the bins that are not empty, mostly few, to the
    // counts of all
    __shared__ __align__(16) int bins_of[3][kBins], own[kBins];
    constexpr int kRuns = KPT > 0 ? 1 : 1024;  // KPT 0: runs of 32 rows placed at a time
    __shared__ uint64_t run_counts[kRuns], totals[kMaxCluster], run_sums[2][32];
    __shared__ int digit_sums[3][32];
    __shared__ uint32_t place_sums[32];
    __shared__ Choice choice[3];
    __shared__ int s_len;
    const int C = p.cluster, rank = blockIdx.x % C, t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int h = blockIdx.x / C % a.n_head_kv, s = blockIdx.x / C / a.n_head_kv;
    for (int i = t; i < 3 * kBins / 4; i += kThreads) reinterpret_cast<int4*>(bins_of)[i] = make_int4(0, 0, 0, 0);
    if (C > 1)
        for (int i = t; i < kBins / 4; i += kThreads) reinterpret_cast<int4*>(own)[i] = make_int4(0, 0, 0, 0);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int64_t sh = (int64_t)s * a.n_head_kv + h;
    const float* acc = a.acc + sh * a.acc_stride;
    const int r0 = rank * p.per, mine = r0 + t * KPT;
    float w[KPT > 0 ? KPT : 1] = {};
    auto load = [&](int end) {
        if constexpr (KPT > 0) {
            const bool quads = (reinterpret_cast<uintptr_t>(acc + r0) & 15) == 0;
#pragma unroll
            for (int i = 0; i < KPT; i += 4) {
                float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
                if (quads && mine + i + 4 <= end) {
                    x = *reinterpret_cast<const float4*>(acc + mine + i);
                } else {
                    if (mine + i < end) x.x = acc[mine + i];
                    if (mine + i + 1 < end) x.y = acc[mine + i + 1];
                    if (mine + i + 2 < end) x.z = acc[mine + i + 2];
                    if (mine + i + 3 < end) x.w = acc[mine + i + 3];
                }
                w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
            }
        }
    };
    // one reading of the length for the whole cluster: its CTAs must take the
    // same turns.  (Weights of rows past it come along where the CTA would have
    // nothing else to do.)
    int n;
    if (C > 1) {
        if (t == 0 && rank == 0) s_len = batch_len(a.src, s, a.err);
        load(min(a.src.max_kv_len, r0 + p.per));
        tc::cluster_sync();
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(n) : "r"(tc::peer_of(&s_len, 0)) : "memory");
    } else {
        if (t == 0) s_len = batch_len(a.src, s, a.err);
        __syncthreads();
        n = s_len;
        load(n);
    }
    const int m = min(n, a.n_keep);
    if (h == 0 && rank == 0 && t == 0) p.kept[s] = m;
    // rows [r0, r1) are this CTA's; [lo, hi) the candidates, of which `want` stay
    const int r1 = min(n, r0 + p.per);
    const int lo = n > m ? a.sink_rows : n, hi = n > m ? n - a.recent_rows : n;
    const int want = n > m ? m - a.sink_rows - a.recent_rows : 0;
    const bool ranked = want > 0;  // else no candidate stays (or there is none)

    constexpr bool kKeys = KPT > 0 && KPT <= 8;  // registers for the keys too
    uint32_t keys[kKeys ? KPT : 1];
    if constexpr (kKeys) {
#pragma unroll
        for (int i = 0; i < KPT; ++i) keys[i] = weight_key(w[i]);
    }
    auto key_of = [&](int i) {
        if constexpr (kKeys) return keys[i];
        else return weight_key(w[i]);
    };
    uint32_t cands = 0;  // bit i: this thread's row i is a candidate
#pragma unroll
    for (int i = 0; i < KPT; ++i) cands |= (uint32_t)(mine + i >= lo && mine + i < min(r1, hi)) << i;
    uint32_t key = 0;
    int ties = 0, known = 0;  // rows that share the key's bits from `known` on are equal
    if (ranked) {  // the same in the whole cluster
        int left = want;
        // one digit; true when all of its bin stays
        auto round = [&](auto digit) {
            constexpr int d = decltype(digit)::value, shift = d == 0 ? 21 : d == 1 ? 10 : 0, bits = d < 2 ? 11 : 10;
            constexpr int bins = 1 << bits;
            int* hist = C > 1 ? own : bins_of[d];
            auto add = [&](uint32_t k) {
                if (d == 0 || (k >> (shift + bits) % 32) == (key >> (shift + bits) % 32))
                    atomicAdd(&hist[(k >> shift) & (bins - 1)], 1);
            };
            if constexpr (KPT > 0) {
#pragma unroll
                for (int i = 0; i < KPT; ++i)
                    if (cands >> i & 1) add(key_of(i));
            } else {
                for (int r = max(r0, lo) + t; r < min(r1, hi); r += kThreads) add(weight_key(acc[r]));
            }
            __syncthreads();
            if (C > 1) {
                for (int b = t; b < bins; b += kThreads) {
                    const int c = own[b];
                    if (c == 0) continue;
                    own[b] = 0;
                    for (int k = 0; k < C; ++k)
                        asm volatile("red.relaxed.cluster.shared::cluster.add.u32 [%0], %1;" ::"r"(
                                         tc::peer_of(&bins_of[d][b], k)),
                                     "r"(c)
                                     : "memory");
                }
                tc::cluster_sync();
            }
            // thread t has kEach bins, counted from the top
            constexpr int kEach = bins / kThreads > 0 ? bins / kThreads : 1;
            int c[kEach], sum = 0;
#pragma unroll
            for (int q = 0; q < kEach; ++q) {
                c[q] = bins_of[d][bins - 1 - (t * kEach + q)];
                sum += c[q];
            }
            int total;
            int above = scan_cta<kWarps>(sum, digit_sums[d], total) - sum;
#pragma unroll
            for (int q = 0; q < kEach; ++q) {
                if (above < left && left <= above + c[q])
                    choice[d] = {bins - 1 - (t * kEach + q), above, c[q] == left - above};
                above += c[q];
            }
            __syncthreads();
            key |= (uint32_t)choice[d].digit << shift;
            left -= choice[d].above;
            known = shift;
            return choice[d].all != 0;  // the whole bin stays: no need to look into it
        };
        if (!round(std::integral_constant<int, 0>()) && !round(std::integral_constant<int, 1>()))
            round(std::integral_constant<int, 2>());
        ties = left;  // rows equal to `key` that stay, the first ones
    }
    // a row stays whatever comes before it, or it equals `key`
    const uint32_t edge = key >> known;
    int32_t* list = p.list + sh * p.cap;
    int32_t* kept_rows = a.kept_rows ? a.kept_rows + sh * a.n_keep : nullptr;
    float* acc_dst = a.acc_dst && (KPT > 0 || a.acc_dst != a.acc) ? a.acc_dst + sh * a.acc_dst_stride : nullptr;
    auto put = [&](int at, int r, float x) {
        list[at] = r;
        if (kept_rows) kept_rows[at] = r;
        if (acc_dst) acc_dst[at] = x;
    };
    // the counts of the CTAs before this one (the last that CTAs have of one
    // another: they may leave when they like)
    auto base_of = [&](uint64_t total) {
        uint64_t base = 0;
        if (C > 1) {
            if (t < C)
                asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(tc::peer_of(&totals[rank], t)), "l"(total) : "memory");
            tc::cluster_sync();
            for (int k = 0; k < rank; ++k) base += totals[k];
        }
        return base;
    };
    if constexpr (KPT > 0) {
        static_assert(KPT <= 32 && KPT * kThreads < 65536, "a bit per row, 16 bits per count");
        uint32_t hards = 0, eqs = 0;
#pragma unroll
        for (int i = 0; i < KPT; ++i) hards |= (uint32_t)(mine + i < r1) << i;
        hards &= ~cands;
        if (ranked) {
#pragma unroll
            for (int i = 0; i < KPT; ++i) {
                const uint32_t k = key_of(i) >> known;
                hards |= (cands >> i & 1 & (uint32_t)(k > edge)) << i;
                eqs |= (cands >> i & 1 & (uint32_t)(k == edge)) << i;
            }
        }
        const uint32_t sum = (uint32_t)__popc(hards) << 16 | (uint32_t)__popc(eqs);
        uint32_t total;
        const uint32_t before = scan_cta<kWarps>(sum, place_sums, total) - sum;
        const uint64_t base = base_of((uint64_t)(total >> 16) << 32 | (total & 0xffff));
        int n_hard = (int)(base >> 32) + (int)(before >> 16), n_eq = (int)(uint32_t)base + (int)(before & 0xffff);
#pragma unroll
        for (int i = 0; i < KPT; ++i) {
            const bool hard = hards >> i & 1, eq = eqs >> i & 1;
            if (hard || (eq && n_eq < ties)) put(n_hard + min(n_eq, ties), mine + i, w[i]);
            n_hard += hard;
            n_eq += eq;
        }
    } else {
        auto mark = [&](int r, float x, bool& hard, bool& eq) {
            const bool cand = r >= lo && r < hi;
            const uint32_t k = weight_key(x) >> known;
            hard = r < r1 && (!cand || (ranked && k > edge));
            eq = r < r1 && cand && ranked && k == edge;
        };
        uint64_t sum = 0, total;
        for (int r = r0 + t; r < r1; r += kThreads) {
            bool hard, eq;
            mark(r, acc[r], hard, eq);
            sum += ((uint64_t)hard << 32) | (uint32_t)eq;
        }
        scan_cta<kWarps>(sum, run_sums[0], total);
        uint64_t base = base_of(total);
        static_assert(kRuns <= kThreads || KPT > 0, "a run per thread");
        for (int c0 = r0; c0 < r1; c0 += kRuns * 32) {
            const int runs = min(kRuns, (r1 - c0 + 31) / 32);
            for (int g = warp; g < runs; g += kWarps) {
                const int r = c0 + g * 32 + lane;
                bool hard, eq;
                mark(r, r < r1 ? acc[r] : 0.f, hard, eq);
                const uint32_t all_hard = __ballot_sync(0xffffffffu, hard), all_eq = __ballot_sync(0xffffffffu, eq);
                if (lane == 0) run_counts[g] = (uint64_t)__popc(all_hard) << 32 | (uint32_t)__popc(all_eq);
            }
            __syncthreads();
            const uint64_t mine_sum = t < runs ? run_counts[t] : 0;
            const uint64_t before = base + scan_cta<kWarps>(mine_sum, run_sums[1], total) - mine_sum;
            if (t < runs) run_counts[t] = before;
            __syncthreads();
            for (int g = warp; g < runs; g += kWarps) {
                const int r = c0 + g * 32 + lane;
                const float x = r < r1 ? acc[r] : 0.f;
                bool hard, eq;
                mark(r, x, hard, eq);
                const uint32_t all_hard = __ballot_sync(0xffffffffu, hard), all_eq = __ballot_sync(0xffffffffu, eq);
                const uint32_t below = (1u << lane) - 1;
                const int n_hard = (int)(run_counts[g] >> 32) + __popc(all_hard & below);
                const int n_eq = (int)(uint32_t)run_counts[g] + __popc(all_eq & below);
                if (hard || (eq && n_eq < ties)) put(n_hard + min(n_eq, ties), r, x);
            }
            base += total;
            __syncthreads();
        }
    }
    if (kept_rows)
        for (int i = m + rank * kThreads + t; i < a.n_keep; i += C * kThreads) kept_rows[i] = -1;
    if (acc_dst)
        for (int i = m + rank * kThreads + t; i < a.acc_dst_stride; i += C * kThreads) acc_dst[i] = 0.f;
}

constexpr int kMoveThreads = 256;
constexpr int kMoveUnroll = 8;  // a thread's loads under way

// Kept rows a warp moves: a row of K and V is 2 NV 16-byte vectors.
constexpr int move_rows(int nv) { return 2 * nv > 32 ? kMoveUnroll / 2 : kMoveUnroll * (32 / (2 * nv)); }

// Grid (rows / (8 warps' rows) * KV heads, 1, sequence): gathers into other rows
// than the source's.
template <int NV>  // 16-byte vectors of a row
__global__ void __launch_bounds__(kMoveThreads) k8b_move(const EvictArgs a, const EvictPlan p) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    constexpr int kRows = move_rows(NV);
    constexpr int kTurns = 2 * NV > 32 ? 2 * NV / 32 : 1;
    constexpr int kAtOnce = 2 * NV > 32 ? 1 : 32 / (2 * NV);
    const int h = blockIdx.x % a.n_head_kv, s = blockIdx.z, lane = threadIdx.x & 31;
    const int i0 = (blockIdx.x / a.n_head_kv * (kMoveThreads / 32) + (threadIdx.x >> 5)) * kRows;
    const int i = i0 + lane;
    // (the list's capacity, not the count, bounds this load: both arrive together)
    const int row = lane < kRows && i < p.cap ? p.list[((int64_t)s * a.n_head_kv + h) * p.cap + i] : -1;
    const int m = p.kept[s];
    if (a.new_lens && blockIdx.x == 0 && threadIdx.x == 0) a.new_lens[s] = m;
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
    // 16 K rows: 40 us with clusters of 8, 28 with 4, 20 with 2.)
    const int64_t runs = (int64_t)n_seq * n_head_kv;
    auto slice = [&](int cluster) { return ((max_kv_len + cluster - 1) / cluster + 31) & ~31; };
    p->cluster = 1;
    while (p->cluster < kMaxCluster &&
           (slice(p->cluster) > kSliceM || (slice(p->cluster) > kSliceS && runs * p->cluster * 2 <= kSms)))
        p->cluster *= 2;
    const int each = p->per = slice(p->cluster);
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
    const int nv = a.head_dim * a.elem_bytes / 16, rows = move_rows(nv) * (kMoveThreads / 32);
    const int64_t ctas = (int64_t)a.src.n_seq * a.n_head_kv * p.cluster;
    const int64_t moves = ((int64_t)p.cap + rows - 1) / rows * a.n_head_kv;  // in x: y and z hold 65535
    if (ctas > 0x7fffffff || moves > 0x7fffffff || a.n_head_kv > 65535) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(p.slice == kSliceS ? 512 : 1024);
    cfg.stream = s;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = p.cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = p.cluster > 1 ? 2 : 1;
    cudaError_t e = p.slice == kSliceS   ? cudaLaunchKernelEx(&cfg, k8a_select_rows<4, 512>, a, p)
                    : p.slice == kSliceM ? cudaLaunchKernelEx(&cfg, k8a_select_rows<8, 1024>, a, p)
                    : p.slice == kSliceL ? cudaLaunchKernelEx(&cfg, k8a_select_rows<32, 1024>, a, p)
                                         : cudaLaunchKernelEx(&cfg, k8a_select_rows<0, 1024>, a, p);
    if (e != cudaSuccess) return e;
    if (a.in_place) {
        e = launch_after(k8c_compact, dim3(nv, a.n_head_kv, a.src.n_seq), kPlaceThreads, s, a, p);
    } else {
        const dim3 grid((unsigned)moves, 1, a.src.n_seq);
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
