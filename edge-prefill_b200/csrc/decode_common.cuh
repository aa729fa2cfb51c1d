// decode_common.cuh -- what the decode kernels over 16-bit / f32 caches (k_decode.cu)
// and over 8-bit ones (k_decode8.cu) share: the split of a batch's units over the
// CTAs, the joins of what several CTAs have of a run, small helpers.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cstdint>

#include "epsp_kernels.h"
#include "tc100.cuh"

namespace epsp {
namespace {

constexpr int kUnit = 32;      // cache rows per unit
constexpr int kCtas = 148;     // one per SM
constexpr int kMinUnits = 4;  // fewest units dealt to a CTA
// What a run costs a CTA besides its units (the merge of the warps' states),
// in units: the ranges are equal in this measure.  (EPSP_RUN_COST: the file that
// includes this one has another.)
#ifndef EPSP_RUN_COST
#define EPSP_RUN_COST 6
#endif
constexpr int kRunCost = EPSP_RUN_COST;
constexpr int kLensOnChip = 1024;  // lengths a CTA keeps in shared memory
constexpr float kLog2e = 1.4426950408889634f;
// Calls that skip the split and the join: one CTA per run of at most
// kDirectUnits units, or a cluster of up to 8 CTAs per run, joined in shared
// memory, with kClusterUnits units for each CTA (twice as many where the
// cluster may not grow, but for weights, which then pay: 1500 rows, 12 us
// against 10 by the split).  1000 rows, 14 heads: 8 us against 10 by the
// split, f32 11.5 against 14.3, with weights 10 against 12.
constexpr int kDirectUnits = 16;
constexpr int kMaxCluster = 8;
constexpr int kClusterUnits = 4;
// CTAs of all clusters together: 14 clusters of 8 run at once (8 us), 16 do
// not (12 us).
constexpr int kClusterCtas = 112;

struct DecodeSplit {
    int32_t ctas;      // grid
    int32_t direct;    // a cluster per run, of
    int32_t cluster;   // so many CTAs
    int32_t fused;     // direct, and the weights are added by the same CTAs
    int32_t by_run;    // cut has a place per run (no more runs than CTAs), not one per CTA
    int32_t joins;     // places of cut
    int32_t pass_heads;  // query heads of a pass, at most
    int32_t passes;    // passes per KV head
    int32_t groups;    // warps that share a unit (1, 2, 4, 8)
    int32_t heads;     // query heads per warp
    int32_t score_stride;
    // workspace
    int32_t* per;        // cost per CTA
    int32_t* run_start;  // [n_seq][Hkv][passes] where each run starts in the cost of all
    int32_t* lens;       // [n_seq] this call's view of the lengths (more sequences than a CTA keeps on chip)
    int4* cut;           // [joins] (sequence, run, start, units) of a run that goes on past the CTA it began in; -1: none
    float* part_o;       // [2 ctas][groups * 8][D]
    float2* part_ml;     // [2 ctas][groups * 8] (maximum, sum), log2 units
    float* lse;          // [n_seq][n_head] log2 units, runs finished by one CTA
    float* scores;       // [n_seq][n_head][score_stride] log2 units
};

__host__ __device__ __forceinline__ int units_of(int n) { return (n + kUnit - 1) / kUnit; }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <bool BF16>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if constexpr (BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Two floats to 16 bits, and what the rounding left over.
template <bool BF16>
__device__ __forceinline__ uint32_t split2(float& x, float& y) {
    uint32_t u;
    if constexpr (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x, y);
        u = *reinterpret_cast<const uint32_t*>(&v);
        x -= __uint_as_float(u << 16);
        y -= __uint_as_float(u & 0xffff0000u);
    } else {
        const __half2 v = __floats2half2_rn(x, y);
        u = *reinterpret_cast<const uint32_t*>(&v);
        const float2 f = __half22float2(v);
        x -= f.x;
        y -= f.y;
    }
    return u;
}

__device__ __forceinline__ void store4(void* out, int32_t dtype, int64_t i, float4 x) {
    if (dtype == 0) {
        *reinterpret_cast<float4*>(static_cast<float*>(out) + i) = x;
    } else if (dtype == 1) {
        const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
        *reinterpret_cast<uint2*>(static_cast<__half*>(out) + i) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x.x, x.y), b = __floats2bfloat162_rn(x.z, x.w);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(out) + i) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
}
static_assert(kUnit == 32, "a lane per row, a page holds whole units of 2^5 rows");

// The sequences' lengths: on chip when there are few, else the copy that
// k6_lengths made.  Either way a CTA reads each once, or from memory that
// nobody else writes: its warps must agree on the segments they meet at.
struct Lens {
    const int32_t* chip;
    __device__ __forceinline__ int32_t at(const DecodeArgs& a, int s) const {
        return chip != nullptr ? chip[s] : batch_len(a.kv, s, a.err);
    }
};

// Walks the segments (a run's part inside this CTA) of a CTA's units.
struct Walk {
    int32_t s, run, u, n, units;  // sequence, run within it (h * passes + pass), next unit, length, units of the run
    int32_t left;                 // cost of the CTA's range from here on
    int32_t at;                   // where the run starts in the cost of all
    int32_t per;                  // cost of a CTA's range
    int32_t whole;                // log2 of the rows of a page that one CTA attends (the last page of a run, which the
                                  // call writes a row into); 0: any unit may end a CTA's range

    // First unit of the run's last page where one CTA attends it (else no unit is in it).
    __device__ __forceinline__ int last_page() const { return whole > 0 ? (n - 1) >> whole << (whole - 5) : units; }
    __device__ __forceinline__ int segment() const {
        const int k = min(units - u, left);
        return whole > 0 && u + k > last_page() ? units - u : k;
    }
    __device__ __forceinline__ void advance(const DecodeArgs& a, const Lens& lens, int runs, int n_seg) {
        left -= n_seg + kRunCost;
        if (left <= 0) return;
        at += units + kRunCost;
        u = 0;
        if (++run < runs) return;
        run = 0;
        units = 0;
        while (units == 0 && ++s < a.kv.n_seq) {
            n = lens.at(a, s);
            units = units_of(n);
        }
        if (units == 0) left = 0;
    }
};
__device__ __forceinline__ int cost_of(int units) { return units > 0 ? units + kRunCost : 0; }

// This CTA's share of all runs' units (every warp on its own): lane i adds up
// a 32nd of the sequences, the lane whose part holds the start of the CTA's
// range looks for its sequence.
__device__ __forceinline__ Walk share_of(const DecodeArgs& a, const DecodeSplit& sp, const Lens& lens, int runs,
                                         int lane) {
    Walk w{};
    const int n_seq = a.kv.n_seq;
    if (n_seq == 1) {  // (the same without the search)
        w.n = lens.at(a, 0);
        w.units = units_of(w.n);
        const int32_t cost = cost_of(w.units), total = cost * runs;
        const int32_t per = max((int32_t)(((uint32_t)total + sp.ctas - 1) / (uint32_t)sp.ctas), kMinUnits);
        if (blockIdx.x == 0 && threadIdx.x == 0) *sp.per = per;
        w.per = per;
        const int64_t first = (int64_t)per * blockIdx.x;
        if (first >= total) return w;
        w.left = min(per, total - (int32_t)first);
        w.run = (int32_t)((uint32_t)first / (uint32_t)cost);
        const int32_t off = (int32_t)first - w.run * cost;
        w.at = (int32_t)first - off;
        w.u = max(0, off - kRunCost);
        w.left -= max(0, kRunCost - off);
        return w;
    }
    const int part = (n_seq + 31) / 32;
    const int s0 = min(n_seq, lane * part), s1 = min(n_seq, s0 + part);
    int32_t mine = 0;
    for (int s = s0; s < s1; ++s) mine += cost_of(units_of(lens.at(a, s)));
    mine *= runs;
    int32_t incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int32_t v = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += v;
    }
    const int32_t total = __shfl_sync(0xffffffffu, incl, 31);
    const int32_t per = max((int32_t)(((uint32_t)total + sp.ctas - 1) / (uint32_t)sp.ctas), kMinUnits);
    if (blockIdx.x == 0 && threadIdx.x == 0) *sp.per = per;
    if (total / per < (int)blockIdx.x) return w;  // (the product below stays under total)
    const int32_t first = per * blockIdx.x;
    w.per = per;
    if (first >= total) return w;
    w.left = min(per, total - first);
    const bool here = mine > 0 && first >= incl - mine && first < incl;
    if (here) {
        int32_t off = first - (incl - mine);
        w.s = s0;
        for (;; ++w.s) {
            w.n = lens.at(a, w.s);
            w.units = units_of(w.n);
            if (off < cost_of(w.units) * runs) break;
            off -= cost_of(w.units) * runs;
        }
        w.run = (int32_t)((uint32_t)off / (uint32_t)cost_of(w.units));
        off -= w.run * cost_of(w.units);
        // a run's cost comes before its units
        w.at = first - off;
        w.u = max(0, off - kRunCost);
        w.left -= max(0, kRunCost - off);
    }
    const int from = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
    w.s = __shfl_sync(0xffffffffu, w.s, from);
    w.n = __shfl_sync(0xffffffffu, w.n, from);
    w.units = __shfl_sync(0xffffffffu, w.units, from);
    w.run = __shfl_sync(0xffffffffu, w.run, from);
    w.u = __shfl_sync(0xffffffffu, w.u, from);
    w.at = __shfl_sync(0xffffffffu, w.at, from);
    w.left = __shfl_sync(0xffffffffu, w.left, from);
    return w;
}
// Joins what the CTAs of a cluster (or this one alone) have of a run: outputs
// [head][D], then (maximum, sum) [head], at the start of each one's shared
// memory; and adds the weights of this CTA's rows.  `lse_s`: [heads] of scratch.
template <int D, int kThreads, int kPass>
__device__ __forceinline__ void join_cluster(const DecodeArgs& a, const DecodeSplit& sp, const unsigned char* smem,
                                             float* lse_s, const Walk& w, int n_seg, int64_t q_row, int n_heads, int h,
                                             int rank) {
    const int C = sp.cluster, lane = threadIdx.x & 31;
    if (C > 1) tc::cluster_sync();
    else tc::named_bar_sync(1, kThreads);
    // weight of each CTA's part of head g, and log2 of the sum over all
    auto weigh = [&](int g, float (&f)[kMaxCluster]) {
        float2 v[kMaxCluster];
        float m = -INFINITY, l = 0.f;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k)
            if (k < C) {
                asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                             : "=f"(v[k].x), "=f"(v[k].y)
                             : "r"(tc::peer_of(smem + kPass * D * 4 + g * 8, k))
                             : "memory");
            } else {
                v[k] = make_float2(0.f, 0.f);
            }
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k)
            if (v[k].y != 0.f) m = fmaxf(m, v[k].x);
        const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) {
            f[k] = v[k].y != 0.f ? ex2(v[k].x - ms) : 0.f;  // 0: nothing but -inf there, its sums may be anything
            l += v[k].y * f[k];
        }
        const float inv = 1.f / l;
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k) f[k] *= inv;
        return ms + log2f(l);
    };
    float f[kMaxCluster];
    for (int j = rank * kThreads + threadIdx.x; j < n_heads * (D / 4); j += C * kThreads) {
        const int g = j / (D / 4), c = j % (D / 4);
        float4 t[kMaxCluster];
#pragma unroll
        for (int k = 0; k < kMaxCluster; ++k)
            if (k < C)
                asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                             : "=f"(t[k].x), "=f"(t[k].y), "=f"(t[k].z), "=f"(t[k].w)
                             : "r"(tc::peer_of(smem + (g * D + c * 4) * 4, k))
                             : "memory");
        const float lse = weigh(g, f);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        if (w.n > 0) {
#pragma unroll
            for (int k = 0; k < kMaxCluster; ++k)
                if (k < C && f[k] != 0.f) o.x += f[k] * t[k].x, o.y += f[k] * t[k].y, o.z += f[k] * t[k].z, o.w += f[k] * t[k].w;
        }
        store4(a.out, a.out_dtype, (q_row + g) * D + c * 4, o);
        if (c == 0 && a.acc != nullptr && !sp.fused) sp.lse[q_row + g] = lse;
    }
    if (!sp.fused) return;
    for (int g = threadIdx.x; g < n_heads; g += kThreads) lse_s[g] = weigh(g, f);
    tc::named_bar_sync(1, kThreads);
    float* acc = a.acc + ((int64_t)w.s * a.n_head_kv + h) * a.acc_stride;
    for (int r = w.u * kUnit + threadIdx.x; r < (w.u + n_seg) * kUnit; r += kThreads) {
        const float* sc = sp.scores + q_row * sp.score_stride + r;
        const float was = r < w.n ? acc[r] : 0.f;
        float sum = 0.f;
#pragma unroll 8
        for (int g = 0; g < n_heads; ++g) sum += ex2(sc[(int64_t)g * sp.score_stride] - lse_s[g]);
        if (r < w.n) acc[r] = was + sum;
        __syncwarp();
        for (int g = lane; g < n_heads; g += 32)
            asm volatile("discard.global.L2 [%0], 128;" ::"l"(sc - lane + (int64_t)g * sp.score_stride) : "memory");
    }
}
// CTAs that share run `at` of sequence s, and each one's slot.
struct Shares {
    int32_t per, start, c0, count;
    __device__ __forceinline__ int slot(int i) const {
        const int c = c0 + i;
        return 2 * c + (i == 0 && start > c * per ? 1 : 0);
    }
};
// (Lengths that change under the call give wrong shares, never ones outside
// the CTAs.)
__device__ __forceinline__ Shares shares_of(const DecodeSplit& sp, int32_t per, int32_t start, int units) {
    const int u0 = start + kRunCost, c0 = min(max(u0 / per, 0), sp.ctas - 1);  // the first unit comes after the run's cost
    return {per, start, c0, max(min((u0 + units - 1) / per, sp.ctas - 1) - c0, 0) + 1};
}

// Maximum and sum of one head over its shares (a warp; the same in every lane).
__device__ __forceinline__ float2 join_ml(const DecodeSplit& sp, const Shares& sh, int stride, int g, int lane) {
    float m = -INFINITY, l = 0.f;
    for (int i = lane; i < sh.count; i += 32) {
        const float2 v = sp.part_ml[(int64_t)sh.slot(i) * stride + g];
        if (v.y != 0.f) m = fmaxf(m, v.x);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
    const float ms = m == -INFINITY ? 0.f : m;
    for (int i = lane; i < sh.count; i += 32) {
        const float2 v = sp.part_ml[(int64_t)sh.slot(i) * stride + g];
        if (v.y != 0.f) l += v.y * ex2(v.x - ms);
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
    return make_float2(ms, l);
}

__global__ void k6_lengths(const DecodeArgs a, int32_t* lens) {
    tc::pdl_wait();
    tc::pdl_launch();
    const int s = blockIdx.x * blockDim.x + threadIdx.x;
    if (s < a.kv.n_seq) lens[s] = batch_len(a.kv, s, a.err);
}

constexpr int kJoinThreads = 256;
constexpr int kJoinRows = 4 * kJoinThreads;  // cache rows per weights CTA
constexpr int kJoinHeads = 8;    // query heads whose scores a thread holds at a time

// The first joins * heads CTAs put together the outputs of the runs that several
// CTAs shared (one CTA per query head of a run; at most one such run begins in
// a CTA of k6a); the others, [n_seq][Hkv][chunks], add the weights of kJoinRows
// rows of one KV head.  Latency bounds it (lengths, then ranges, then sums, then
// weights), so registers are held to four CTAs per SM.  NAN_NONE: a head whose
// scores are all -inf gets NaN, as the quotient 0 / 0 of a run in one CTA gives.
template <int D, bool NAN_NONE>
__global__ void __launch_bounds__(kJoinThreads, 4) k6b_join(const DecodeArgs a, const DecodeSplit sp, int heads,
                                                         int chunks) {
    __shared__ float wgt[kCtas];
    __shared__ float part[kJoinThreads * 4];
    __shared__ float lse[128];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int G = a.n_head / a.n_head_kv, runs = a.n_head_kv * sp.passes, stride = sp.groups * sp.heads;
    const int joins = sp.joins * heads;
    tc::pdl_wait();
    tc::pdl_launch();
    if ((int)blockIdx.x < joins) {
        const int4 cut = sp.cut[blockIdx.x / heads];
        const int32_t per = *sp.per;
        if (cut.x < 0 || cut.x >= a.kv.n_seq || cut.y < 0 || cut.y >= runs) return;
        const int gi = blockIdx.x % heads, h = cut.y / sp.passes, g = cut.y % sp.passes * sp.pass_heads + gi;
        if (g >= G) return;
        const int64_t out = ((int64_t)cut.x * a.n_head + h * G + g) * D;
        const Shares sh = shares_of(sp, per, cut.z, cut.w);
        constexpr int kLanes = D / 4, kRows = kJoinThreads / kLanes, kHeld = 4;
        const int c = threadIdx.x % kLanes, r = threadIdx.x / kLanes;
        auto part_of = [&](int i) {
            return *reinterpret_cast<const float4*>(sp.part_o + ((int64_t)sh.slot(i) * stride + gi) * D + c * 4);
        };
        // the first few shares' outputs are on their way while the weights are made
        float4 held[kHeld];
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
            if (r + k * kRows < sh.count) held[k] = part_of(r + k * kRows);
        if (warp == 0) {
            const float2 v = join_ml(sp, sh, stride, gi, lane);
            for (int i = lane; i < sh.count; i += 32) {
                const float2 p = sp.part_ml[(int64_t)sh.slot(i) * stride + gi];
                wgt[i] = p.y != 0.f ? ex2(p.x - v.x) / v.y : NAN_NONE && v.y == 0.f ? __int_as_float(0x7fffffff) : 0.f;
            }
        }
        __syncthreads();
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        auto add = [&](int i, const float4& t) {
            const float f = wgt[i];
            if (f == 0.f) return;  // nothing but -inf there: its sums may be anything
            o.x += f * t.x, o.y += f * t.y, o.z += f * t.z, o.w += f * t.w;
        };
#pragma unroll
        for (int k = 0; k < kHeld; ++k)
            if (r + k * kRows < sh.count) add(r + k * kRows, held[k]);
        for (int i = r + kHeld * kRows; i < sh.count; i += kRows) add(i, part_of(i));
        reinterpret_cast<float4*>(part)[threadIdx.x] = o;
        __syncthreads();
        if (r == 0) {
            for (int i = 1; i < kRows; ++i) {
                const float4 t = reinterpret_cast<float4*>(part)[i * kLanes + c];
                o.x += t.x, o.y += t.y, o.z += t.z, o.w += t.w;
            }
            store4(a.out, a.out_dtype, out + c * 4, o);
        }
        return;
    }
    const int id = blockIdx.x - joins, s = id / chunks / a.n_head_kv;
    const int h = id / chunks % a.n_head_kv, j0 = (id % chunks) * kJoinRows;
    // the first heads' scores are on their way while the sums are put together
    // (rows past the length are read where there are any, and not used)
    const int r0 = j0 + 4 * threadIdx.x;
    const float* sc = sp.scores + ((int64_t)s * a.n_head + (int64_t)h * G) * sp.score_stride +
                      min(r0, sp.score_stride - 4);
    float4 x[kJoinHeads];
    auto fetch = [&](int g0) {
#pragma unroll
        for (int g = 0; g < kJoinHeads; ++g)
            if (g0 + g < G) x[g] = *reinterpret_cast<const float4*>(sc + (int64_t)(g0 + g) * sp.score_stride);
    };
    fetch(0);
    const int n = batch_len(a.kv, s, a.err), units = units_of(n);
    if (j0 >= n) return;
    const int32_t per = sp.direct ? 1 : *sp.per;
    for (int g = warp; g < G; g += kJoinThreads / 32) {
        const int pass = g / sp.pass_heads;
        const Shares sh = sp.direct ? Shares{1, 0, 0, 1}
                                    : shares_of(sp, per, sp.run_start[(int64_t)s * runs + h * sp.passes + pass], units);
        float v;
        if (sh.count == 1) {
            v = sp.lse[(int64_t)s * a.n_head + h * G + g];
        } else {
            const float2 t = join_ml(sp, sh, stride, g % sp.pass_heads, lane);
            v = t.x + log2f(t.y);
        }
        if (lane == 0) lse[g] = v;
    }
    float* acc = a.acc + ((int64_t)s * a.n_head_kv + h) * a.acc_stride;
    acc += r0;
    const bool quad = r0 + 4 <= n && (reinterpret_cast<uintptr_t>(acc) & 15) == 0;
    float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
    if (quad) {
        w = *reinterpret_cast<const float4*>(acc);
    } else {
        if (r0 < n) w.x = acc[0];
        if (r0 + 1 < n) w.y = acc[1];
        if (r0 + 2 < n) w.z = acc[2];
        if (r0 + 3 < n) w.w = acc[3];
    }
    __syncthreads();
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int g0 = 0;;) {
#pragma unroll
        for (int g = 0; g < kJoinHeads; ++g)
            if (g0 + g < G) {
                const float z = lse[g0 + g];
                sum.x += ex2(x[g].x - z), sum.y += ex2(x[g].y - z);
                sum.z += ex2(x[g].z - z), sum.w += ex2(x[g].w - z);
            }
        // the warp has all it wants of these lines: they need not go to memory
        __syncwarp();
        if (lane % 8 == 0 && r0 < sp.score_stride)
            for (int g = 0; g < kJoinHeads && g0 + g < G; ++g)
                asm volatile("discard.global.L2 [%0], 128;" ::"l"(sc + (int64_t)(g0 + g) * sp.score_stride) : "memory");
        g0 += kJoinHeads;
        if (g0 >= G) break;
        fetch(g0);
    }
    w.x += sum.x, w.y += sum.y, w.z += sum.z, w.w += sum.w;
    if (quad) {
        *reinterpret_cast<float4*>(acc) = w;
    } else {
        if (r0 < n) acc[0] = w.x;
        if (r0 + 1 < n) acc[1] = w.y;
        if (r0 + 2 < n) acc[2] = w.z;
        if (r0 + 3 < n) acc[3] = w.w;
    }
}
PFN_cuTensorMapEncodeTiled_v12000 get_encode() {
    static std::atomic<PFN_cuTensorMapEncodeTiled_v12000> fn{nullptr};
    PFN_cuTensorMapEncodeTiled_v12000 f = fn.load(std::memory_order_acquire);
    if (!f) {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            f = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
        fn.store(f, std::memory_order_release);
    }
    return f;
}
size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

}  // namespace
}  // namespace epsp
