// k_decode.cu -- K6: attention of one new token per sequence over its cache.
//
//   x_j = q . k_j * scale,  out = sum_j exp(x_j - m) v_j / sum_j exp(x_j - m)
//
// over the rows j < lens[s] of each (sequence, KV head), for the G query heads
// of the group at once.  Every cache byte is used G times only, so the bytes
// bound it: what matters is that all SMs stream all the time.
//
// Split.  A run is one (sequence, KV head, pass over its query heads, 8 per warp); its
// rows are cut into units of 32.  All runs' units, laid end to end, are dealt
// to the CTAs in equal contiguous ranges (computed on the device from the
// lengths), so ragged batches and one long sequence load the SMs alike.  A run
// inside one CTA is finished there; one that several CTAs share leaves its
// running (maximum, sum, output) in the workspace, two slots per CTA, and
// k6b_join puts them together in a fixed order.  Calls of few short runs give
// each a cluster of CTAs, which join in shared memory: one launch.
//
// CTA: one warp streams K and V units into a ring by TMA (128-byte swizzled
// rows); units go round robin to the streams of the 8 other warps (4 for f32 rows of 512 bytes), each warp with its
// own online softmax over 8 query heads (groups of more than 8 heads give a
// unit to 2, 4 or 8 warps).  No barrier is shared until a run's end, where the
// warps' states are merged in shared memory.
//
// 16-bit: S = Q K^T and O = P V on mma.sync m16n8k16 with 8 heads in rows 0-7.
// The tensor work is 1/8 of what the pipe could do in the time a unit's bytes
// take, and the fragments come straight from the ring by ldmatrix; tcgen05
// would want 128 rows where there are 8.  Rows 8-15 of the P operand carry
// P - round16(P), so P keeps 16 bits of mantissa (bf16; 22 in f16) at no extra
// MMA; f32 outputs of bf16 caches add a third part.  f16 has few exponents: P
// is 2^7 times the weight against the running maximum there (2^15 at most), and
// the remainder, summed in accumulators of its own, 2^12 times itself.  A
// weight keeps 2^-16 of itself down to 2^-28 of the largest, and an absolute
// step of 2^-44 of it below.
// f32: FMA on the CUDA cores, one key per lane for S, 4 (or 2) columns per
// lane for O.
//
// Weights: the scores are kept in the workspace (4 bytes per query head and
// row against the 4 d / G of K and V) and k6b_join adds exp(x - lse).  They are
// written with evict_last, so that the cache streaming past leaves them in L2,
// and given up there once read, so that they never go out to memory (8 x 16-32 K
// rows, 28 heads, 22 MB of scores: 95.5 us without either, 90 with the first, 85
// with both).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdint>

#include "decode_common.cuh"
#include "epsp_kernels.h"
#include "tc100.cuh"

namespace epsp {
namespace {

constexpr int kChunk = kUnit * 128;  // one 128-byte column block of a unit

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

// ET 0 f32, 1 f16, 2 bf16; W consumer warps (and a producer).
// HW query heads per warp.
template <int ET, int D, int W, int HW>
struct Layout {
    static constexpr int kEs = ET == 0 ? 4 : 2;
    static constexpr int kCols = D * kEs / 128;          // 128-byte column blocks of a row
    static constexpr int kHalf = kCols * kChunk;         // K (or V) of a unit
    static constexpr int kStage = 2 * kHalf;
    // A stage always falls to the same stream of warps (kStages is a multiple
    // of the streams; f32 rows of 512 bytes have 4 stages and at most 4
    // streams, of two warps or more): a warp that found its stage full knows that the stage's earlier
    // fill had landed, which the barrier's one phase bit cannot tell it.
    static constexpr int kWarps = W;
    static constexpr int kStages = (W == 4 && ET != 0 ? 196608 : 131072) / kStage;
    static constexpr int kPass = W == 4 ? 16 : W * (ET == 0 ? 4 : 8);  // query heads of a pass, at most
    static constexpr int kOffQ = kStages * kStage;       // [2][kPass][D] queries of a segment
    static constexpr int kQBytes = kPass * D * kEs;
    static constexpr int kOffO = kOffQ + 2 * kQBytes;    // [kWarps][HW][D] merge buffer
    static constexpr int kOffP = kOffO + kWarps * HW * D * 4;  // f32: [kWarps][32 keys][HW]
    static constexpr int kOffMl = kOffP + (ET == 0 ? kWarps * kUnit * HW * 4 : 0);
    static constexpr int kOffBar = kOffMl + 2 * kWarps * HW * 8;
    static constexpr int kOffLens = kOffBar + (2 * kStages + 4) * 8;
    static constexpr int kBytes = kOffLens + kLensOnChip * 4;
    static_assert((kStages % kWarps == 0 || (ET == 0 && D == 128 && kStages == 4)) && kBytes + 1024 <= 232448, "shared memory");
};

// The weights of one key for a warp's heads (f32).
template <int GH>
struct PVec {
    using type = float4;
};
template <>
struct PVec<2> {
    using type = float2;
};
template <>
struct PVec<1> {
    using type = float;
};

// Overwrites what TMA brought of a sequence's last rows [from, 32) of a unit:
// row `fresh` (>= 0) from the new token's K and V, V rows from `lim` on with
// zeros (their P is 0, and 0 * NaN is not 0).
template <int ET, int D>
__device__ __forceinline__ void patch_unit(unsigned char* stage, int lane, int lim, int fresh, const char* kn,
                                           const char* vn) {
    using LY = Layout<ET, D, 8, 1>;
    constexpr int nc = LY::kCols * 8;  // 16-byte chunks per row
    auto at = [&](unsigned char* base, int r, int c) {
        return reinterpret_cast<uint4*>(base + (c >> 3) * kChunk + r * 128 + (((c & 7) ^ (r & 7)) << 4));
    };
    if (fresh >= 0)
        for (int i = lane; i < 2 * nc; i += 32) {
            const int c = i % nc;
            *at(stage + (i < nc ? 0 : LY::kHalf), fresh, c) = *reinterpret_cast<const uint4*>((i < nc ? kn : vn) + c * 16);
        }
    for (int i = lane; i < (kUnit - lim) * nc; i += 32)
        *at(stage + LY::kHalf, lim + i / nc, i % nc) = make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // TMA writes the stage next
    __syncwarp();
}
// JOIN: the calls that join_cluster finishes (kept apart: 64 runs of up to
// 4096 rows, 90 us without its code and 92 with it).
template <int ET, int D, int W, bool P3, int GH, bool JOIN>
__global__ void __launch_bounds__((W + 1) * 32, 1)
    k6a_decode(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const DecodeArgs a,
               const DecodeSplit sp) {
    constexpr int kHeads = ET == 0 ? GH : 8;  // query heads per warp
    using LY = Layout<ET, D, W, kHeads>;
    constexpr bool BF16 = ET == 2;
    constexpr float kUp = ET == 1 ? 7.f : 0.f;         // the maximum is kept this much lower, in log2 units
    constexpr float kLow = ET == 1 ? 4096.f : 1.f;     // factor of P's remainder
    constexpr int kWarps = LY::kWarps, kThreads = (W + 1) * 32, kPass = LY::kPass;
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + LY::kOffBar);
    uint64_t* empty = full + LY::kStages;
    uint64_t* q_full = empty + LY::kStages;
    uint64_t* q_empty = q_full + 2;
    int32_t* lens_s = reinterpret_cast<int32_t*>(smem + LY::kOffLens);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int Hkv = a.n_head_kv, G = a.n_head / Hkv;
    const int runs = Hkv * sp.passes;

    if (threadIdx.x == 0) {
        for (int i = 0; i < LY::kStages; ++i) {
            tc::mbar_init(&full[i], 1);
            tc::mbar_init(&empty[i], sp.groups);
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&q_full[i], 1);
            tc::mbar_init(&q_empty[i], kWarps);
        }
        tc::fence_mbar_init();
        tc::tma_prefetch_desc(&tmK);
        tc::tma_prefetch_desc(&tmV);
    }
    tc::pdl_wait();
    tc::pdl_launch();

    // ----------------------------------------- this CTA's range of the units
    Walk w0{};
    Lens lens{nullptr};
    const int C = JOIN ? sp.cluster : 1, rank = blockIdx.x & (C - 1);
    if (JOIN || sp.direct) {
        const int id = blockIdx.x >> (__ffs(C) - 1);
        w0.s = id / runs;
        w0.run = id % runs;
        if (threadIdx.x == 0) lens_s[0] = batch_len(a.kv, w0.s, a.err);
        __syncthreads();
        w0.n = lens_s[0];
        w0.units = units_of(w0.n);
        const int per = (w0.units + C - 1) >> (__ffs(C) - 1);
        w0.u = min(rank * per, w0.units);
        w0.left = min(per, w0.units - w0.u);
    } else {
        if (a.kv.n_seq <= kLensOnChip) {
            for (int s = threadIdx.x; s < a.kv.n_seq; s += kThreads) lens_s[s] = batch_len(a.kv, s, a.err);
            lens.chip = lens_s;
        }
        __syncthreads();
        w0 = share_of(a, sp, lens, runs, lane);
        // sequences without rows, dealt out to the CTAs
        for (int s = blockIdx.x; s < a.kv.n_seq; s += gridDim.x)
            if (lens.at(a, s) == 0) {
                for (int i = threadIdx.x; i < a.n_head * (D / 4); i += kThreads)
                    store4(a.out, a.out_dtype, (int64_t)s * a.n_head * D + i * 4, make_float4(0.f, 0.f, 0.f, 0.f));
                if (sp.by_run)
                    for (int i = threadIdx.x; i < runs; i += kThreads) sp.cut[s * runs + i] = make_int4(-1, 0, 0, 0);
            }
        if (w0.left <= 0 && !sp.by_run && threadIdx.x == 0) sp.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
    }
    // (a cluster's CTAs meet whatever their lengths)
    if (w0.left <= 0 && C == 1) {
        if (sp.direct) {  // a sequence without rows
            const int g0 = (w0.run % sp.passes) * kPass, n = min(kPass, G - g0) * (D / 4);
            const int64_t at = ((int64_t)w0.s * a.n_head + (w0.run / sp.passes) * G + g0) * D;
            for (int i = threadIdx.x; i < n; i += kThreads)
                store4(a.out, a.out_dtype, at + i * 4, make_float4(0.f, 0.f, 0.f, 0.f));
        }
        return;
    }
    const uint64_t tmo = a.timeout_ns;

    if (warp == kWarps) {
        // ------------------------------------------------------- producer --
        // 32 units' rows at a time (one table entry per lane), lane 0 issues.
        Walk w = w0;
        int it = 0;
        bool ok = true;
        int seg = 0;
        const uint64_t policy = tc::policy_evict_first();  // the cache is read once
        for (; (w.left > 0 || (C > 1 && seg == 0)) && ok; ++seg) {
            const int n_seg = w.segment();
            const int h = w.run / sp.passes, pass = w.run % sp.passes;
            if (lane == 0) {
                const int b = seg & 1;
                ok = tc::mbar_wait(&q_empty[b], ((seg >> 1) & 1) ^ 1, tmo);
                if (ok) {
                    const uint32_t bytes = min(kPass, G - pass * kPass) * D * LY::kEs;
                    tc::mbar_arrive_expect_tx(&q_full[b], bytes);
                    tc::bulk_load(smem + LY::kOffQ + b * LY::kQBytes,
                                  static_cast<const char*>(a.q) +
                                      ((int64_t)w.s * a.n_head + (int64_t)h * G + pass * kPass) * D * LY::kEs,
                                  bytes, &q_full[b]);
                }
            }
            ok = __shfl_sync(0xffffffffu, ok, 0);
            if (!ok) break;
            for (int i0 = 0; i0 < n_seg && ok; i0 += 32) {
                int row = a.kv.rows;  // past the end: zeros
                if (i0 + lane < n_seg) {
                    const int r = batch_row(a.kv, w.s, (w.u + i0 + lane) * kUnit, a.err);
                    if (r >= 0) row = r;
                }
                const int cnt = min(32, n_seg - i0);
                for (int i = 0; i < cnt; ++i, ++it) {
                    const int st = it % LY::kStages;
                    const int r = __shfl_sync(0xffffffffu, row, i);
                    if (lane == 0) {
                        ok = tc::mbar_wait(&empty[st], ((it / LY::kStages) & 1) ^ 1, tmo);
                        if (ok) {
                            tc::mbar_arrive_expect_tx(&full[st], LY::kStage);
                            unsigned char* base = smem + st * LY::kStage;
#pragma unroll
                            for (int c = 0; c < LY::kCols; ++c)
                                tc::tma_load_3d(base + c * kChunk, &tmK, &full[st], c * (128 / LY::kEs), h, r, policy);
#pragma unroll
                            for (int c = 0; c < LY::kCols; ++c)
                                tc::tma_load_3d(base + LY::kHalf + c * kChunk, &tmV, &full[st], c * (128 / LY::kEs), h,
                                                r, policy);
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                    if (!ok) break;
                }
            }
            w.advance(a, lens, runs, n_seg);
        }
        if (!ok) {
            if (lane == 0) report_error(a.err, kDevWaitDecode, 0xa1, it);
            // copies still in flight land before the CTA ends
            for (int j = max(0, it - LY::kStages); j < it; ++j)
                tc::mbar_wait(&full[j % LY::kStages], (j / LY::kStages) & 1, tmo);
            for (int j = max(0, seg - 1); j <= seg; ++j) tc::mbar_wait(&q_full[j & 1], (j >> 1) & 1, tmo);
        }
        return;
    }

    // ---------------------------------------------------------- consumers --
    const int groups = sp.groups, streams = kWarps / groups;
    const int grp = warp & (groups - 1), stream = warp / groups;
    const float sl2 = a.kq_scale * kLog2e;
    const uint64_t keep = tc::policy_evict_last();  // scores: read once more, by k6b_join
    float* om = reinterpret_cast<float*>(smem + LY::kOffO);
    float* om_w = om + warp * kHeads * D;
    float* ps = reinterpret_cast<float*>(smem + LY::kOffP) + warp * kUnit * kHeads;
    Walk w = w0;
    int it = 0;
    bool ok = true;
    for (int seg = 0; w.left > 0 || (C > 1 && seg == 0); ++seg) {
        const int n_seg = w.segment();
        const int h = w.run / sp.passes, pass = w.run % sp.passes;
        const int g0 = pass * kPass + grp * kHeads;  // this warp's first query head of the group
        const int64_t q_row = (int64_t)w.s * a.n_head + (int64_t)h * G;
        // state: 16-bit o[2 columns x 8 heads in MMA fragments], f32 o[head][columns]
        constexpr int NO = ET == 0 ? GH * (D / 32) : D / 2;
        float o[NO];
#pragma unroll
        for (int i = 0; i < NO; ++i) o[i] = 0.f;
        constexpr int NM = ET == 0 ? GH : 1;
        float m[NM], l[NM];
#pragma unroll
        for (int i = 0; i < NM; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.f;
        }
        uint32_t qf[ET == 0 ? 1 : D / 8];
        const int hd = lane >> 2, qc = (lane & 3) * 2;  // 16-bit: head and columns of this lane's fragments
        const unsigned char* qs = smem + LY::kOffQ + (seg & 1) * LY::kQBytes + grp * kHeads * D * LY::kEs;
        if (ok) {
            ok = __all_sync(0xffffffffu, tc::mbar_wait(&q_full[seg & 1], (seg >> 1) & 1, tmo));
            if (!ok && lane == 0) report_error(a.err, kDevWaitDecode, 0xa3, seg);
        }
        if constexpr (ET != 0) {
#pragma unroll
            for (int i = 0; i < D / 8; ++i)
                qf[i] = g0 + hd < G ? *reinterpret_cast<const uint32_t*>(qs + (hd * D + qc + i * 8) * 2) : 0u;
        }
        // first unit of the segment that falls to this stream
        int i = (stream - it) & (streams - 1);
        for (; i < n_seg; i += streams) {
            const int at = it + i, st = at % LY::kStages;
            if (ok) {
                ok = tc::mbar_wait(&full[st], (at / LY::kStages) & 1, tmo);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok && lane == 0) report_error(a.err, kDevWaitDecode, 0xa2, at);
            }
            if (!ok) break;
            unsigned char* stage = smem + st * LY::kStage;
            const int u = w.u + i, lim = min(kUnit, w.n - u * kUnit);
            if (u == w.units - 1) {
                const bool fresh = a.k_new != nullptr;
                // (held_back's word: asked for here, ahead of the new rows, it costs nothing; where it is wanted 1.5 us of 90)
                const int32_t held = fresh && a.kv.block_rows > 0 ? a.err[kErrRefused] : 0;
                const int64_t nr = ((int64_t)w.s * Hkv + h) * D * LY::kEs;
                const char* kn = static_cast<const char*>(a.k_new) + nr;
                const char* vn = static_cast<const char*>(a.v_new) + nr;
                if (fresh || lim < kUnit) patch_unit<ET, D>(stage, lane, lim, fresh ? lim - 1 : -1, kn, vn);
                if (fresh && grp == 0 && pass == 0) {
                    const int row = batch_row(a.kv, w.s, w.n - 1, a.err);
                    constexpr int nc = D * LY::kEs / 16;
                    if (row >= 0 && held == 0)
                        for (int c = lane; c < 2 * nc; c += 32) {
                            const int64_t to = ((int64_t)row * Hkv + h) * D * LY::kEs + (c % nc) * 16;
                            *reinterpret_cast<uint4*>(static_cast<char*>(c < nc ? a.k : a.v) + to) =
                                *reinterpret_cast<const uint4*>((c < nc ? kn : vn) + (c % nc) * 16);
                        }
                }
            }
            if constexpr (ET != 0) {
                const uint32_t kb = tc::smem_u32(stage), vb = kb + LY::kHalf;
                float s4[4][4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    s4[t][0] = s4[t][1] = s4[t][2] = s4[t][3] = 0.f;
                    const int r = t * 8 + (lane & 7);
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {  // 32 columns (4 chunks) a time
                        const int ch = (c & 1) * 4 + (lane >> 3);
                        uint32_t b[4];
                        ldsm4(b, kb + (c >> 1) * kChunk + r * 128 + ((ch ^ (r & 7)) << 4));
                        mma16816<BF16>(s4[t], qf[4 * c], 0, qf[4 * c + 1], 0, b[0], b[1]);
                        mma16816<BF16>(s4[t], qf[4 * c + 2], 0, qf[4 * c + 3], 0, b[2], b[3]);
                    }
                }
                float mx = -INFINITY;
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        s4[t][e] = t * 8 + qc + e < lim ? s4[t][e] * sl2 : -INFINITY;
                        mx = fmaxf(mx, s4[t][e]);
                    }
                if (a.acc != nullptr && g0 + hd < G) {
                    float* sc = sp.scores + (q_row + g0 + hd) * sp.score_stride + u * kUnit + qc;
#pragma unroll
                    for (int t = 0; t < 4; ++t)
                        asm volatile("st.global.L2::cache_hint.v2.f32 [%0], {%1, %2}, %3;" ::"l"(sc + t * 8),
                                     "f"(s4[t][0]), "f"(s4[t][1]), "l"(keep)
                                     : "memory");
                }
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                // the running maximum follows when it is 2^8 behind: p stays below 2^8 (f16: 2^15)
                const bool need = mx > m[0] + (8.f + kUp);
                if (__any_sync(0xffffffffu, need)) {
                    const float alpha = need ? ex2(m[0] - (mx - kUp)) : 1.f;
                    if (need) m[0] = mx - kUp;
                    l[0] *= alpha;
#pragma unroll
                    for (int j = 0; j < NO; ++j) o[j] *= alpha;
                }
                const float ms = m[0] == -INFINITY ? 0.f : m[0];
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        s4[t][e] = ex2(s4[t][e] - ms);
                        l[0] += s4[t][e];
                    }
#pragma unroll
                for (int kb16 = 0; kb16 < 2; ++kb16) {
                    float* p0 = s4[2 * kb16];
                    float* p1 = s4[2 * kb16 + 1];
                    const uint32_t a0 = split2<BF16>(p0[0], p0[1]), a2 = split2<BF16>(p1[0], p1[1]);
                    if constexpr (kLow != 1.f) p0[0] *= kLow, p0[1] *= kLow, p1[0] *= kLow, p1[1] *= kLow;
                    const uint32_t a1 = split2<BF16>(p0[0], p0[1]), a3 = split2<BF16>(p1[0], p1[1]);
                    uint32_t t0 = 0, t2 = 0;
                    if constexpr (P3) {
                        t0 = split2<BF16>(p0[0], p0[1]);
                        t2 = split2<BF16>(p1[0], p1[1]);
                    }
                    const int r = kb16 * 16 + (lane & 7) + ((lane >> 3) & 1) * 8;
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {  // 16 columns (2 chunks) a time
                        const int ch = (c & 3) * 2 + (lane >> 4);
                        uint32_t b[4];
                        ldsm4_t(b, vb + (c >> 2) * kChunk + r * 128 + ((ch ^ (r & 7)) << 4));
                        float(&o0)[4] = *reinterpret_cast<float(*)[4]>(&o[8 * c]);
                        float(&o1)[4] = *reinterpret_cast<float(*)[4]>(&o[8 * c + 4]);
                        mma16816<BF16>(o0, a0, a1, a2, a3, b[0], b[1]);
                        mma16816<BF16>(o1, a0, a1, a2, a3, b[2], b[3]);
                        if constexpr (P3) {  // (P again in rows 0-7: a zero or a third part there would spoil an infinite V)
                            mma16816<BF16>(o0, a0, t0, a2, t2, b[0], b[1]);
                            mma16816<BF16>(o1, a0, t0, a2, t2, b[2], b[3]);
                        }
                    }
                }
            } else {
                // S: one key per lane
                alignas(16) float x[GH];
#pragma unroll
                for (int g = 0; g < GH; ++g) x[g] = 0.f;
                const float4* q4 = reinterpret_cast<const float4*>(qs);  // (heads past the group: any values, not used)
#pragma unroll 4
                for (int c = 0; c < D / 4; ++c) {
                    const float4 kk = *reinterpret_cast<const float4*>(stage + (c >> 3) * kChunk + lane * 128 +
                                                                       (((c & 7) ^ (lane & 7)) << 4));
#pragma unroll
                    for (int g = 0; g < GH; ++g) {
                        const float4 qq = q4[g * (D / 4) + c];
                        x[g] = fmaf(qq.x, kk.x, x[g]);
                        x[g] = fmaf(qq.y, kk.y, x[g]);
                        x[g] = fmaf(qq.z, kk.z, x[g]);
                        x[g] = fmaf(qq.w, kk.w, x[g]);
                    }
                }
                bool need = false;
                float mx[GH];
#pragma unroll
                for (int g = 0; g < GH; ++g) {
                    x[g] = lane < lim ? x[g] * sl2 : -INFINITY;
                    if (a.acc != nullptr && g0 + g < G)
                        asm volatile("st.global.L2::cache_hint.f32 [%0], %1, %2;" ::"l"(
                                         sp.scores + (q_row + g0 + g) * sp.score_stride + u * kUnit + lane),
                                     "f"(x[g]), "l"(keep)
                                     : "memory");
                    mx[g] = x[g];
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) mx[g] = fmaxf(mx[g], __shfl_xor_sync(0xffffffffu, mx[g], d));
                    need |= mx[g] > m[g] + 8.f;
                }
                if (need) {
#pragma unroll
                    for (int g = 0; g < GH; ++g)
                        if (mx[g] > m[g]) {
                            const float alpha = ex2(m[g] - mx[g]);
                            m[g] = mx[g];
                            l[g] *= alpha;
#pragma unroll
                            for (int j = 0; j < D / 32; ++j) o[g * (D / 32) + j] *= alpha;
                        }
                }
#pragma unroll
                for (int g = 0; g < GH; ++g) {
                    x[g] = ex2(x[g] - (m[g] == -INFINITY ? 0.f : m[g]));
                    l[g] += x[g];
                }
                using Vec = typename PVec<GH>::type;
                reinterpret_cast<Vec*>(ps)[lane] = *reinterpret_cast<const Vec*>(x);
                __syncwarp();
                // O: D / 32 columns per lane, over the unit's keys
                constexpr int NC = D / 32;
                const int cb = lane * NC * 4;  // byte of the first column
                const unsigned char* vbase = stage + LY::kHalf + (cb >> 7) * kChunk;
                const int ch = (cb >> 4) & 7, in = cb & 15;
#pragma unroll 4
                for (int j = 0; j < lim; ++j) {
                    const unsigned char* vp = vbase + j * 128 + ((ch ^ (j & 7)) << 4) + in;
                    float vv[NC];
                    if constexpr (NC == 4) {
                        const float4 t = *reinterpret_cast<const float4*>(vp);
                        vv[0] = t.x, vv[1] = t.y, vv[2] = t.z, vv[3] = t.w;
                    } else {
                        const float2 t = *reinterpret_cast<const float2*>(vp);
                        vv[0] = t.x, vv[1] = t.y;
                    }
                    alignas(16) float p[GH];
                    *reinterpret_cast<Vec*>(p) = reinterpret_cast<const Vec*>(ps)[j];
#pragma unroll
                    for (int g = 0; g < GH; ++g)
#pragma unroll
                        for (int e = 0; e < NC; ++e) o[g * NC + e] = fmaf(p[g], vv[e], o[g * NC + e]);
                }
                __syncwarp();
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&empty[st]);
        }

        // ------------------------------------------- merge the warps' states
        // (ml alternates between two buffers: a warp may write the next
        // segment's before another has read this one's sums)
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&q_empty[seg & 1]);
        float2* ml = reinterpret_cast<float2*>(smem + LY::kOffMl) + (seg & 1) * kWarps * kHeads;
        if constexpr (ET != 0) {
            l[0] += __shfl_xor_sync(0xffffffffu, l[0], 1);
            l[0] += __shfl_xor_sync(0xffffffffu, l[0], 2);
            if ((lane & 3) == 0) ml[warp * kHeads + hd] = make_float2(m[0], l[0]);
        } else {
#pragma unroll
            for (int g = 0; g < GH; ++g) {
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) l[g] += __shfl_xor_sync(0xffffffffu, l[g], d);
                if (lane == 0) ml[warp * kHeads + g] = make_float2(m[g], l[g]);
            }
        }
        tc::named_bar_sync(1, kWarps * 32);
        // the streams' common maximum of a head of this warp's group
        auto top = [&](int g) {
            float mt = -INFINITY;
#pragma unroll
            for (int r = 0; r < kWarps; ++r)
                if (r < streams) mt = fmaxf(mt, ml[(r * groups + grp) * kHeads + g].x);
            return mt == -INFINITY ? 0.f : mt;
        };
        if constexpr (ET != 0) {
            // the sum over P and that over its remainders, which says nothing
            // where V is infinite: a remainder may be 0 or negative
            auto whole_sum = [](float hi, float lo) {
                if constexpr (P3) hi *= 0.5f;  // added twice
                return isinf(hi) ? hi : fmaf(lo, 1.f / kLow, hi);
            };
            const float f = ex2(m[0] - top(hd));
#pragma unroll
            for (int c = 0; c < D / 8; ++c)  // rows 8-15 hold the P remainders' part
                *reinterpret_cast<float2*>(om_w + hd * D + c * 8 + qc) =
                    make_float2(whole_sum(o[4 * c], o[4 * c + 2]) * f, whole_sum(o[4 * c + 1], o[4 * c + 3]) * f);
        } else {
            constexpr int NC = D / 32;
#pragma unroll
            for (int g = 0; g < GH; ++g) {
                const float f = ex2(m[g] - top(g));
#pragma unroll
                for (int e = 0; e < NC; ++e) om_w[g * D + lane * NC + e] = o[g * NC + e] * f;
            }
        }
        tc::named_bar_sync(1, kWarps * 32);
        const bool whole = w.u == 0 && n_seg == w.units;
        const int n_heads = min(min(groups * kHeads, kPass), G - pass * kPass);
        const int slot = blockIdx.x * 2 + (seg == 0 ? 0 : 1);
        for (int j = threadIdx.x; j < n_heads * (D / 4); j += kWarps * 32) {
            const int g = j / (D / 4), c = j % (D / 4), gw = g / kHeads, gh = g % kHeads;
            float2 v[kWarps];
            float4 t[kWarps];
            float mt = -INFINITY;
#pragma unroll
            for (int r = 0; r < kWarps; ++r)
                if (r < streams) {
                    const int wr = (r * groups + gw) * kHeads + gh;
                    v[r] = ml[wr];
                    t[r] = *reinterpret_cast<const float4*>(om + wr * D + c * 4);
                    mt = fmaxf(mt, v[r].x);
                }
            const float ms = mt == -INFINITY ? 0.f : mt;
            float lt = 0.f;
            float4 ot = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int r = 0; r < kWarps; ++r)
                if (r < streams) {
                    lt += v[r].y * ex2(v[r].x - ms);
                    ot.x += t[r].x, ot.y += t[r].y, ot.z += t[r].z, ot.w += t[r].w;
                }
            if constexpr (JOIN) {
                // (the ring: this CTA's last copy has landed)
                *reinterpret_cast<float4*>(smem + (g * D + c * 4) * 4) = ot;
                if (c == 0) *reinterpret_cast<float2*>(smem + kPass * D * 4 + g * 8) = make_float2(ms, lt);
            } else if (whole) {
                const float inv = 1.f / lt;
                store4(a.out, a.out_dtype, (q_row + pass * kPass + g) * D + c * 4,
                       make_float4(ot.x * inv, ot.y * inv, ot.z * inv, ot.w * inv));
                if (c == 0 && a.acc != nullptr) sp.lse[q_row + pass * kPass + g] = ms + log2f(lt);
            } else {
                const int64_t p = (int64_t)slot * groups * kHeads + g;
                *reinterpret_cast<float4*>(sp.part_o + p * D + c * 4) = ot;
                if (c == 0) sp.part_ml[p] = make_float2(ms, lt);
            }
        }
        if constexpr (JOIN) {
            join_cluster<D, kWarps * 32, kPass>(a, sp, smem, om, w, n_seg, q_row + pass * kPass, n_heads, h, rank);
            if (C > 1) tc::cluster_sync();  // nobody reads this CTA's part any more
        }
        if (!sp.direct && threadIdx.x == 0) {
            if (w.u == 0) sp.run_start[(int64_t)w.s * runs + w.run] = w.at;
            const int4 c =
                w.u == 0 && n_seg < w.units ? make_int4(w.s, w.run, w.at, w.units) : make_int4(-1, 0, 0, 0);
            if (!sp.by_run)
                sp.cut[blockIdx.x] = c;  // the CTA's last segment has the last word
            else if (w.u == 0)
                sp.cut[w.s * runs + w.run] = c;
        }
        it += n_seg;
        w.advance(a, lens, runs, n_seg);
    }
}
// ---------------------------------------------------------------- host side --
// Cache rows [rows][Hkv][d] in boxes of 32 rows x 128 bytes of one head.
bool cache_map(CUtensorMap* m, const void* base, int32_t dtype, int32_t d, int32_t n_head_kv, int32_t rows) {
    auto enc = get_encode();
    if (!enc) return false;
    const uint64_t es = dtype == 0 ? 4 : 2;
    const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)n_head_kv, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {d * es, d * es * n_head_kv};
    const cuuint32_t box[3] = {(cuuint32_t)(128 / es), 1, kUnit};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUtensorMapDataType t = dtype == 0   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : dtype == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                               : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    return enc(m, t, 3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
constexpr int kSmallGroup = 16;  // query heads per KV head up to which 4 warps do (16-bit)

// Split of a call and its workspace layout; returns the bytes (SIZE_MAX: more
// units than the 32-bit counts hold).
size_t split_of(int32_t n_seq, int32_t max_kv_len, int32_t n_head, int32_t n_head_kv, int32_t d, int32_t dtype,
                bool weights, char* ws, DecodeSplit* sp) {
    const int G = n_head / n_head_kv;
    if (dtype == 0) {
        // 4 heads per warp keep a unit's latency low; rows of 512 bytes want
        // two warps per unit at least (4 stages)
        sp->pass_heads = 32;
        const int least = d == 128 ? 2 : 1;
        sp->heads = G <= least ? 1 : G <= 2 * least ? 2 : 4;
        sp->groups = least;
    } else {
        sp->pass_heads = G <= kSmallGroup ? 16 : 64;
        sp->heads = 8;
        sp->groups = 1;
    }
    const int in_pass = G < sp->pass_heads ? G : sp->pass_heads;
    while (sp->groups * sp->heads < in_pass) sp->groups *= 2;
    sp->passes = (G + sp->pass_heads - 1) / sp->pass_heads;
    const int64_t all_runs = (int64_t)n_seq * n_head_kv * sp->passes;
    const int64_t units = units_of(max_kv_len), total = all_runs * (units + kRunCost);
    if (total > INT_MAX) return SIZE_MAX;
    sp->cluster = 1;
    sp->direct = all_runs <= kCtas && units <= kDirectUnits;
    if (!sp->direct) {
        while (sp->cluster < kMaxCluster && units > sp->cluster * kClusterUnits && all_runs * sp->cluster * 2 <= kClusterCtas)
            sp->cluster *= 2;
        sp->direct = sp->cluster > 1 && units <= sp->cluster * (weights ? 1 : 2) * kClusterUnits;
        if (!sp->direct) sp->cluster = 1;
    }
    sp->fused = sp->direct && weights && sp->passes == 1;  // (several passes would add to the same rows)
    const int64_t ctas = sp->direct ? all_runs * sp->cluster : (total + kMinUnits - 1) / kMinUnits;
    sp->ctas = (int32_t)(ctas < kCtas ? ctas : kCtas);
    sp->by_run = !sp->direct && all_runs <= sp->ctas;
    sp->joins = sp->direct ? 0 : sp->by_run ? (int32_t)all_runs : sp->ctas;
    sp->score_stride = (int32_t)(units * kUnit);
    size_t at = 16;
    auto take = [&](size_t bytes) {
        const size_t was = at;
        at += up16(bytes);
        return ws + was;
    };
    sp->per = reinterpret_cast<int32_t*>(ws);
    const int stride = sp->groups * sp->heads;
    if (!sp->direct) {
        sp->run_start = reinterpret_cast<int32_t*>(take(all_runs * sizeof(int32_t)));
        sp->cut = reinterpret_cast<int4*>(take(sp->joins * sizeof(int4)));
        if (n_seq > kLensOnChip) sp->lens = reinterpret_cast<int32_t*>(take(n_seq * sizeof(int32_t)));
        sp->part_ml = reinterpret_cast<float2*>(take((size_t)2 * sp->ctas * stride * sizeof(float2)));
        sp->part_o = reinterpret_cast<float*>(take((size_t)2 * sp->ctas * stride * d * sizeof(float)));
    }
    if (weights) {
        if (!sp->fused) sp->lse = reinterpret_cast<float*>(take((size_t)n_seq * n_head * sizeof(float)));
        // whole 128-byte lines, which k6b_join gives up
        const uintptr_t sc = reinterpret_cast<uintptr_t>(
            take((size_t)n_seq * n_head * sp->score_stride * sizeof(float) + 112));
        sp->scores = reinterpret_cast<float*>((sc + 127) & ~(uintptr_t)127);
    }
    return at;
}

template <int ET, int D, int W, bool P3, int GH, bool JOIN>
cudaError_t launch_join(DecodeArgs a, const DecodeSplit& sp, cudaStream_t s) {
    constexpr int kThreads = (W + 1) * 32;
    CUtensorMap mk, mv;
    if (!cache_map(&mk, a.k, a.dtype, D, a.n_head_kv, a.kv.rows) ||
        !cache_map(&mv, a.v, a.dtype, D, a.n_head_kv, a.kv.rows))
        return cudaErrorInvalidValue;
    const int smem = Layout<ET, D, W, ET == 0 ? GH : 8>::kBytes + 1024;
    int dev = 0;
    cudaGetDevice(&dev);
    // one bit per device ordinal < 32 whose attribute is set
    static std::atomic<unsigned> set_mask{0};
    if (dev >= 32 || !(set_mask.load(std::memory_order_acquire) & (1u << dev))) {
        const cudaError_t e = cudaFuncSetAttribute(k6a_decode<ET, D, W, P3, GH, JOIN>,
                                                   cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < 32) set_mask.fetch_or(1u << dev, std::memory_order_release);
    }
    // both kernels may start before what precedes them on the stream has
    // ended: they wait for it on the device
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = sp.cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cfg.stream = s;
    if (sp.lens) {
        cfg.gridDim = dim3((a.kv.n_seq + 255) / 256);
        cfg.blockDim = dim3(256);
        const cudaError_t e = cudaLaunchKernelEx(&cfg, k6_lengths, a, sp.lens);
        if (e != cudaSuccess) return e;
        a.kv.lens = sp.lens;
    }
    cfg.gridDim = dim3(sp.ctas);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.numAttrs = sp.cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, k6a_decode<ET, D, W, P3, GH, JOIN>, mk, mv, a, sp);
    if (e != cudaSuccess || (sp.direct && (!a.acc || sp.fused))) return e;
    const int chunks = a.acc ? (a.kv.max_kv_len + kJoinRows - 1) / kJoinRows : 0;
    const int heads = std::min(a.n_head / a.n_head_kv, sp.pass_heads);
    const int64_t grid = (int64_t)sp.joins * heads + (int64_t)a.kv.n_seq * a.n_head_kv * chunks;
    if (grid > INT_MAX) return cudaErrorInvalidValue;
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k6b_join<D, false>, a, sp, heads, chunks);
}

template <int ET, int D, int W, bool P3, int GH>
cudaError_t launch_t(const DecodeArgs& a, const DecodeSplit& sp, cudaStream_t s) {
    return sp.cluster > 1 || sp.fused ? launch_join<ET, D, W, P3, GH, true>(a, sp, s)
                                      : launch_join<ET, D, W, P3, GH, false>(a, sp, s);
}

template <int ET, int D, int W>
cudaError_t launch_w(const DecodeArgs& a, const DecodeSplit& sp, cudaStream_t s) {
    if constexpr (ET == 2) {
        if (a.out_dtype == 0) return launch_t<2, D, W, true, 8>(a, sp, s);
    }
    return launch_t<ET, D, W, false, 8>(a, sp, s);
}

template <int ET, int D>
cudaError_t launch_d(const DecodeArgs& a, const DecodeSplit& sp, cudaStream_t s) {
    const int G = a.n_head / a.n_head_kv;
    if constexpr (ET == 0) {
        if (sp.heads == 1) return launch_t<0, D, 8, false, 1>(a, sp, s);
        if (sp.heads == 2) return launch_t<0, D, 8, false, 2>(a, sp, s);
        return launch_t<0, D, 8, false, 4>(a, sp, s);
    } else {
        return G <= kSmallGroup ? launch_w<ET, D, 4>(a, sp, s) : launch_w<ET, D, 8>(a, sp, s);
    }
}

}  // namespace

size_t decode_ws_bytes(int32_t n_seq, int32_t max_kv_len, int32_t n_head, int32_t n_head_kv, int32_t head_dim,
                       int32_t dtype, bool weights) {
    DecodeSplit sp{};
    return split_of(n_seq, max_kv_len, n_head, n_head_kv, head_dim, dtype, weights, nullptr, &sp);
}

cudaError_t launch_decode(const DecodeArgs& a, cudaStream_t s) {
    DecodeSplit sp{};
    split_of(a.kv.n_seq, a.kv.max_kv_len, a.n_head, a.n_head_kv, a.head_dim, a.dtype, a.acc != nullptr,
             static_cast<char*>(a.ws), &sp);
    const bool wide = a.head_dim == 128;
    switch (a.dtype) {
        case 0: return wide ? launch_d<0, 128>(a, sp, s) : launch_d<0, 64>(a, sp, s);
        case 1: return wide ? launch_d<1, 128>(a, sp, s) : launch_d<1, 64>(a, sp, s);
        default: return wide ? launch_d<2, 128>(a, sp, s) : launch_d<2, 64>(a, sp, s);
    }
}

}  // namespace epsp
