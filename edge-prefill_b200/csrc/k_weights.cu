// k_weights.cu -- K7: softmax weights of a prompt's last rows over its cache.
//
//   acc[h][j] = sum over rows t and heads g of exp(x_tgj - lse_tg),  x = q . k * scale
//
// in two passes over the scores: the statistics pass leaves each query row's
// (maximum, sum) per key split, k7_join its lse, the sums pass each key's sum.
// Storing the scores instead would cost 8 bytes a pair; recomputing them costs
// 2 d flops, which the tensor cores do in a quarter of the time the pair's two
// exponentials take.  Those take most of both passes (16 MUFU results per clock
// and SM, a fifth of the pairs on the FMA pipe instead).  Every key has one
// writer (k7_add where the rows are split) and a fixed order of additions.
//
// 16-bit (tcgen05): a query tile packs T = 128 / G tokens x G heads into 128
// rows.  The two passes are one kernel with the MMA operands exchanged: with
// queries as the M side a thread (TMEM lane) owns a query row and reduces over
// keys; with keys as the M side it owns a key and reduces over queries.  Both
// reductions stay in the thread's registers, no shuffles.  One warp loads
// tiles by TMA, one issues MMAs into 3 S buffers in TMEM, and 24 warps take
// the exponentials.
// f32: the same passes on the CUDA cores, 64 x 64 tiles, 4 x 4 per thread; few
// scores are kept by the first pass instead, and the second only adds up their
// exponentials.
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdint>
#include <type_traits>

#include "epsp_kernels.h"
#include "tc100.cuh"

namespace epsp {
namespace {

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3f(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}

// acc + 2^x of a pair on the FMA pipe.  x >= -126.5 (below: 0, as ex2 has it;
// the exponent's bits come out 0 at -127; NaN stays) is split into n + r,
// n = round(x), r in [-0.5, 0.5]: adding 1.5 * 2^23 + 127 leaves n + 127 in the
// low mantissa bits, which shifted up are 2^n's bits.  2^r is a polynomial of
// degree 5, fitted here for the least relative error on that interval (7.5e-8,
// 2.4e-7 with f32 coefficients and steps: ex2's own error).
__device__ __forceinline__ float2 exp2_poly_add(float2 x, float2 acc) {
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.x) : "f"(-127.f));
    asm("max.NaN.f32 %0, %0, %1;" : "+f"(x.y) : "f"(-127.f));
    const float2 t = __fadd2_rn(x, make_float2(12583039.f, 12583039.f));
    const float2 n = __fadd2_rn(t, make_float2(-12583039.f, -12583039.f));
    const float2 r = __ffma2_rn(n, make_float2(-1.f, -1.f), x);
    float2 p = __ffma2_rn(make_float2(1.3276472454890609e-3f, 1.3276472454890609e-3f), r,
                          make_float2(9.675540961325169e-3f, 9.675540961325169e-3f));
    p = __ffma2_rn(p, r, make_float2(5.550713092088699e-2f, 5.550713092088699e-2f));
    p = __ffma2_rn(p, r, make_float2(0.24022120237350464f, 0.24022120237350464f));
    p = __ffma2_rn(p, r, make_float2(0.6931469440460205f, 0.6931469440460205f));
    p = __ffma2_rn(p, r, make_float2(1.0000001192092896f, 1.0000001192092896f));
    return __ffma2_rn(
        p, make_float2(__int_as_float(__float_as_int(t.x) << 23), __int_as_float(__float_as_int(t.y) << 23)), acc);
}

// acc + 2^x of pair i of a run of pairs: one pair in kPolyEvery on the FMA
// pipe, the rest on MUFU.
constexpr int kPolyEvery = 5;
__device__ __forceinline__ float2 exp2_add(float2 x, int i, float2 acc) {
    return i % kPolyEvery == kPolyEvery - 1 ? exp2_poly_add(x, acc)
                                            : __fadd2_rn(acc, make_float2(ex2(x.x), ex2(x.y)));
}

// ---------------------------------------------------------- 16-bit: tcgen05 --
constexpr int BM = 128;                 // rows of a query tile, keys of a key tile
constexpr int kPairs = 3;               // pairs of softmax warpgroups
constexpr int kWgs = 2 * kPairs;
constexpr int kTcThreads = 128 + kWgs * 128;  // producer, MMA, 2 idle warps, the softmax warps
constexpr int kHalfTile = BM * 128;     // [128][64 x 16-bit], 128-byte swizzled
constexpr int kMaxGroup = 4;            // query tiles a statistics CTA keeps on chip
// S tiles in TMEM (128 columns each), one per pair: a buffer's fills are all
// awaited by the same warps, in order, as the barrier's one phase bit demands.
constexpr int kSBufs = kPairs;
constexpr int kTmemCols = 512;          // a power of two
constexpr int kSms = 148;
constexpr int kBatch = 4;               // key tiles whose sums are put together at a time

template <int D>
struct TcLayout {
    static constexpr int kTile = D / 64 * kHalfTile;
    static constexpr int kSlots = D == 128 ? 6 : 12;  // query + key tiles on chip
    // statistics pass: float2 [kWgs][kMaxGroup * BM]; sums pass: float
    // [kSlots][BM] lse of the query tiles on chip, then [2][kBatch][kWgs][BM] sums
    static constexpr int kOffStat = kSlots * kTile;
    static constexpr int kOffRed = kOffStat + kSlots * BM * 4;
    static constexpr int kOffBar = kOffRed + 2 * kBatch * kWgs * BM * 4;
    static_assert(kOffStat + kWgs * kMaxGroup * BM * 8 <= kOffBar, "statistics pass");
    static constexpr int kBars = 2 * 12 + 2 * 12 + 2 * kSBufs + 1;
    static constexpr int kBytes = kOffBar + kBars * 8 + 32;
    static_assert(kBytes + 1024 <= 232448, "shared memory");
};

struct WeightPlan {
    int32_t T;         // tokens of a query tile (128 / G)
    int32_t n_rt;      // query tiles of the window, per KV head
    int32_t n_kt;      // key tiles
    int32_t group;     // query tiles of a statistics CTA
    int32_t n_groups;
    int32_t splits;    // key splits of the statistics pass
    int32_t resident;  // sums pass: every query tile stays on chip
    int32_t q_slots, k_slots;  // sums pass
    int32_t kg;        // sums pass: key tiles a CTA works on at a time (1, 2)
    int32_t b_splits;  // sums pass: CTAs per KV head (and row split)
    int32_t r_splits;  // sums pass: parts the query tiles are split into
    float* part;       // [r_splits][Hkv][n_kt * 128] sums of each part (r_splits > 1)
    float2* ml;        // [splits][Hkv][n_rt * 128]
    float* nlse;       // [Hkv][n_rt * 128]: minus the lse, log2 units, -inf for rows that are none
};

// Barriers of a CTA.
struct TcBars {
    uint64_t *qf, *qe, *kf, *ke, *sf, *se, *done;
    __device__ __forceinline__ explicit TcBars(unsigned char* p) {
        uint64_t* b = reinterpret_cast<uint64_t*>(p);
        qf = b, qe = b + 12, kf = b + 24, ke = b + 36, sf = b + 48, se = sf + kSBufs, done = se + kSBufs;
    }
};

// Key tile kt of KV head h into `dst`, one page-sized segment at a time.
template <int D, int SEG>
__device__ __forceinline__ void load_keys(const WeightArgs& a, const CUtensorMap* tm, unsigned char* dst, uint64_t* bar,
                                          int kt, int h) {
    int rows[BM / SEG];
#pragma unroll
    for (int i = 0; i < BM / SEG; ++i) {
        const int r = kt * BM + i * SEG;
        rows[i] = r;
        if (a.paging.block_rows > 0) {
            rows[i] = a.paging.pool_rows;  // past the pool: zeros
            if (r < a.kv_len) {
                bool bad = false;
                const int pr = phys_row(a.paging, r, bad);
                if (bad) report_error(a.err, kDevBadBlockTable, 0x92, r);
                else rows[i] = pr;
            }
        }
    }
    tc::mbar_arrive_expect_tx(bar, TcLayout<D>::kTile);
#pragma unroll
    for (int i = 0; i < BM / SEG; ++i)
#pragma unroll
        for (int hf = 0; hf < D / 64; ++hf)
            tc::tma_load_3d(dst + hf * kHalfTile + i * SEG * 128, tm, bar, hf * 64, h, rows[i]);
}

template <int D>
__device__ __forceinline__ void load_queries(const WeightArgs& a, const WeightPlan& p, const CUtensorMap* tm,
                                             unsigned char* dst, uint64_t* bar, int rt, int h) {
    const int G = a.n_head / a.n_head_kv;
#pragma unroll
    for (int hf = 0; hf < D / 64; ++hf)
        tc::tma_load_3d(dst + hf * kHalfTile, tm, bar, hf * 64, h * G, a.row_begin + rt * p.T);
}

// A position in a ring of tiles: its slot and the parity of that slot's fill.
struct Ring {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next(int slots) {
        if (++slot == slots) {
            slot = 0;
            phase ^= 1;
        }
    }
};

// S (columns of one TMEM buffer) = A B^T over D; operand descriptors of a tile
// in slot i are the base plus i tiles.
template <bool BF16, int D>
__device__ __forceinline__ void issue_s(uint32_t tmem, int buf, uint64_t da, uint64_t db) {
    constexpr uint32_t idesc = tc::make_idesc_f16(BF16, BM, BM, false);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
        const uint64_t off = (uint64_t)(((kk >> 2) * kHalfTile + (kk & 3) * 32) >> 4);
        tc::mma_ss(tmem + buf * BM, da + off, db + off, idesc, kk > 0 ? 1u : 0u);
    }
}

// 32 columns of S of this thread's lane.
__device__ __forceinline__ void take_s(uint32_t addr, float (&s)[32]) {
    uint32_t u[32];
    tc::tmem_ld32(addr, u);
    tc::tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 32; ++i) s[i] = __uint_as_float(u[i]);
}
// (once the last column has left it)
__device__ __forceinline__ void give_back(uint64_t* se, int lane) {
    tc::fence_before_sync();
    __syncwarp();
    if (lane == 0) tc::mbar_arrive(se);
}

// What rows [c0, c1) of the query tile whose first token is `tok0` of the window
// give one key.  Rows of a tile that are none are zeros with an lse of -inf:
// they add nothing to a finite key, but 0 * inf to one with an infinity.  A NaN
// sum of a tile that has such rows is therefore taken again, here, without
// them; `lse`: minus the tile's lse.  (In line and in loops that stay loops, 64
// rows of 32 heads over 64K keys 107.2 us, 107.0 without it; as a call 3 % more,
// with the columns masked in every step 4 to 6 %.)
template <bool BF16, int D>
__device__ __forceinline__ float weigh_again(const WeightArgs& a, const float* lse, int c0, int c1, int tok0, int h, int key) {
    const int G = a.n_head / a.n_head_kv, at = a.kv_len - a.n_tok + a.row_begin + tok0;  // cache row of the first token
    const float sl2 = a.kq_scale * 1.4426950408889634f;
    bool bad = false;
    const int kr = phys_row(a.paging, key, bad);
    if (bad) return 0.f;  // (reported when the tile was loaded)
    auto two = [](uint32_t u) {
        if constexpr (BF16) return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
        else return __half22float2(*reinterpret_cast<const __half2*>(&u));
    };
    const uint4* k = static_cast<const uint4*>(a.k) + ((int64_t)kr * a.n_head_kv + h) * (D / 8);
    float sum = 0.f;
#pragma unroll 1
    for (int c = max(c0, (key - at) * G); c < c1 && sum == sum; ++c) {  // from the first row that sees the key
        const uint4* q = static_cast<const uint4*>(a.q) +
                         ((int64_t)(a.row_begin + tok0 + c / G) * a.n_head + h * G + c % G) * (D / 8);
        float x = 0.f;
#pragma unroll 1
        for (int i = 0; i < D / 8; ++i) {
            const uint4 u = q[i], v = k[i];
            const uint32_t us[4] = {u.x, u.y, u.z, u.w}, vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 y = two(us[j]), z = two(vs[j]);
                x = fmaf(y.x, z.x, x);
                x = fmaf(y.y, z.y, x);
            }
        }
        sum += ex2(fmaf(x, sl2, lse[c]));
    }
    return sum;
}

// PASS 0: statistics.  CTA (key split, group of query tiles, KV head): the
// group's query tiles stay, key tiles stream; TMEM lane = query row, so each
// thread keeps the maximum and sum of one row over its columns.
// PASS 1: sums.  CTA (slice of key tiles, KV head): TMEM lane = key, columns =
// query rows, so each thread sums one key's weights in registers; key tiles
// (kg at a time) against all query tiles, which stay when they fit and
// stream otherwise.
// A step is one (query tile, key tile); three pairs of warpgroups, an S buffer
// each, take the steps in turn, each warpgroup 64 of the 128 columns, 32 at a
// time (the buffer goes back to the MMA warp halfway).  MUFU (57 to 68 %) and
// the issue slots (53 to 56 %) are the busiest units: 24 warps hide more of each
// other's waits than 16 with 64 columns in registers (96 against 101 us for 64
// rows of 32 heads over 64K keys); a warpgroup per step measured 99 us.
// STREAM: the sums pass whose query tiles stream.
template <bool BF16, int D, int SEG, int PASS, bool STREAM>
__global__ void __launch_bounds__(kTcThreads, 1)
    k7_pass(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
            const __grid_constant__ WeightArgs a, const __grid_constant__ WeightPlan p) {
    using LY = TcLayout<D>;
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
    TcBars b(smem + LY::kOffBar);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + LY::kOffBar + LY::kBars * 8);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int Hkv = a.n_head_kv, G = a.n_head / Hkv;
    const int t_first = a.kv_len - a.n_tok + a.row_begin;  // cache row of the window's first token
    const uint64_t tmo = a.timeout_ns;

    // the CTA's part
    int h, rs = 0, rt0 = 0, n_q, k0, k1, q_slots, k_slots;
    constexpr bool stream_q = STREAM;
    static_assert(PASS == 1 || !STREAM, "the statistics pass keeps its query tiles");
    if constexpr (PASS == 0) {
        const int sp = blockIdx.x % p.splits, rest = blockIdx.x / p.splits;
        h = rest / p.n_groups;
        // late groups first: they see the most keys
        rt0 = (p.n_groups - 1 - rest % p.n_groups) * p.group;
        n_q = min(p.group, p.n_rt - rt0);
        const int last = min(t_first + (rt0 + n_q) * p.T, a.kv_len) - 1;
        const int n_kt = last / BM + 1;
        k0 = (int)((int64_t)n_kt * sp / p.splits);
        k1 = (int)((int64_t)n_kt * (sp + 1) / p.splits);
        q_slots = p.group;
        k_slots = LY::kSlots - p.group;
    } else {
        const int rest = blockIdx.x / p.r_splits;
        rs = p.r_splits - 1 - blockIdx.x % p.r_splits;  // late rows first
        h = rest / p.b_splits;
        rt0 = (int)((int64_t)p.n_rt * rs / p.r_splits);
        n_q = (int)((int64_t)p.n_rt * (rs + 1) / p.r_splits) - rt0;
        k0 = rest % p.b_splits;  // groups of kg key tiles: k0, k0 + b_splits, ...
        // (no row of the part sees the key tiles after its last)
        k1 = ((min(t_first + (rt0 + n_q) * p.T, a.kv_len) - 1) / BM + p.kg) / p.kg;
        q_slots = p.q_slots;
        k_slots = p.k_slots;
    }
    unsigned char* kbase = smem + q_slots * LY::kTile;
    float* lse_s = reinterpret_cast<float*>(smem + LY::kOffStat);

    if (threadIdx.x == 0) {
        for (int i = 0; i < q_slots; ++i) {
            tc::mbar_init(&b.qf[i], 1);
            tc::mbar_init(&b.qe[i], 1 + 4 * kWgs);  // the MMAs' commit and the softmax warps
        }
        for (int i = 0; i < k_slots; ++i) {
            tc::mbar_init(&b.kf[i], 1);
            tc::mbar_init(&b.ke[i], 1);
        }
        for (int i = 0; i < kSBufs; ++i) {
            tc::mbar_init(&b.sf[i], 1);
            tc::mbar_init(&b.se[i], 8);  // the warps of two warpgroups
        }
        tc::mbar_init(b.done, 1);
        tc::fence_mbar_init();
        tc::tma_prefetch_desc(&tmQ);
        tc::tma_prefetch_desc(&tmK);
    }
    if (warp == 1) {
        tc::tmem_alloc(tmem_slot, kTmemCols);
        tc::tmem_relinquish();
    }
    // Query rows past T * G are never written by TMA: zeros, so that no stale
    // shared memory reaches the tensor cores.
    if (const int used = p.T * G; used < BM) {
        const int n16 = (BM - used) * 8;
        for (int i = threadIdx.x; i < n16 * q_slots * (D / 64); i += kTcThreads)
            *(reinterpret_cast<uint4*>(smem + (i / n16) * kHalfTile + used * 128) + i % n16) = make_uint4(0, 0, 0, 0);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tc::pdl_wait();
    tc::pdl_launch();
    tc::fence_before_sync();
    __syncthreads();
    tc::fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    const int q_bytes = D / 64 * 64 * 2 * p.T * G;

    // first of the CTA's query tiles that sees any key of group kgi, n_q or
    // more if none does (sums pass; on chip, all are taken: there are few)
    auto rt_from = [&](int kgi) {
        const int late = kgi * p.kg * BM - t_first;
        return !stream_q || late < p.T ? 0 : max(0, late / p.T - rt0);
    };

    if (warp == 0) {
        // ------------------------------------------------------ producer --
        if (lane == 0) {
            bool ok = true;
            int kt_n = 0, qt_n = 0;  // tiles issued into each ring
            Ring kr, qr;
            auto keys = [&](int kt) {
                ok = tc::mbar_wait(&b.ke[kr.slot], kr.phase ^ 1, tmo);
                if (!ok) return;
                load_keys<D, SEG>(a, &tmK, kbase + kr.slot * LY::kTile, &b.kf[kr.slot], kt, h);
                kr.next(k_slots);
                ++kt_n;
            };
            if (!stream_q) {
                tc::mbar_arrive_expect_tx(&b.qf[0], (q_bytes + (PASS == 1 ? BM * 4 : 0)) * n_q);
                for (int i = 0; i < n_q; ++i)
                    load_queries<D>(a, p, &tmQ, smem + i * LY::kTile, &b.qf[0], rt0 + i, h);
                if constexpr (PASS == 1)
                    tc::bulk_load(lse_s, p.nlse + ((int64_t)h * p.n_rt + rt0) * BM, BM * 4 * n_q, &b.qf[0]);
            }
            if constexpr (PASS == 0) {
                for (int kt = k0; kt < k1 && ok; ++kt) keys(kt);
            } else {
                for (int g = k0; g < k1 && ok; g += p.b_splits) {
                    const int r0 = rt_from(g);
                    if (r0 >= n_q) continue;
                    for (int k = 0; k < p.kg && g * p.kg + k < p.n_kt && ok; ++k) keys(g * p.kg + k);
                    if constexpr (STREAM) {
                        for (int rt = r0; rt < n_q && ok; ++rt) {
                            const int s = qr.slot;
                            ok = tc::mbar_wait(&b.qe[s], qr.phase ^ 1, tmo);
                            if (!ok) break;
                            tc::mbar_arrive_expect_tx(&b.qf[s], q_bytes + BM * 4);
                            load_queries<D>(a, p, &tmQ, smem + s * LY::kTile, &b.qf[s], rt0 + rt, h);
                            tc::bulk_load(lse_s + s * BM, p.nlse + ((int64_t)h * p.n_rt + rt0 + rt) * BM, BM * 4, &b.qf[s]);
                            qr.next(q_slots);
                            ++qt_n;
                        }
                    }
                }
            }
            if (!ok) report_error(a.err, kDevWaitWeights, 0xb0 + PASS, kt_n);
            // copies still in flight land before the CTA ends
            for (int j = max(0, kt_n - k_slots); j < kt_n; ++j)
                tc::mbar_wait(&b.kf[j % k_slots], (j / k_slots) & 1, tmo);
            if (!stream_q) tc::mbar_wait(&b.qf[0], 0, tmo);
            for (int j = max(0, qt_n - q_slots); j < qt_n; ++j)
                tc::mbar_wait(&b.qf[j % q_slots], (j / q_slots) & 1, tmo);
        }
    } else if (warp == 1) {
        // ----------------------------------------------------------- MMA --
        const bool leader = tc::elect_one();
        bool ok = true;
        int step = 0;
        Ring kr, qr;
        constexpr uint64_t kTileD = LY::kTile >> 4;
        const uint64_t dq = tc::make_sdesc_sw128(tc::smem_u32(smem), 16, 1024);
        const uint64_t dk = tc::make_sdesc_sw128(tc::smem_u32(kbase), 16, 1024);
        auto wait = [&](uint64_t* bar, uint32_t par) {
            if (ok) ok = __all_sync(0xffffffffu, tc::mbar_wait(bar, par, tmo));
            return ok;
        };
        auto commit = [&](uint64_t* bar) {
            if (leader) tc::mma_commit(bar);
            __syncwarp();
        };
        auto one = [&](uint64_t q, uint64_t k) {
            const int buf = step % kSBufs;
            if (!wait(&b.se[buf], ((step / kSBufs) & 1) ^ 1)) return;
            tc::fence_after_sync();
            if (leader) {
                issue_s<BF16, D>(tmem, buf, PASS == 0 ? q : k, PASS == 0 ? k : q);
                tc::mma_commit(&b.sf[buf]);
            }
            __syncwarp();
            ++step;
        };
        if (!stream_q) wait(&b.qf[0], 0);
        if constexpr (PASS == 0) {
            for (int kt = k0; kt < k1 && ok; ++kt) {
                wait(&b.kf[kr.slot], kr.phase);
                for (int r = 0; r < n_q && ok; ++r) one(dq + r * kTileD, dk + kr.slot * kTileD);
                if (ok) commit(&b.ke[kr.slot]);
                kr.next(k_slots);
            }
        } else {
            for (int g = k0; g < k1 && ok; g += p.b_splits) {
                const int r0 = rt_from(g), nk = min(p.kg, p.n_kt - g * p.kg);
                if (r0 >= n_q) continue;
                Ring k2 = kr;
                k2.next(k_slots);
                for (int rt = r0; rt < n_q && ok; ++rt) {
                    const int qs = stream_q ? qr.slot : rt;
                    if (stream_q) wait(&b.qf[qs], qr.phase);
                    if (rt == r0) wait(&b.kf[kr.slot], kr.phase);
                    if (ok) one(dq + qs * kTileD, dk + kr.slot * kTileD);
                    if (nk == 2) {
                        if (rt == r0) wait(&b.kf[k2.slot], k2.phase);
                        if (ok) one(dq + qs * kTileD, dk + k2.slot * kTileD);
                    }
                    if (stream_q) {
                        if (ok) commit(&b.qe[qs]);
                        qr.next(q_slots);
                    }
                }
                if (!ok) break;
                commit(&b.ke[kr.slot]);
                kr.next(k_slots);
                if (nk == 2) {
                    commit(&b.ke[kr.slot]);
                    kr.next(k_slots);
                }
            }
        }
        if (!ok && lane == 0) report_error(a.err, kDevWaitWeights, 0xb2 + PASS, step);
        // every MMA retires before TMEM is freed
        commit(b.done);
        tc::mbar_wait(b.done, 0, tmo);
        __syncwarp();
    } else if (warp >= 4) {
        // ------------------------------------------------------- softmax --
        const int wg = (warp - 4) >> 2, pair = wg >> 1, half = wg & 1, wq = warp & 3, row = wq * 32 + lane;
        const uint32_t s_addr = tmem + ((uint32_t)(wq * 32) << 16) + half * 64;
        const float sl2 = a.kq_scale * 1.4426950408889634f;
        const float2 sl2_2 = make_float2(sl2, sl2);
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t par, int step) {
            if (ok) {
                ok = __all_sync(0xffffffffu, tc::mbar_wait(bar, par, tmo));
                if (!ok && lane == 0) report_error(a.err, kDevWaitWeights, 0xb4 + PASS, step);
            }
            return ok;
        };
        if constexpr (PASS == 0) {
            float2* stats = reinterpret_cast<float2*>(smem + LY::kOffStat);
            float2* stat = stats + wg * kMaxGroup * BM + row;
            for (int r = 0; r < n_q; ++r) stat[r * BM] = make_float2(-INFINITY, 0.f);
            const int steps = (k1 - k0) * n_q;
            int kt = k0, r = pair, r_held = -1;
            while (r >= n_q) r -= n_q, ++kt;
            float2 st = make_float2(-INFINITY, 0.f);  // of query tile r_held
            for (int step = pair; step < steps; step += kPairs) {
                const int buf = pair;  // = step % kSBufs
                if (!wait(&b.sf[buf], (step / kSBufs) & 1, step)) break;
                tc::fence_after_sync();
                if (r != r_held) {
                    if (r_held >= 0) stat[r_held * BM] = st;
                    st = stat[r * BM];
                    r_held = r;
                }
                const int tt = t_first + (rt0 + r) * p.T, key = kt * BM + half * 64;
                const bool cut = key + 63 > tt;
                const int lim = tt + row / G - key;
#pragma unroll
                for (int hc = 0; hc < 2; ++hc) {
                    float s[32];
                    take_s(s_addr + buf * BM + hc * 32, s);
                    if (hc == 1) give_back(&b.se[buf], lane);
                    if (cut) {
#pragma unroll
                        for (int c = 0; c < 32; ++c)
                            if (hc * 32 + c > lim) s[c] = -INFINITY;
                    }
                    float mx[2] = {s[0], s[1]};
#pragma unroll
                    for (int c = 2; c < 30; c += 4)
#pragma unroll
                        for (int i = 0; i < 2; ++i) mx[i] = max3f(mx[i], s[c + i], s[c + 2 + i]);
                    mx[0] = max3f(mx[0], s[30], s[31]);
                    const float m = fmaxf(st.x, fmaxf(mx[0], mx[1]) * sl2);
                    const float ms = m == -INFINITY ? 0.f : m;
                    const float2 nm = make_float2(-ms, -ms);
                    float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                    for (int c = 0; c < 16; ++c)
                        acc[c & 1] = exp2_add(__ffma2_rn(make_float2(s[2 * c], s[2 * c + 1]), sl2_2, nm), hc * 16 + c, acc[c & 1]);
                    const float2 t = __fadd2_rn(acc[0], acc[1]);
                    st = make_float2(m, st.y * ex2(st.x - ms) + (t.x + t.y));
                }
                r += kPairs;
                while (r >= n_q) r -= n_q, ++kt;
            }
            if (r_held >= 0) stat[r_held * BM] = st;
            // the warpgroups' statistics of each row
            tc::named_bar_sync(1, kWgs * 128);
            const int sp = blockIdx.x % p.splits;
            float2* out = p.ml + ((int64_t)sp * Hkv + h) * p.n_rt * BM + rt0 * BM;
            for (int i = wg * BM + row; i < n_q * BM; i += kWgs * BM) {
                float2 v[kWgs];
                float m = -INFINITY, l = 0.f;
#pragma unroll
                for (int w = 0; w < kWgs; ++w) {
                    v[w] = stats[w * kMaxGroup * BM + i];
                    m = fmaxf(m, v[w].x);
                }
                const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
                for (int w = 0; w < kWgs; ++w) l += v[w].y * ex2(v[w].x - ms);
                out[i] = make_float2(m, l);
            }
        } else {
            // sums of up to kBatch key tiles wait in shared memory for the
            // other warpgroups': one barrier per batch
            float* red = reinterpret_cast<float*>(smem + LY::kOffRed);  // [2 turns][kBatch][kWgs][BM]
            int turn = 0, held = 0;
            auto put = [&](float v) { red[((turn * kBatch + held++) * kWgs + wg) * BM + row] = v; };
            auto flush = [&](int g_first) {
                tc::named_bar_sync(1, kWgs * 128);
                for (int i = wg * BM + row; i < held * BM && ok; i += kWgs * BM) {
                    const int j = i / BM, gj = p.kg == 1 ? j : j >> 1;
                    const int kt = (g_first + gj * p.b_splits) * p.kg + (p.kg == 1 ? 0 : j & 1), key = kt * BM + row;
                    if (key >= a.kv_len) continue;
                    const float* from = red + (turn * kBatch + j) * kWgs * BM + row;
                    float v = 0.f;
#pragma unroll
                    for (int w = 0; w < kWgs; ++w) v += from[w * BM];
                    if (p.r_splits > 1) {
                        p.part[((int64_t)rs * Hkv + h) * p.n_kt * BM + key] = v;
                        continue;
                    }
                    float* out = a.acc + (int64_t)h * a.acc_stride + key;
                    *out = a.accumulate ? *out + v : v;
                }
                turn ^= 1;
                held = 0;
            };
            // one step: the weights that the 64 rows of query tile rt (slot qs) in `half` give this thread's key of tile kt, summed
            auto take_step = [&](int step, int kt, int rt, int qs) -> float {
                const int buf = pair;  // = step % kSBufs
                if (!wait(&b.sf[buf], (step / kSBufs) & 1, step)) return 0.f;
                tc::fence_after_sync();
                const float4* l4 = reinterpret_cast<const float4*>(lse_s + qs * BM + half * 64);
                const int key0 = kt * BM, tt = t_first + (rt0 + rt) * p.T;
                float2 acc[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                for (int hc = 0; hc < 2; ++hc) {
                    float s[32];
                    take_s(s_addr + buf * BM + hc * 32, s);
                    if (hc == 1) give_back(&b.se[buf], lane);
                    if (key0 + BM - 1 > tt) {
                        int tok = tt + (half * 64 + hc * 32) / G, rem = (half * 64 + hc * 32) % G;
#pragma unroll
                        for (int c = 0; c < 32; ++c) {
                            if (key0 + row > tok) s[c] = -INFINITY;
                            if (++rem == G) rem = 0, ++tok;
                        }
                    }
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        const float4 l = l4[hc * 8 + c];
                        acc[0] = exp2_add(__ffma2_rn(make_float2(s[4 * c], s[4 * c + 1]), sl2_2, make_float2(l.x, l.y)), hc * 16 + 2 * c,
                                          acc[0]);
                        acc[1] = exp2_add(__ffma2_rn(make_float2(s[4 * c + 2], s[4 * c + 3]), sl2_2, make_float2(l.z, l.w)),
                                          hc * 16 + 2 * c + 1, acc[1]);
                    }
                }
                const float2 t = __fadd2_rn(acc[0], acc[1]);
                float v = t.x + t.y;
                if (__any_sync(0xffffffffu, v != v)) {
                    const int live = min(p.T, a.kv_len - tt) * G - half * 64;  // of this thread's 64 columns
                    if (v != v && live < 64 && key0 + row < a.kv_len)
                        v = weigh_again<BF16, D>(a, lse_s + qs * BM, half * 64, half * 64 + live, (rt0 + rt) * p.T, h, key0 + row);
                    __syncwarp();
                }
                return v;
            };
            if constexpr (!STREAM) {
                // steps (key tile, query tile) in turn; this pair of warpgroups has every third one
                wait(&b.qf[0], 0, 0);
                const int n_mine = k0 < k1 ? (k1 - 1 - k0) / p.b_splits + 1 : 0;
                int i = 0, rt = pair, kt = k0, g_first = k0;
                float sum = 0.f;
                for (int step = pair; i < n_mine; step += kPairs) {
                    while (rt >= n_q && i < n_mine) {
                        put(sum);
                        sum = 0.f;
                        rt -= n_q;
                        kt += p.b_splits;
                        if (++i == n_mine || held == kBatch) {
                            flush(g_first);
                            g_first = kt;
                        }
                    }
                    if (i == n_mine) break;
                    sum += take_step(step, kt, rt, rt);
                    rt += kPairs;
                }
            } else {
                Ring qr;
                int step = 0, g_first = k0;
                for (int g = k0; g < k1; g += p.b_splits) {
                    const int r0 = rt_from(g), nk = min(p.kg, p.n_kt - g * p.kg);
                    float sum0 = 0.f, sum1 = 0.f;
                    for (int rt = r0; rt < n_q && ok; ++rt) {
                        const int qs = qr.slot;
                        wait(&b.qf[qs], qr.phase, step);
                        for (int k = 0; k < nk; ++k, ++step) {
                            if (step % kPairs != pair) continue;
                            const float v = take_step(step, g * p.kg + k, rt, qs);
                            if (k == 0) sum0 += v;
                            else sum1 += v;
                        }
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive(&b.qe[qs]);
                        qr.next(q_slots);
                    }
                    put(sum0);
                    if (p.kg == 2) put(sum1);
                    if (held == kBatch || g + p.b_splits >= k1) {
                        flush(g_first);
                        g_first = g + p.b_splits;
                    }
                }
            }
        }
    }
    tc::fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc::fence_after_sync();
        tc::tmem_dealloc(tmem, kTmemCols);
    }
}

// The rows' (minus) log-sum-exp from the splits' statistics: 16 lanes to a row.
// `there`: whether row i of a head's n is one.
constexpr int kJoinThreads = 256;
template <class F>
__device__ __forceinline__ void join_rows(const float2* ml, float* nlse, int64_t n, int heads, int splits, F&& there) {
    const int64_t at = (int64_t)blockIdx.x * (kJoinThreads / 16) + threadIdx.x / 16, stride = n * heads;
    const int part = threadIdx.x % 16;
    if (at >= stride) return;  // (whole groups of 16 lanes)
    const uint32_t lanes = 0xffffu << (threadIdx.x & 16);
    float m = -INFINITY, l = 0.f;
    for (int s = part; s < splits; s += 16) m = fmaxf(m, ml[s * stride + at].x);
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor_sync(lanes, m, d));
    const float ms = m == -INFINITY ? 0.f : m;
    for (int s = part; s < splits; s += 16) {
        const float2 v = ml[s * stride + at];
        l += v.y * ex2(v.x - ms);
    }
#pragma unroll
    for (int d = 8; d > 0; d >>= 1) l += __shfl_xor_sync(lanes, l, d);
    if (part == 0) nlse[at] = there(at % n) ? -(ms + log2f(l)) : -INFINITY;
}

// The parts' sums of each key, in order, into acc; `stride`: keys of a row of
// `part` [splits][Hkv][stride].  T > 0: parts of n_rt query tiles of T tokens,
// which only wrote the key tiles that they see.
__global__ void __launch_bounds__(kJoinThreads) k7_add(const WeightArgs a, const float* part, int stride, int splits,
                                                       int T, int n_rt) {
    tc::pdl_wait();
    tc::pdl_launch();
    const int key = blockIdx.x * kJoinThreads + threadIdx.x, h = blockIdx.y;
    if (key >= a.kv_len) return;
    int first = 0;
    if (const int late = key / BM * BM - (a.kv_len - a.n_tok + a.row_begin); T > 0 && late > 0)
        while (first + 1 < splits && (int)((int64_t)n_rt * (first + 1) / splits) * T <= late) ++first;
    float v = 0.f;
#pragma unroll 8
    for (int s = first; s < splits; ++s) v += part[((int64_t)s * a.n_head_kv + h) * stride + key];
    float* out = a.acc + (int64_t)h * a.acc_stride + key;
    *out = a.accumulate ? *out + v : v;
}

__global__ void __launch_bounds__(kJoinThreads) k7_join(const WeightArgs a, const WeightPlan p) {
    tc::pdl_wait();
    tc::pdl_launch();
    const int G = a.n_head / a.n_head_kv;
    join_rows(p.ml, p.nlse, (int64_t)p.n_rt * BM, a.n_head_kv, p.splits, [&](int64_t i) {
        const int r = (int)(i % BM);
        return r < p.T * G && (int)(i / BM) * p.T + r / G < a.n_tok - a.row_begin;
    });
}

// ------------------------------------------------------------ f32: CUDA cores --
constexpr int FT = 64;          // query rows, and keys, of a tile
constexpr int kF32Threads = 256;  // 16 x 16 threads, 4 rows x 4 keys each

struct F32Plan {
    int32_t n_rows;  // (token, head) rows of the window per KV head
    int32_t n_rt, n_kt, splits, r_splits;
    float* part;     // [r_splits][Hkv][n_kt * 64] (r_splits > 1)
    float2* ml;      // [splits][Hkv][n_rt * 64]
    float* nlse;     // [Hkv][n_rt * 64]: minus the lse, -inf for rows that are none
    float* scores;   // [Hkv][n_rt * 64][n_kt * 64] log2 units, of the tiles with a visible key (null: not kept)
};

// Scores that fit L2 next to everything else are written and read once instead
// of being computed twice, and given up there once read: 2 launches, not 3 or 4.
// (14 heads of 64, 32 rows over 4096 keys: 25 us against 30; 32 heads of 128,
// 128 rows, 64 MB of scores: 165 against 287.)
constexpr int64_t kKeptScores = 16 << 20;
constexpr int kKeptCtas = 4 * kSms;  // of the second pass, at once

// 64 rows of D floats on their way into shared memory: fetch has all of a
// thread's loads under way at once, store follows when the buffer is free.
// Rows are padded by 16 bytes (the 4 x 4 product reads 8 rows at once without
// a bank conflict).
template <int D>
struct RowsF32 {
    static constexpr int kN = FT * (D / 4) / kF32Threads;
    float4 v[kN];
    // src(r): the row's address, null for zeros; four threads to a row
    template <class F>
    __device__ __forceinline__ void fetch(F&& src) {
        static_assert(kF32Threads == 4 * FT, "four threads to a row");
        const float* p = src(threadIdx.x / 4);
#pragma unroll
        for (int n = 0; n < kN; ++n)
            v[n] = p != nullptr ? *reinterpret_cast<const float4*>(p + threadIdx.x % 4 * 4 + n * 16)
                                : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __device__ __forceinline__ void store(float* dst) const {
#pragma unroll
        for (int n = 0; n < kN; ++n)
            *reinterpret_cast<float4*>(dst + threadIdx.x / 4 * (D + 4) + threadIdx.x % 4 * 4 + n * 16) = v[n];
    }
    __device__ __forceinline__ void fetch_queries(const WeightArgs& a, int n_rows, int rt, int h) {
        const int G = a.n_head / a.n_head_kv;
        fetch([&](int r) -> const float* {
            const int i = rt * FT + r;
            if (i >= n_rows) return nullptr;
            const int tok = i / G;
            return static_cast<const float*>(a.q) +
                   ((int64_t)(a.row_begin + tok) * a.n_head + h * G + (i - tok * G)) * D;
        });
    }
    __device__ __forceinline__ void fetch_keys(const WeightArgs& a, int kt, int h) {
        fetch([&](int r) -> const float* {
            const int j = kt * FT + r;
            if (j >= a.kv_len) return nullptr;
            bool bad = false;
            const int row = phys_row(a.paging, j, bad);
            if (bad) {
                report_error(a.err, kDevBadBlockTable, 0x92, j);
                return nullptr;
            }
            return static_cast<const float*>(a.k) + ((int64_t)row * a.n_head_kv + h) * D;
        });
    }
};

// x[i][j] = q row (ty + 16 i) . k row (tx + 16 j), i < NI
template <int D, int NI>
__device__ __forceinline__ void scores_f32(const float* q, const float* k, int ty, int tx, float (&x)[NI][4]) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i][j] = 0.f;
#pragma unroll 4
    for (int c = 0; c < D; c += 4) {
        float4 qq[NI], kk[4];
#pragma unroll
        for (int i = 0; i < NI; ++i) qq[i] = *reinterpret_cast<const float4*>(q + (ty + 16 * i) * (D + 4) + c);
#pragma unroll
        for (int i = 0; i < 4; ++i) kk[i] = *reinterpret_cast<const float4*>(k + (tx + 16 * i) * (D + 4) + c);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[i][j] = fmaf(qq[i].x, kk[j].x, x[i][j]);
                x[i][j] = fmaf(qq[i].y, kk[j].y, x[i][j]);
                x[i][j] = fmaf(qq[i].z, kk[j].z, x[i][j]);
                x[i][j] = fmaf(qq[i].w, kk[j].w, x[i][j]);
            }
    }
}

template <int D>
__global__ void __launch_bounds__(kF32Threads) k7_stats_f32(const WeightArgs a, const F32Plan p) {
    extern __shared__ __align__(16) float sm[];
    float *q = sm, *k = sm + FT * (D + 4);
    tc::pdl_wait();
    tc::pdl_launch();
    const int sp = blockIdx.x % p.splits, rest = blockIdx.x / p.splits;
    const int rt = p.n_rt - 1 - rest % p.n_rt, h = rest / p.n_rt;  // late rows first: they see the most keys
    const int G = a.n_head / a.n_head_kv, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int t_first = a.kv_len - a.n_tok + a.row_begin;
    const float sl2 = a.kq_scale * 1.4426950408889634f;
    const int last_row = min(rt * FT + FT, p.n_rows) - 1;
    const int n_kt = (t_first + last_row / G) / FT + 1;
    const int k0 = (int)((int64_t)n_kt * sp / p.splits), k1 = (int)((int64_t)n_kt * (sp + 1) / p.splits);
    int tok[4], seen_to[4];
    float m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = rt * FT + ty + 16 * i;
        tok[i] = t_first + r / G;
        seen_to[i] = r < p.n_rows ? tok[i] / FT : -1;  // a row that is none is not kept
        m[i] = -INFINITY;
        l[i] = 0.f;
    }
    const bool few = p.n_rows - rt * FT <= 16;  // a small window: the rows past it cost nothing
    const uint64_t keep = tc::policy_evict_last();
    const int64_t wide = (int64_t)p.n_kt * FT;
    float* scores = p.scores + (((int64_t)h * p.n_rt + rt) * FT + ty) * wide + tx;
    RowsF32<D> next;
    {
        RowsF32<D> rows;
        rows.fetch_queries(a, p.n_rows, rt, h);
        if (k0 < k1) next.fetch_keys(a, k0, h);
        rows.store(q);
    }
    for (int kt = k0; kt < k1; ++kt) {
        __syncthreads();
        next.store(k);
        __syncthreads();
        if (kt + 1 < k1) next.fetch_keys(a, kt + 1, h);
        auto tile = [&](auto ni) {
            constexpr int NI = decltype(ni)::value;
            float x[NI][4];
            scores_f32<D, NI>(q, k, ty, tx, x);
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                float mx = m[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    x[i][j] = kt * FT + tx + 16 * j <= tok[i] ? x[i][j] * sl2 : -INFINITY;
                    mx = fmaxf(mx, x[i][j]);
                }
                // (only scores that are read, and given up, by the second pass: others would stay in L2)
                if (p.scores != nullptr && kt <= seen_to[i]) {
                    const float* to = scores + 16 * i * wide + kt * FT;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        asm volatile("st.global.L2::cache_hint.f32 [%0], %1, %2;" ::"l"(to + 16 * j), "f"(x[i][j]),
                                     "l"(keep)
                                     : "memory");
                }
                const float ms = mx == -INFINITY ? 0.f : mx;
                l[i] *= ex2(m[i] - ms);
#pragma unroll
                for (int j = 0; j < 4; ++j) l[i] += ex2(x[i][j] - ms);
                m[i] = mx;
            }
        };
        if (few) tile(std::integral_constant<int, 1>{});
        else tile(std::integral_constant<int, 4>{});
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int d = 8; d > 0; d >>= 1) {
            const float m2 = __shfl_xor_sync(0xffffffffu, m[i], d), l2 = __shfl_xor_sync(0xffffffffu, l[i], d);
            const float mx = fmaxf(m[i], m2), ms = mx == -INFINITY ? 0.f : mx;
            l[i] = l[i] * ex2(m[i] - ms) + l2 * ex2(m2 - ms);
            m[i] = mx;
        }
        if (tx == 0)
            p.ml[((int64_t)sp * a.n_head_kv + h) * p.n_rt * FT + (int64_t)rt * FT + ty + 16 * i] =
                make_float2(m[i], l[i]);
    }
}

__global__ void __launch_bounds__(kJoinThreads) k7_join_f32(const WeightArgs a, const F32Plan p) {
    tc::pdl_wait();
    tc::pdl_launch();
    join_rows(p.ml, p.nlse, (int64_t)p.n_rt * FT, a.n_head_kv, p.splits, [&](int64_t i) { return i < p.n_rows; });
}

template <int D>
__global__ void __launch_bounds__(kF32Threads) k7_sums_f32(const WeightArgs a, const F32Plan p) {
    extern __shared__ __align__(16) float sm[];
    float *q = sm, *k = sm + FT * (D + 4);
    const int rs = blockIdx.x % p.r_splits, rest = blockIdx.x / p.r_splits;
    const int kt = rest % p.n_kt, h = rest / p.n_kt;
    const int r1 = (int)((int64_t)p.n_rt * (rs + 1) / p.r_splits);  // this part's last row tile + 1
    const int G = a.n_head / a.n_head_kv, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int t_first = a.kv_len - a.n_tok + a.row_begin;
    const float sl2 = a.kq_scale * 1.4426950408889634f;
    tc::pdl_wait();
    tc::pdl_launch();
    const float* nlse = p.nlse + (int64_t)h * p.n_rt * FT;
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    // first of the part's row tiles with a row that sees the keys
    const int r0 = max((int)((int64_t)p.n_rt * rs / p.r_splits), (int)((int64_t)(kt * FT - t_first) * G / FT));
    RowsF32<D> next;
    {
        RowsF32<D> rows;
        rows.fetch_keys(a, kt, h);
        if (r0 < r1) next.fetch_queries(a, p.n_rows, r0, h);
        rows.store(k);
    }
    for (int rt = r0; rt < r1; ++rt) {
        __syncthreads();
        next.store(q);
        __syncthreads();
        if (rt + 1 < r1) next.fetch_queries(a, p.n_rows, rt + 1, h);
        auto tile = [&](auto ni) {
            constexpr int NI = decltype(ni)::value;
            float x[NI][4];
            scores_f32<D, NI>(q, k, ty, tx, x);
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                // (a row that is none sees no key: its query is zeros, and a key may hold infinities)
                const int r = rt * FT + ty + 16 * i, tok = r < p.n_rows ? t_first + r / G : -1;
                const float ls = nlse[r];
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (kt * FT + tx + 16 * j <= tok) sum[j] += ex2(fmaf(x[i][j], sl2, ls));
            }
        };
        if (p.n_rows - rt * FT <= 16) tile(std::integral_constant<int, 1>{});
        else tile(std::integral_constant<int, 4>{});
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) q[ty * FT + tx + 16 * j] = sum[j];
    __syncthreads();
    if (threadIdx.x < FT && kt * FT + (int)threadIdx.x < a.kv_len) {
        float v = 0.f;
        for (int i = 0; i < 16; ++i) v += q[i * FT + threadIdx.x];
        if (p.r_splits > 1) {
            p.part[(((int64_t)rs * a.n_head_kv + h) * p.n_kt + kt) * FT + threadIdx.x] = v;
            return;
        }
        float* out = a.acc + (int64_t)h * a.acc_stride + kt * FT + threadIdx.x;
        *out = a.accumulate ? *out + v : v;
    }
}

// Sums pass over kept scores: a cluster of CTAs per 64 keys of a head, which
// share its rows (3500 rows over 8 tiles of 2 heads: one CTA each 57 us, 8 each
// 33).  The rows' sums are put together from the splits' by every cluster (L2
// holds them), a thread to a row and a part of the splits.
constexpr int kKeptThreads = 256;
constexpr int kKeptRows = 1024;  // rows whose sums a CTA holds
__global__ void __launch_bounds__(kKeptThreads) k7_kept_f32(const WeightArgs a, const F32Plan p) {
    __shared__ float nlse[kKeptRows];
    __shared__ float4 part[kKeptThreads];
    __shared__ float2 halves[kKeptThreads];
    __shared__ float sums[FT];
    tc::pdl_wait();
    tc::pdl_launch();
    const int C = p.r_splits, rank = blockIdx.x % C, kt = blockIdx.x / C % p.n_kt, h = blockIdx.x / C / p.n_kt;
    const int G = a.n_head / a.n_head_kv, t_first = a.kv_len - a.n_tok + a.row_begin;
    const int tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    const int64_t rows = (int64_t)p.n_rt * FT, stride = rows * a.n_head_kv, wide = (int64_t)p.n_kt * FT;
    const float* scores = p.scores + h * rows * wide + kt * FT + 4 * tx;
    const float2* ml = p.ml + h * rows;
    // from the first row that sees a key of the tile
    const int first = (int)max((int64_t)0, (int64_t)(kt * FT - t_first) * G), n_rows = max(0, p.n_rows - first);
    const int b1 = first + (int)((int64_t)n_rows * (rank + 1) / C);
    float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int b = first + (int)((int64_t)n_rows * rank / C); b < b1; b += kKeptRows) {
        const int n = min(kKeptRows, b1 - b);
        for (int r0 = 0; r0 < n; r0 += kKeptThreads) {
            const int here = min(n - r0, kKeptThreads), lanes = (here + 31) & ~31, parts = kKeptThreads / lanes;
            const int r = threadIdx.x % lanes, part_of = threadIdx.x / lanes;
            float m = -INFINITY, l = 0.f;
            if (r < here && part_of < parts) {
                constexpr int kAtOnce = 8;
                for (int s = part_of; s < p.splits; s += parts * kAtOnce) {
                    float2 v[kAtOnce];
                    float mx = m;
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i)
                        v[i] = s + i * parts < p.splits ? ml[(s + i * parts) * stride + b + r0 + r]
                                                        : make_float2(-INFINITY, 0.f);
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) mx = fmaxf(mx, v[i].x);
                    const float ms = mx == -INFINITY ? 0.f : mx;
                    l *= ex2(m - ms);
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) l += v[i].y * ex2(v[i].x - ms);
                    m = mx;
                }
            }
            halves[threadIdx.x] = make_float2(m, l);
            __syncthreads();
            if (part_of == 0 && r < here) {
                for (int i = 1; i < parts; ++i) {
                    const float2 u = halves[i * lanes + r];
                    const float mx = fmaxf(m, u.x), ms = mx == -INFINITY ? 0.f : mx;
                    l = l * ex2(m - ms) + u.y * ex2(u.x - ms);
                    m = mx;
                }
                nlse[r0 + r] = -(m + log2f(l));
            }
            __syncthreads();
        }
#pragma unroll 8
        for (int r = ty; r < n; r += kKeptThreads / 16) {
            const float4 x = *reinterpret_cast<const float4*>(scores + (b + r) * wide);
            const float ls = nlse[r];
            sum.x += ex2(x.x + ls), sum.y += ex2(x.y + ls), sum.z += ex2(x.z + ls), sum.w += ex2(x.w + ls);
        }
        __syncthreads();
        if (tx % 8 == 0)
            for (int r = ty; r < n; r += kKeptThreads / 16)
                asm volatile("discard.global.L2 [%0], 128;" ::"l"(scores + (b + r) * wide) : "memory");
    }
    part[threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.x < FT) {
        const float* of = reinterpret_cast<const float*>(part) + threadIdx.x;
        float v = 0.f;
#pragma unroll
        for (int i = 0; i < kKeptThreads / 16; ++i) v += of[i * FT];
        sums[threadIdx.x] = v;
    }
    if (C > 1) tc::cluster_sync();
    if (rank == 0 && threadIdx.x < FT && kt * FT + (int)threadIdx.x < a.kv_len) {
        float v = sums[threadIdx.x];
        for (int k = 1; k < C; ++k) {
            float u;
            asm volatile("ld.shared::cluster.f32 %0, [%1];"
                         : "=f"(u)
                         : "r"(tc::peer_of(&sums[threadIdx.x], k))
                         : "memory");
            v += u;
        }
        float* out = a.acc + (int64_t)h * a.acc_stride + kt * FT + threadIdx.x;
        *out = a.accumulate ? *out + v : v;
    }
    if (C > 1) tc::cluster_sync();  // nobody reads this CTA's sums any more
}

// ---------------------------------------------------------------- host side --
size_t up16(size_t n) { return (n + 15) & ~(size_t)15; }

// Workspace layouts; they return the bytes (SIZE_MAX: more rows than 32 bits
// count).
size_t plan_f32(int32_t kv_len, int32_t rows, int32_t n_head, int32_t n_head_kv, char* ws, F32Plan* p) {
    const int64_t n_rows = (int64_t)rows * (n_head / n_head_kv);
    if (n_rows > INT_MAX - FT) return SIZE_MAX;
    p->n_rows = (int32_t)n_rows;
    p->n_rt = (p->n_rows + FT - 1) / FT;
    p->n_kt = (kv_len + FT - 1) / FT;
    // two CTAs fit an SM: split the keys until the device is full
    const int64_t ctas = (int64_t)n_head_kv * p->n_rt;
    p->splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>(p->n_kt, 2 * kSms / ctas));
    const size_t n = (size_t)n_head_kv * p->n_rt * FT, ml = up16(n * p->splits * sizeof(float2));
    p->ml = reinterpret_cast<float2*>(ws);
    if ((int64_t)n * p->n_kt * FT <= kKeptScores) {  // whole lines of 128 bytes
        p->scores = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(ws + ml) + 127) & ~(uintptr_t)127);
        p->r_splits = 1;
        while (p->r_splits < 8 && p->n_rows >= 64 * p->r_splits &&
               (int64_t)n_head_kv * p->n_kt * p->r_splits * 2 <= kKeptCtas)
            p->r_splits *= 2;
        return ml + n * p->n_kt * FT * sizeof(float) + 112;
    }
    p->nlse = reinterpret_cast<float*>(ws + ml);
    // few key tiles and many rows: split the rows of the sums pass too
    p->r_splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>(p->n_rt / 2, 2 * kSms / ((int64_t)n_head_kv * p->n_kt)));
    const size_t lse = up16(n * sizeof(float));
    p->part = reinterpret_cast<float*>(ws + ml + lse);
    return ml + lse + (p->r_splits > 1 ? up16((size_t)p->r_splits * n_head_kv * p->n_kt * FT * sizeof(float)) : 0);
}

constexpr int64_t kPartSums = 16 << 20;  // sums of all parts, at most

size_t plan_tc(int32_t kv_len, int32_t rows, int32_t n_head, int32_t n_head_kv, int32_t d, char* ws, WeightPlan* p) {
    const int slots = d == 128 ? TcLayout<128>::kSlots : TcLayout<64>::kSlots;
    p->T = BM / (n_head / n_head_kv);
    p->n_rt = (rows + p->T - 1) / p->T;
    if ((int64_t)p->n_rt * BM > INT_MAX) return SIZE_MAX;
    p->n_kt = (kv_len + BM - 1) / BM;
    // statistics pass: large groups load the keys less often; smaller ones where
    // they split into clearly fewer steps for a CTA (8192 keys, 29 query tiles of
    // 2 heads: groups of 3, 59.6 us against 61.4 with 4)
    int64_t best = INT64_MAX;
    for (int g = std::min<int>(kMaxGroup, p->n_rt); g > 0; --g) {
        const int groups = (p->n_rt + g - 1) / g;
        const int splits = (int)std::max<int64_t>(1, std::min<int64_t>(p->n_kt, kSms / ((int64_t)n_head_kv * groups)));
        const int64_t waves = ((int64_t)n_head_kv * groups * splits + kSms - 1) / kSms;
        const int64_t steps = waves * ((p->n_kt + splits - 1) / splits) * g;
        if (steps < best - best / 20) best = steps, p->group = g, p->n_groups = groups, p->splits = splits;
    }
    // sums pass: a CTA per key tile, the rows split too when there are few key
    // tiles and many rows
    p->r_splits = (int32_t)std::max<int64_t>(1, std::min<int64_t>(p->n_rt / 4, kSms / ((int64_t)n_head_kv * p->n_kt)));
    // Query tiles that leave two slots for keys stay on chip.  More of them are
    // split until they do (the split with the fewest steps for a CTA), as long
    // as the parts' sums stay small; else they stream, and two key tiles share
    // each query tile's load once there are enough key tiles to fill the
    // device that way.  (14 heads of 64, 512 rows over 8192 keys: 61 us split, 66
    // streaming; 32 heads of 128, 256 over 65536: 316 and 363.)
    auto tiles = [&](int r) { return (p->n_rt + r - 1) / r; };
    auto ctas = [&](int r) { return std::max(1, std::min(p->n_kt, kSms / (n_head_kv * r))); };
    if (const int least = tiles(slots - 2); tiles(p->r_splits) > slots - 2 &&
                                            (int64_t)least * n_head_kv * p->n_kt * BM <= kPartSums) {
        best = INT64_MAX;
        for (int r = least; r <= std::min(2 * least, least + 16) && (int64_t)r * n_head_kv * p->n_kt * BM <= kPartSums; ++r) {
            const int64_t waves = ((int64_t)n_head_kv * r * ctas(r) + kSms - 1) / kSms;
            const int64_t steps = waves * ((p->n_kt + ctas(r) - 1) / ctas(r)) * tiles(r);
            if (steps < best) best = steps, p->r_splits = r;
        }
    }
    p->resident = tiles(p->r_splits) <= slots - 2;
    p->q_slots = p->resident ? tiles(p->r_splits) : slots / 2;
    p->k_slots = slots - p->q_slots;
    p->kg = !p->resident && (int64_t)n_head_kv * p->n_kt >= 2 * kSms ? 2 : 1;
    const int n_kg = (p->n_kt + p->kg - 1) / p->kg;
    p->b_splits = std::max(1, std::min(n_kg, kSms / (n_head_kv * p->r_splits)));
    const size_t n = (size_t)n_head_kv * p->n_rt * BM, ml = up16(n * p->splits * sizeof(float2));
    const size_t lse = up16(n * sizeof(float));
    p->ml = reinterpret_cast<float2*>(ws);
    p->nlse = reinterpret_cast<float*>(ws + ml);
    p->part = reinterpret_cast<float*>(ws + ml + lse);
    return ml + lse + (p->r_splits > 1 ? up16((size_t)p->r_splits * n_head_kv * p->n_kt * BM * sizeof(float)) : 0);
}

// A launch that may start before what precedes it on the stream has ended (the
// kernels wait for it on the device).
template <class... P, class... A>
cudaError_t launch_after(void (*k)(P...), int64_t grid, int heads, int threads, int smem, cudaStream_t s, int cluster,
                         const A&... args) {
    if (grid < 1 || grid > INT_MAX) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)grid, heads);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, k, args...);
}

// Dynamic shared memory of a kernel, set once per device (`mask`: a bit per
// device ordinal < 32).
cudaError_t allow_smem(const void* f, int bytes, std::atomic<unsigned>& mask) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 32 && (mask.load(std::memory_order_acquire) & (1u << dev))) return cudaSuccess;
    const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess && dev < 32) mask.fetch_or(1u << dev, std::memory_order_release);
    return e;
}

template <int D>
cudaError_t launch_f32(const WeightArgs& a, cudaStream_t s) {
    F32Plan p{};
    plan_f32(a.kv_len, a.n_tok - a.row_begin, a.n_head, a.n_head_kv, static_cast<char*>(a.ws), &p);
    const int smem = 2 * FT * (D + 4) * (int)sizeof(float);
    static std::atomic<unsigned> m0{0}, m1{0};
    cudaError_t e = allow_smem(reinterpret_cast<const void*>(&k7_stats_f32<D>), smem, m0);
    if (e == cudaSuccess) e = allow_smem(reinterpret_cast<const void*>(&k7_sums_f32<D>), smem, m1);
    if (e != cudaSuccess) return e;
    const int64_t K = a.n_head_kv, rows = K * p.n_rt * FT;
    e = launch_after(k7_stats_f32<D>, K * p.n_rt * p.splits, 1, kF32Threads, smem, s, 1, a, p);
    if (e == cudaSuccess && p.scores != nullptr)
        return launch_after(k7_kept_f32, K * p.n_kt * p.r_splits, 1, kKeptThreads, 0, s, p.r_splits, a, p);
    if (e == cudaSuccess) e = launch_after(k7_join_f32, rows / (kJoinThreads / 16), 1, kJoinThreads, 0, s, 1, a, p);
    if (e == cudaSuccess) e = launch_after(k7_sums_f32<D>, K * p.n_kt * p.r_splits, 1, kF32Threads, smem, s, 1, a, p);
    if (e != cudaSuccess || p.r_splits == 1) return e;
    return launch_after(k7_add, (a.kv_len + kJoinThreads - 1) / kJoinThreads, a.n_head_kv, kJoinThreads, 0, s, 1, a,
                        (const float*)p.part, p.n_kt * FT, p.r_splits, 0, 0);
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

// [rows][heads][d] 16-bit elements in boxes of box_rows x box_heads x 64.
bool make_map(CUtensorMap* m, const void* base, bool bf16, int d, int heads, int rows, int box_heads, int box_rows) {
    auto enc = get_encode();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {(cuuint64_t)d * 2, (cuuint64_t)d * 2 * heads};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_rows};
    const cuuint32_t estr[3] = {1, 1, 1};
    return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base),
               dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool BF16, int D, int SEG>
cudaError_t launch_tc(const WeightArgs& a, cudaStream_t s) {
    WeightPlan p{};
    plan_tc(a.kv_len, a.n_tok - a.row_begin, a.n_head, a.n_head_kv, D, static_cast<char*>(a.ws), &p);
    CUtensorMap mq, mk;
    const int rows = a.paging.block_rows > 0 ? a.paging.pool_rows : a.kv_len;
    if (!make_map(&mq, a.q, BF16, D, a.n_head, a.n_tok, a.n_head / a.n_head_kv, p.T) ||
        !make_map(&mk, a.k, BF16, D, a.n_head_kv, rows, 1, SEG))
        return cudaErrorInvalidValue;
    const int smem = TcLayout<D>::kBytes + 1024;
    static std::atomic<unsigned> m0{0}, m1{0}, m2{0};
    cudaError_t e = allow_smem(reinterpret_cast<const void*>(&k7_pass<BF16, D, SEG, 0, false>), smem, m0);
    if (e == cudaSuccess) e = allow_smem(reinterpret_cast<const void*>(&k7_pass<BF16, D, SEG, 1, false>), smem, m1);
    if (e == cudaSuccess) e = allow_smem(reinterpret_cast<const void*>(&k7_pass<BF16, D, SEG, 1, true>), smem, m2);
    if (e != cudaSuccess) return e;
    const int64_t K = a.n_head_kv;
    e = launch_after(k7_pass<BF16, D, SEG, 0, false>, K * p.n_groups * p.splits, 1, kTcThreads, smem, s, 1, mq, mk, a, p);
    if (e == cudaSuccess) e = launch_after(k7_join, K * p.n_rt * BM / (kJoinThreads / 16), 1, kJoinThreads, 0, s, 1, a, p);
    if (e == cudaSuccess)
        e = launch_after(p.resident ? k7_pass<BF16, D, SEG, 1, false> : k7_pass<BF16, D, SEG, 1, true>,
                         K * p.b_splits * p.r_splits, 1, kTcThreads, smem, s, 1, mq, mk, a, p);
    if (e != cudaSuccess || p.r_splits == 1) return e;
    return launch_after(k7_add, (a.kv_len + kJoinThreads - 1) / kJoinThreads, a.n_head_kv, kJoinThreads, 0, s, 1, a,
                        (const float*)p.part, p.n_kt * BM, p.r_splits, p.T, p.n_rt);
}

template <bool BF16, int D>
cudaError_t launch_seg(const WeightArgs& a, cudaStream_t s) {
    switch (a.page_size) {
        case 32: return launch_tc<BF16, D, 32>(a, s);
        case 64: return launch_tc<BF16, D, 64>(a, s);
        default: return launch_tc<BF16, D, 128>(a, s);
    }
}

}  // namespace

size_t weights_ws_bytes(int32_t kv_len, int32_t rows, int32_t n_head, int32_t n_head_kv, int32_t head_dim,
                        int32_t dtype) {
    if (dtype == 0) {
        F32Plan p{};
        return plan_f32(kv_len, rows, n_head, n_head_kv, nullptr, &p);
    }
    WeightPlan p{};
    return plan_tc(kv_len, rows, n_head, n_head_kv, head_dim, nullptr, &p);
}

cudaError_t launch_prompt_weights(const WeightArgs& a, cudaStream_t s) {
    const bool wide = a.head_dim == 128;
    switch (a.dtype) {
        case 0: return wide ? launch_f32<128>(a, s) : launch_f32<64>(a, s);
        case 1: return wide ? launch_seg<false, 128>(a, s) : launch_seg<false, 64>(a, s);
        default: return wide ? launch_seg<true, 128>(a, s) : launch_seg<true, 64>(a, s);
    }
}

}  // namespace epsp
