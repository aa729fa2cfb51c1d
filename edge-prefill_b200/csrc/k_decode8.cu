// k_decode8.cu -- K10: attention of one new token per sequence over a cache in
// 8 bits (bytes kq, vq with a scale ks, vs per page and KV head).
//
//   x_j = q . kq_j ks * scale,  out = sum_j exp(x_j - m) vq_j vs / sum_j exp(x_j - m)
//
// Half the bytes of K6, and they bound it; the split of the rows over the CTAs,
// the ring and the joins are K6's (decode_common.cuh).  A new token's row is
// quantised into the cache by k9_append first.
//
// CTA: units (32 rows of one head, so one scale each of K and V) go round robin
// to the streams of 8 warps, each with its own online softmax over 8 query heads
// (groups of more than 8 heads give a unit to 2, 4 or 8 warps).  A stream has
// its own stages and fetches for itself: K and V by TMA, the two scales by
// cp.async on the same barrier.
//
// S = Q K^T and O = P V on mma.sync m16n8k16 in f16, which holds both 8-bit
// types exactly.  The order of the contracted dimension is free, so a lane
// takes 16 neighbouring bytes of a K row (its fragments of four steps) and the
// bytes of one column block of V from the rows it needs: 16-byte reads without
// a transpose, and one byte permutation pairs two rows of V.  q is scaled to a
// largest magnitude of 2^14 to 2^15 by a power of two, so f16 takes its 16-bit
// types as they are; an f32 q has its rounding remainder (times 2^12) in rows
// 8-15.  P is the weight times V's scale, against the running maximum of just
// that, so that units of other scales add up in the accumulators as they are;
// the weights' sum takes P over the scale.  P is held 2^7 up (2^15 at most);
// rows 8-15 of its operand carry its rounding remainder, times 2^12: an element
// keeps 22 bits of itself and an absolute 2^-44 of the largest.
#include <cuda.h>
#include <cudaTypedefs.h>
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

constexpr int kWarps8 = 8;
constexpr int kThreads8 = kWarps8 * 32;
constexpr float kUp8 = 7.f;       // P is 2^7 times the weight against the running maximum (2^15 at most)
constexpr float kLow8 = 4096.f;   // factor of a remainder
constexpr int kPass8 = 64;        // query heads of a pass, at most

template <int D>
struct Layout8 {
    static constexpr int kHalf = kUnit * D;      // K (or V) of a unit
    static constexpr int kStage = 2 * kHalf;
    static constexpr int kStages = 131072 / kStage;  // dealt to the streams in equal parts
    static constexpr int kOffQ = kStages * kStage;   // [2] queries of a segment
    static constexpr int kQBytes = 16384;
    static constexpr int kOffO = kOffQ + 2 * kQBytes;  // [kWarps8][8][D] merge buffer
    static constexpr int kOffMl = kOffO + kWarps8 * 8 * D * 4;
    static constexpr int kOffScale = kOffMl + 2 * kWarps8 * 8 * 8;  // [kStages] (ks, vs)
    static constexpr int kOffBar = kOffScale + kStages * 8;
    static constexpr int kOffLens = kOffBar + (2 * kStages + 2) * 8;
    static constexpr int kBytes = kOffLens + kLensOnChip * 4;
    static_assert(kStages % kWarps8 == 0 && kBytes + 1024 <= 232448, "shared memory");
};

// Byte of row r, 16-byte chunk ch, in a swizzled tile of rows of D bytes.
template <int D>
__device__ __forceinline__ uint32_t tile_at(int r, int ch) {
    return D == 128 ? r * 128 + ((ch ^ (r & 7)) << 4) : r * 64 + ((ch ^ ((r >> 1) & 3)) << 4);
}

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) { return __byte_perm(a, b, sel); }

// Bytes (0, 1) and (2, 3) of w as two pairs of f16.
template <bool I8>
__device__ __forceinline__ void pairs8(uint32_t w, uint32_t& p01, uint32_t& p23) {
    if constexpr (I8) {
        // b ^ 0x80 is b + 128; as the low bits of 0x64.. it is 1024 + 128 + b
        const uint32_t u = w ^ 0x80808080u, off = 0x64806480u;  // 1152
        const uint32_t x = prmt(u, 0x64646464u, 0x4140), y = prmt(u, 0x64646464u, 0x4342);
        const __half2 o = *reinterpret_cast<const __half2*>(&off);
        const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&x), o), b = __hsub2(*reinterpret_cast<const __half2*>(&y), o);
        p01 = *reinterpret_cast<const uint32_t*>(&a);
        p23 = *reinterpret_cast<const uint32_t*>(&b);
    } else {
        asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
            : "=r"(p01), "=r"(p23)
            : "r"(w));
    }
}

// D += A B in f16 with f32 sums.  (Not volatile: the products may be put in any
// order that keeps each sum's.)
__device__ __forceinline__ void mma8(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                     uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// D = A B.
__device__ __forceinline__ void mma8_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                           uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// Four neighbouring query elements.
__device__ __forceinline__ float4 q_of(const unsigned char* q, int32_t dtype, int i) {
    if (dtype == 0) return *reinterpret_cast<const float4*>(q + i * 4);
    const uint2 w = *reinterpret_cast<const uint2*>(q + i * 2);
    if (dtype == 1) {
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
        return make_float4(a.x, a.y, b.x, b.y);
    }
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xffff0000u));
}

// Units of a block, and the place of a unit: dividing by a number that is known
// at run time only costs forty instructions, by its reciprocal five.
struct Blocks {
    int32_t units;   // of a block; 0: no blocks
    uint32_t inverse;
    __device__ __forceinline__ explicit Blocks(int block_rows) {
        units = block_rows / kUnit;
        inverse = units > 0 ? 0xffffffffu / (uint32_t)units : 0;
    }
    // Block of unit u (under 2^26), and the unit's place in it.  The product is
    // short of u / units by less than 2^-5.
    __device__ __forceinline__ int2 of(int u) const {
        int q = (int)__umulhi((uint32_t)u, inverse), r = u - q * units;
        if (r >= units) ++q, r -= units;
        return make_int2(q, r);
    }
};

// What a stream of warps fetches next: the units of the CTA's range that fall to
// it, one segment after the other.
struct Fetch {
    Walk w;          // the segment
    int32_t h;       // its KV head
    int32_t before;  // units of the CTA's range before it
    int32_t at;      // the unit, counted from the range's start
    int32_t place;   // of the unit in its block
    int32_t entry;   // its table entry, on its way

    __device__ __forceinline__ bool more() const { return w.left > 0; }
    // To the segment that holds unit `at`, and for its table entry.
    __device__ __forceinline__ void find(const DecodeArgs& a, const Blocks& bl, const Lens& lens, int runs, int passes) {
        while (w.left > 0 && at - before >= w.segment()) {
            before += w.segment();
            w.advance(a, lens, runs, w.segment());
            h = w.run / passes;
        }
        if (w.left <= 0 || bl.units == 0) return;
        const int2 b = bl.of(w.u + at - before);
        place = b.y;
        entry = a.kv.tables[(int64_t)w.s * a.kv.table_stride + b.x];
    }
    // Cache row of the unit; the tensors' row count (zeros are read there) for a
    // table entry outside the pool, which is recorded.
    __device__ __forceinline__ int row(const DecodeArgs& a, const Blocks& bl) const {
        if (bl.units == 0) return w.s * a.kv.seq_rows + (w.u + at - before) * kUnit;
        const int64_t x = (int64_t)entry * a.kv.block_rows + place * kUnit;
        if (entry >= 0 && x < a.kv.rows) return (int)x;
        report_error(a.err, kDevBadBlockTable, 0x95, w.s);
        return a.kv.rows;
    }
};

// LO: q has remainders (f32).  JOIN: the calls that join_cluster finishes.
template <int D, bool I8, bool LO, bool JOIN>
__global__ void __launch_bounds__(kThreads8, 1)
    k10_decode8(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const DecodeArgs a,
                const Cache8 c8, const DecodeSplit sp) {
    using LY = Layout8<D>;
    constexpr int kSteps = D / 16, kCols = D / 8;  // steps of a score, columns (of 8 lanes) of an output
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + LY::kOffBar);
    uint64_t* empty = full + LY::kStages;
    uint64_t* q_full = empty + LY::kStages;
    int32_t* lens_s = reinterpret_cast<int32_t*>(smem + LY::kOffLens);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int Hkv = a.n_head_kv, G = a.n_head / Hkv, es = a.dtype == 0 ? 4 : 2;
    const int runs = Hkv * sp.passes;

    if (threadIdx.x == 0) {
        for (int i = 0; i < LY::kStages; ++i) {
            tc::mbar_init(&full[i], 2);  // the bytes' announcement, and the scales
            tc::mbar_init(&empty[i], sp.groups);
        }
        for (int i = 0; i < 2; ++i) tc::mbar_init(&q_full[i], 1);
        tc::fence_mbar_init();
        tc::tma_prefetch_desc(&tmK);
        tc::tma_prefetch_desc(&tmV);
    }
    tc::pdl_wait();
    tc::pdl_launch();

    // ----------------------------------------- this CTA's range of the units
    Walk w0;
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
            for (int s = threadIdx.x; s < a.kv.n_seq; s += kThreads8) lens_s[s] = batch_len(a.kv, s, a.err);
            lens.chip = lens_s;
        }
        __syncthreads();
        w0 = share_of(a, sp, lens, runs, lane);
        // sequences without rows, dealt out to the CTAs
        for (int s = blockIdx.x; s < a.kv.n_seq; s += gridDim.x)
            if (lens.at(a, s) == 0) {
                for (int i = threadIdx.x; i < a.n_head * (D / 4); i += kThreads8)
                    store4(a.out, a.out_dtype, (int64_t)s * a.n_head * D + i * 4, make_float4(0.f, 0.f, 0.f, 0.f));
                if (sp.by_run)
                    for (int i = threadIdx.x; i < runs; i += kThreads8) sp.cut[s * runs + i] = make_int4(-1, 0, 0, 0);
            }
        if (w0.left <= 0 && !sp.by_run && threadIdx.x == 0) sp.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
    }
    // (a cluster's CTAs meet whatever their lengths)
    if (w0.left <= 0 && C == 1) {
        if (sp.direct) {  // a sequence without rows
            const int g0 = (w0.run % sp.passes) * sp.pass_heads, n = min(sp.pass_heads, G - g0) * (D / 4);
            const int64_t at = ((int64_t)w0.s * a.n_head + (w0.run / sp.passes) * G + g0) * D;
            for (int i = threadIdx.x; i < n; i += kThreads8)
                store4(a.out, a.out_dtype, at + i * 4, make_float4(0.f, 0.f, 0.f, 0.f));
        }
        return;
    }
    const uint64_t tmo = a.timeout_ns;
    float2* scale_s = reinterpret_cast<float2*>(smem + LY::kOffScale);

    const int groups = sp.groups, streams = kWarps8 / groups;
    const int grp = warp & (groups - 1), stream = warp / groups;
    // this stream's stages
    const int lg_depth = __ffs(LY::kStages / kWarps8 * groups) - 1, depth = 1 << lg_depth, st0 = stream << lg_depth;
    const Blocks blocks(a.kv.block_rows);
    const uint64_t policy = tc::policy_evict_first();               // the cache is read once
    const int lg_page = __ffs(c8.page_size) - 1;
    bool ok = true;

    // The stream's first warp fetches for it, a stage as soon as its warps are
    // done with it: eight warps issue copies, which one alone does at no more
    // than 5.2 TB/s (over all SMs, 8 KB units).
    Fetch f{w0, w0.run / sp.passes, 0, stream, 0, 0};
    int fetched = 0;
    if (grp == 0) f.find(a, blocks, lens, runs, sp.passes);
    auto fetch = [&]() {
        const Fetch x = f;
        f.at += streams;
        f.find(a, blocks, lens, runs, sp.passes);  // (the next entry is on its way while this one's copies are issued)
        const int st = st0 + (fetched & (depth - 1)), r = x.row(a, blocks);
        if (groups > 1) {
            ok = ok && __all_sync(0xffffffffu, tc::mbar_wait(&empty[st], ((fetched >> lg_depth) & 1) ^ 1, tmo));
            if (!ok) return;
        }
        ++fetched;
        if (lane == 0) {
            tc::mbar_arrive_expect_tx(&full[st], LY::kStage);
            unsigned char* base = smem + st * LY::kStage;
            tc::tma_load_3d(base, &tmK, &full[st], 0, x.h, r, policy);
            tc::tma_load_3d(base + LY::kHalf, &tmV, &full[st], 0, x.h, r, policy);
            if (r < a.kv.rows) {
                const int64_t page = (int64_t)(r >> lg_page) * Hkv + x.h;
                tc::copy4_async(&scale_s[st].x, c8.k_scale + page);
                tc::copy4_async(&scale_s[st].y, c8.v_scale + page);
                tc::copies_arrive(&full[st]);
            } else {
                scale_s[st] = make_float2(0.f, 1.f);
                tc::mbar_arrive(&full[st]);
            }
        }
        __syncwarp();
    };
    // The queries of segment n_q, by thread 0, while the segment before is
    // attended (its buffer's readers met at the end of the one before that).
    Walk wq = w0;
    int n_q = 0;
    auto fetch_q = [&]() {
        if (threadIdx.x == 0 && (wq.left > 0 || (C > 1 && n_q == 0))) {
            const int h = wq.run / sp.passes, pass = wq.run % sp.passes, b = n_q & 1;
            const uint32_t bytes = min(sp.pass_heads, G - pass * sp.pass_heads) * D * es;
            tc::mbar_arrive_expect_tx(&q_full[b], bytes);
            tc::bulk_load(smem + LY::kOffQ + b * LY::kQBytes,
                          static_cast<const char*>(a.q) +
                              ((int64_t)wq.s * a.n_head + (int64_t)h * G + pass * sp.pass_heads) * D * es,
                          bytes, &q_full[b]);
            ++n_q;
            if (wq.left > 0) wq.advance(a, lens, runs, wq.segment());
        }
    };
    fetch_q();
    for (int i = 0; i < depth && grp == 0 && f.more(); ++i) fetch();

    float* om = reinterpret_cast<float*>(smem + LY::kOffO);
    float* om_w = om + warp * 8 * D;
    Walk w = w0;
    int it = 0, used = 0;  // units of the range before the segment; units that this warp is done with
    for (int seg = 0; w.left > 0 || (C > 1 && seg == 0); ++seg) {
        const int n_seg = w.segment();
        const int h = w.run / sp.passes, pass = w.run % sp.passes;
        const int g0 = pass * sp.pass_heads + grp * 8;  // this warp's first query head of the group
        const int64_t q_row = (int64_t)w.s * a.n_head + (int64_t)h * G;
        fetch_q();
        const int hd = lane >> 2, tq = lane & 3;  // this lane's head (or column block of V) and quarter
        // head hd, columns kCols (2 tq + e) + j: the sum over P at [j][e], over its remainders at [j][2 + e]
        float o[kCols][4];
#pragma unroll
        for (int j = 0; j < kCols; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
        float m = -INFINITY, l = 0.f;
        if (ok) {
            ok = __all_sync(0xffffffffu, tc::mbar_wait(&q_full[seg & 1], (seg >> 1) & 1, tmo));
            if (!ok && lane == 0) report_error(a.err, kDevWaitDecode, 0xb3, seg);
        }
        // q in f16, dims D / 4 tq + 4 j + {0, 1, 2, 3} for step j
        uint32_t qh[2 * kSteps], ql[LO ? 2 * kSteps : 1];
        float sl;
        {
            const unsigned char* qs = smem + LY::kOffQ + (seg & 1) * LY::kQBytes + (grp * 8 + hd) * D * es;
            float4 x[kSteps];
            float top = 0.f;
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
                x[j] = g0 + hd < G ? q_of(qs, a.dtype, D / 4 * tq + 4 * j) : make_float4(0.f, 0.f, 0.f, 0.f);
                top = fmaxf(fmaxf(fmaxf(fabsf(x[j].x), fabsf(x[j].y)), fmaxf(fabsf(x[j].z), fabsf(x[j].w))), top);
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int e = (int)(__float_as_uint(top) >> 23) - 127;
            const int up = e < 128 ? min(14 - e, 126) : 0;  // (at least -113)
            const float f = __uint_as_float((uint32_t)(up + 127) << 23);
            sl = a.kq_scale * kLog2e * __uint_as_float((uint32_t)(127 - up) << 23);
#pragma unroll
            for (int j = 0; j < kSteps; ++j) {
                x[j].x *= f, x[j].y *= f, x[j].z *= f, x[j].w *= f;
                qh[2 * j] = split2<false>(x[j].x, x[j].y);
                qh[2 * j + 1] = split2<false>(x[j].z, x[j].w);
                if constexpr (LO) {
                    x[j].x *= kLow8, x[j].y *= kLow8, x[j].z *= kLow8, x[j].w *= kLow8;
                    ql[2 * j] = split2<false>(x[j].x, x[j].y);
                    ql[2 * j + 1] = split2<false>(x[j].z, x[j].w);
                }
            }
        }
        // first unit of the segment that falls to this stream
        int i = (stream - it) & (streams - 1);
        for (; i < n_seg; i += streams) {
            const int st = st0 + (used & (depth - 1));
            if (ok) {
                ok = __all_sync(0xffffffffu, tc::mbar_wait(&full[st], (used >> lg_depth) & 1, tmo));
                if (!ok && lane == 0) report_error(a.err, kDevWaitDecode, 0xb2, it + i);
            }
            if (!ok) break;
            ++used;
            unsigned char* stage = smem + st * LY::kStage;
            const int u = w.u + i, lim = min(kUnit, w.n - u * kUnit);
            const unsigned char* vb = stage + LY::kHalf;
            if (!I8 && lim < kUnit) {
                // V rows past the length may hold NaN codes: their P is 0, and 0 * NaN is not 0
                for (int j = lane; j < (kUnit - lim) * (D / 16); j += 32)
                    *reinterpret_cast<uint4*>(stage + LY::kHalf + lim * D + j * 16) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // TMA writes the stage next
                __syncwarp();
            }
            const float2 sc = scale_s[st];
            // (the four tiles of keys in turn: each one's products wait for one another)
            float s4[4][4];
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                uint4 b[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) b[t] = *reinterpret_cast<const uint4*>(stage + tile_at<D>(t * 8 + hd, (D / 64) * tq + c));
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const int j = 4 * c + e;
                        uint32_t b0, b1;
                        pairs8<I8>(e == 0 ? b[t].x : e == 1 ? b[t].y : e == 2 ? b[t].z : b[t].w, b0, b1);
                        const uint32_t a1 = LO ? ql[LO ? 2 * j : 0] : 0u, a3 = LO ? ql[LO ? 2 * j + 1 : 0] : 0u;
                        if (j == 0) mma8_first(s4[t], qh[0], a1, qh[1], a3, b0, b1);
                        else mma8(s4[t], qh[2 * j], a1, qh[2 * j + 1], a3, b0, b1);
                    }
            }
            // log2 of the weight times V's scale: that is what O is the sum of
            const float slk = sl * sc.x, lv = __log2f(sc.y);
            float mx = -INFINITY;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    if constexpr (LO) s4[t][e] = fmaf(s4[t][e + 2], 1.f / kLow8, s4[t][e]);
                    s4[t][e] = t * 8 + 2 * tq + e < lim ? fmaf(s4[t][e], slk, lv) : -INFINITY;
                    mx = fmaxf(mx, s4[t][e]);
                }
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            // the running maximum follows when it is 2^8 behind
            const bool need = mx > m + (8.f + kUp8);
            if (__any_sync(0xffffffffu, need)) {
                const float alpha = need ? ex2(m - (mx - kUp8)) : 1.f;
                if (need) m = mx - kUp8;
                l *= alpha;
#pragma unroll
                for (int j = 0; j < kCols; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[j][e] *= alpha;
            }
            const float ms = m == -INFINITY ? 0.f : m;
            uint32_t p[2][4];
            float sum = 0.f;
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    float x = ex2(s4[2 * b + t][0] - ms), y = ex2(s4[2 * b + t][1] - ms);
                    sum += x + y;
                    p[b][2 * t] = split2<false>(x, y);
                    x *= kLow8, y *= kLow8;
                    p[b][2 * t + 1] = split2<false>(x, y);
                }
            l = fmaf(sum, ex2(-lv), l);  // (the weights alone)
            // rows 16 b + 8 t + 2 tq + {0, 1} of V, D / 8 columns from D / 8 hd
            uint32_t v[2][2][2][D / 32];
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int r = 16 * b + 8 * t + 2 * tq + e;
                        if constexpr (D == 128) {
                            const uint4 x = *reinterpret_cast<const uint4*>(vb + tile_at<D>(r, hd));
                            v[b][t][e][0] = x.x, v[b][t][e][1] = x.y, v[b][t][e][2] = x.z, v[b][t][e][3] = x.w;
                        } else {
                            const uint2 x = *reinterpret_cast<const uint2*>(vb + tile_at<D>(r, hd >> 1) + (hd & 1) * 8);
                            v[b][t][e][0] = x.x, v[b][t][e][1] = x.y;
                        }
                    }
#pragma unroll
            for (int x = 0; x < D / 32; ++x)
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    uint32_t b0[4], b1[4];
                    pairs8<I8>(prmt(v[b][0][0][x], v[b][0][1][x], 0x5140), b0[0], b0[1]);
                    pairs8<I8>(prmt(v[b][0][0][x], v[b][0][1][x], 0x7362), b0[2], b0[3]);
                    pairs8<I8>(prmt(v[b][1][0][x], v[b][1][1][x], 0x5140), b1[0], b1[1]);
                    pairs8<I8>(prmt(v[b][1][0][x], v[b][1][1][x], 0x7362), b1[2], b1[3]);
#pragma unroll
                    for (int j = 0; j < 4; ++j) mma8(o[4 * x + j], p[b][0], p[b][1], p[b][2], p[b][3], b0[j], b1[j]);
                }
            __syncwarp();
            if (groups > 1 && lane == 0) tc::mbar_arrive(&empty[st]);
            if (grp == 0 && f.more()) fetch();
        }

        // ------------------------------------------- merge the warps' states
        // (ml alternates between two buffers: a warp may write the next
        // segment's before another has read this one's sums)
        float2* ml = reinterpret_cast<float2*>(smem + LY::kOffMl) + (seg & 1) * kWarps8 * 8;
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (tq == 0) ml[warp * 8 + hd] = make_float2(m, l);
        tc::named_bar_sync(1, kWarps8 * 32);
        {
            // the streams' common maximum of this lane's head
            float mt = -INFINITY;
#pragma unroll
            for (int r = 0; r < kWarps8; ++r)
                if (r < streams) mt = fmaxf(mt, ml[(r * groups + grp) * 8 + hd].x);
            const float f = ex2(m - (mt == -INFINITY ? 0.f : mt));
            auto whole_sum = [](const float (&x)[4], int e) { return fmaf(x[2 + e], 1.f / kLow8, x[e]); };
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int j = 0; j < kCols; j += 4)
                    *reinterpret_cast<float4*>(om_w + hd * D + kCols * (2 * tq + e) + j) =
                        make_float4(whole_sum(o[j], e) * f, whole_sum(o[j + 1], e) * f, whole_sum(o[j + 2], e) * f,
                                    whole_sum(o[j + 3], e) * f);
        }
        tc::named_bar_sync(1, kWarps8 * 32);
        const bool whole = w.u == 0 && n_seg == w.units;
        const int n_heads = min(min(groups * 8, sp.pass_heads), G - pass * sp.pass_heads);
        const int slot = blockIdx.x * 2 + (seg == 0 ? 0 : 1);
        for (int j = threadIdx.x; j < n_heads * (D / 4); j += kWarps8 * 32) {
            const int g = j / (D / 4), c = j % (D / 4), gw = g >> 3, gh = g & 7;
            float2 v[kWarps8];
            float4 t[kWarps8];
            float mt = -INFINITY;
#pragma unroll
            for (int r = 0; r < kWarps8; ++r)
                if (r < streams) {
                    const int wr = (r * groups + gw) * 8 + gh;
                    v[r] = ml[wr];
                    t[r] = *reinterpret_cast<const float4*>(om + wr * D + c * 4);
                    mt = fmaxf(mt, v[r].x);
                }
            const float ms = mt == -INFINITY ? 0.f : mt;
            float lt = 0.f;
            float4 ot = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int r = 0; r < kWarps8; ++r)
                if (r < streams) {
                    lt += v[r].y * ex2(v[r].x - ms);
                    ot.x += t[r].x, ot.y += t[r].y, ot.z += t[r].z, ot.w += t[r].w;
                }
            if constexpr (JOIN) {
                // (the ring: this CTA's last copy has landed)
                *reinterpret_cast<float4*>(smem + (g * D + c * 4) * 4) = ot;
                if (c == 0) *reinterpret_cast<float2*>(smem + kPass8 * D * 4 + g * 8) = make_float2(ms, lt);
            } else if (whole) {
                const float inv = 1.f / lt;
                store4(a.out, a.out_dtype, (q_row + pass * sp.pass_heads + g) * D + c * 4,
                       make_float4(ot.x * inv, ot.y * inv, ot.z * inv, ot.w * inv));
            } else {
                const int64_t p = (int64_t)slot * groups * 8 + g;
                *reinterpret_cast<float4*>(sp.part_o + p * D + c * 4) = ot;
                if (c == 0) sp.part_ml[p] = make_float2(ms, lt);
            }
        }
        if constexpr (JOIN) {
            join_cluster<D, kWarps8 * 32, kPass8>(a, sp, smem, om, w, n_seg, q_row + pass * sp.pass_heads, n_heads, h,
                                                  rank);
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
    if (!ok) {
        // copies still in flight land before the CTA ends
        if (lane == 0) report_error(a.err, kDevWaitDecode, 0xb1, used);
        for (int j = max(0, fetched - depth); j < fetched; ++j) tc::mbar_wait(&full[st0 + (j & (depth - 1))], (j >> lg_depth) & 1, tmo);
        for (int j = max(0, n_q - 2); j < n_q; ++j) tc::mbar_wait(&q_full[j & 1], (j >> 1) & 1, tmo);
    }
}

// ---------------------------------------------------------------- host side --
// Cache rows [rows][Hkv][d] of bytes in boxes of 32 rows of one head.
bool cache8_map(CUtensorMap* m, const void* base, int32_t d, int32_t n_head_kv, int32_t rows) {
    auto enc = get_encode();
    if (!enc) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)n_head_kv, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {(cuuint64_t)d, (cuuint64_t)d * n_head_kv};
    const cuuint32_t box[3] = {(cuuint32_t)d, 1, kUnit};
    const cuuint32_t estr[3] = {1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Split of a call and its workspace layout; returns the bytes (SIZE_MAX: more
// units than the 32-bit counts hold).
size_t split8_of(int32_t n_seq, int32_t max_kv_len, int32_t n_head, int32_t n_head_kv, int32_t d, int32_t dtype,
                 char* ws, DecodeSplit* sp) {
    const int G = n_head / n_head_kv;
    // (what the query buffer holds)
    sp->pass_heads = G <= 16 ? 16 : dtype == 0 ? 32 : 64;
    sp->heads = 8;
    sp->groups = 1;
    const int in_pass = std::min(G, sp->pass_heads);
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
        sp->direct = sp->cluster > 1 && units <= sp->cluster * 2 * kClusterUnits;
        if (!sp->direct) sp->cluster = 1;
    }
    const int64_t ctas = sp->direct ? all_runs * sp->cluster : (total + kMinUnits - 1) / kMinUnits;
    sp->ctas = (int32_t)std::min<int64_t>(ctas, kCtas);
    sp->by_run = !sp->direct && all_runs <= sp->ctas;
    sp->joins = sp->direct ? 0 : sp->by_run ? (int32_t)all_runs : sp->ctas;
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
    return at;
}

template <int D, bool I8, bool LO, bool JOIN>
cudaError_t launch8_join(DecodeArgs a, const Cache8& c, const DecodeSplit& sp, cudaStream_t s) {
    CUtensorMap mk, mv;
    if (!cache8_map(&mk, c.k, D, a.n_head_kv, a.kv.rows) || !cache8_map(&mv, c.v, D, a.n_head_kv, a.kv.rows))
        return cudaErrorInvalidValue;
    const int smem = Layout8<D>::kBytes + 1024;
    int dev = 0;
    cudaGetDevice(&dev);
    // one bit per device ordinal < 32 whose attribute is set
    static std::atomic<unsigned> set_mask{0};
    if (dev >= 32 || !(set_mask.load(std::memory_order_acquire) & (1u << dev))) {
        const cudaError_t e =
            cudaFuncSetAttribute(k10_decode8<D, I8, LO, JOIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev < 32) set_mask.fetch_or(1u << dev, std::memory_order_release);
    }
    // the kernels may start before what precedes them on the stream has ended:
    // they wait for it on the device
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
    cfg.blockDim = dim3(kThreads8);
    cfg.dynamicSmemBytes = smem;
    cfg.numAttrs = sp.cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, k10_decode8<D, I8, LO, JOIN>, mk, mv, a, c, sp);
    if (e != cudaSuccess || sp.direct) return e;
    const int heads = std::min(a.n_head / a.n_head_kv, sp.pass_heads);
    const int64_t grid = (int64_t)sp.joins * heads;
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k6b_join<D>, a, sp, heads, 0);
}

template <int D, bool I8>
cudaError_t launch8_t(const DecodeArgs& a, const Cache8& c, const DecodeSplit& sp, cudaStream_t s) {
    if (a.dtype == 0)
        return sp.cluster > 1 ? launch8_join<D, I8, true, true>(a, c, sp, s) : launch8_join<D, I8, true, false>(a, c, sp, s);
    return sp.cluster > 1 ? launch8_join<D, I8, false, true>(a, c, sp, s) : launch8_join<D, I8, false, false>(a, c, sp, s);
}

}  // namespace

size_t decode8_ws_bytes(int32_t n_seq, int32_t max_kv_len, int32_t n_head, int32_t n_head_kv, int32_t head_dim,
                        int32_t dtype) {
    DecodeSplit sp{};
    return split8_of(n_seq, max_kv_len, n_head, n_head_kv, head_dim, dtype, nullptr, &sp);
}

cudaError_t launch_decode8(const DecodeArgs& a, const Cache8& c, cudaStream_t s) {
    if (a.k_new) {
        const AppendArgs w{a.kv, a.k_new, a.v_new, c, a.dtype, a.n_head_kv, a.head_dim, a.err};
        const cudaError_t e = launch_append8(w, s);
        if (e != cudaSuccess) return e;
    }
    DecodeSplit sp{};
    split8_of(a.kv.n_seq, a.kv.max_kv_len, a.n_head, a.n_head_kv, a.head_dim, a.dtype, static_cast<char*>(a.ws), &sp);
    if (a.head_dim == 128) return c.i8 ? launch8_t<128, true>(a, c, sp, s) : launch8_t<128, false>(a, c, sp, s);
    return c.i8 ? launch8_t<64, true>(a, c, sp, s) : launch8_t<64, false>(a, c, sp, s);
}

}  // namespace epsp
