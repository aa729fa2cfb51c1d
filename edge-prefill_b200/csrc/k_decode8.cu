// k_decode8.cu -- K10: attention of one new token per sequence over a cache in
// 8 bits (bytes kq, vq with a scale ks, vs per page and KV head).
//
//   x_j = q . kq_j ks * scale,  out = sum_j exp(x_j - m) vq_j vs / sum_j exp(x_j - m)
//
// Half the bytes of K6; the split of the rows over the CTAs, the ring and the
// joins are K6's (decode_common.cuh).  64 K rows (8 heads of 128) take 33 us, 4.1
// TB/s, 64 sequences of up to 4096 rows 61, 4.4 TB/s; without the arithmetic 26 and
// 52: the bytes bound it first, then the attending warps, two a scheduler, whose
// products and conversions wait for one another (issue slots 35 to 47 % busy).  A
// new token's row is quantised into the cache by the CTA that attends it: the last
// page of a run is never split, and its copies wait for the row (as a kernel
// before, k9_append, it took 3 to 4 us more; calls of several passes still have
// that).
//
// CTA: units (32 rows of one head, so one scale each of K and V) go round robin
// to the streams of 8 warps, each with its own online softmax over 8 query heads
// (groups of more than 8 heads give a unit to 2, 4 or 8 warps).  A stream has
// its own stages; four more warps fetch, a lane for each stream: K and V by TMA,
// the two scales by cp.async on the same barrier.
//
// S^T = K Q^T and O^T = V^T P^T on mma.sync m16n8k16 in f16, which holds both
// 8-bit types exactly: keys, then columns of V, on the 16 side and 8 query heads
// on the other, so no row of the tensor work is empty and O takes 32 registers.
// The order of the contracted dimension is free, so a lane takes 16 neighbouring
// bytes of a K row (its fragments of four steps) and the bytes of one column
// block of V from the rows it needs: 16-byte reads without a transpose, and one
// byte permutation pairs two rows of V.  q is scaled to a
// largest magnitude of 2^14 to 2^15 by a power of two, so f16 takes its 16-bit
// types as they are; an f32 q is two f16 (a second product).  P is the weight
// times V's scale, so that units of any scales add up in the accumulators as they
// are.  Two running maxima, in whole powers of two: that of the scores, for the
// weights and their sum, and that of score and scale, for P; a unit's weights
// become P by one factor.  (Of the products alone, the sum would lose the weights
// of pages with small scales and the range of large ones; 1 to 2 % faster.)  The
// largest P is held between 2^14 and 2^15, and P is two f16: an element keeps 22
// bits of itself and an absolute 2^-39 of the largest (half of f16's smallest step).
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdint>
#include <type_traits>

// (in units of 32 rows of 8 bits; 64 sequences of up to 4096 rows: 6 71.5 us, 10
// 64.7, 14 61.0, 20 60.7; 64 K rows: 10 32.3, 14 32.4, 20 32.5)
#define EPSP_RUN_COST 14
#include "cache8.cuh"
#include "decode_common.cuh"
#include "epsp_kernels.h"
#include "tc100.cuh"

namespace epsp {
namespace {

constexpr int kWarps8 = 8;
constexpr int kThreads8 = kWarps8 * 32;  // that attend
constexpr int kFetchers = 4;             // warps that fetch
// Either maximum follows once something would pass 2^15: that of the weights to
// where the largest is 1 to 2, P's to where it is 2^14 to 2^15.
constexpr float kUp8 = 14.f;
constexpr float kMost8 = 15.f;
constexpr float kNone8 = -3.402823466e38f;  // either of no rows: a number, so that -inf lies below it
constexpr int kPass8 = 64;        // query heads of a pass, at most
// Units for each CTA of a cluster up to which a run is joined in shared memory
// instead of being split over the device: one launch. One sequence of 6000, 12,000,
// 16,000 and 24,000 rows, split 14.1, 16.3, 17.9 and 20.2 us, in clusters of 8 11.4,
// 15.6, 17.7 and 22.8 (32 heads on 8); split 13.5, 14.9, 16.1 and 17.8, in clusters
// 11.8, 16.4, 19.1 and 24.9 (28 on 4); f32, 14 on 2, split 11.8, 12.6, 14.4 and 13.9, in
// clusters 9.7, 13.0, 15.0 and 19.0.
constexpr int kClusterMost8 = 48;

// Shared memory: the stages, then what follows by offset.
template <int D>
struct Layout8 {
    static constexpr int kHalf = kUnit * D;      // K (or V) of a unit
    static constexpr int kStage = 2 * kHalf;
    static constexpr int kMost = 196608 / kStage;  // stages, at most
    int32_t stages;   // dealt to the streams as evenly as they go
    int32_t q_bytes;  // of a segment's queries: two buffers
    __host__ __device__ int off_q() const { return stages * kStage; }
    __host__ __device__ int off_o() const { return off_q() + 2 * q_bytes; }        // [kWarps8][8][D] the warps' sums
    __host__ __device__ int off_ml() const { return off_o() + kWarps8 * 8 * D * 4; }  // [kWarps8][8] (maximum, sum)
    __host__ __device__ int off_mp() const { return off_ml() + kWarps8 * 8 * 8; }     // [kWarps8][8] P's over it
    __host__ __device__ int off_scale() const { return off_mp() + kWarps8 * 8 * 4; }  // [stages] (ks, vs)
    __host__ __device__ int off_bar() const { return off_scale() + kMost * 8; }
    __host__ __device__ int off_lens() const { return off_bar() + (2 * kMost + 7) * 8; }
    __host__ __device__ int bytes() const { return off_lens() + kLensOnChip * 4; }
    // For `pass` query heads of `es` bytes: as many stages as 227 KB hold.
    static Layout8 make(int pass, int es) {
        Layout8 l;
        l.stages = 0;
        l.q_bytes = pass * D * es;
        l.stages = std::min(kMost, (232448 - 1024 - l.bytes()) / kStage);
        return l;
    }
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
// The 8 x 8 tile of 16-bit values (row lane / 4, columns 2 (lane % 4) + {0, 1}) turned over.
__device__ __forceinline__ uint32_t turned(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// D = A B.
__device__ __forceinline__ void mma8_first(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                           uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// 2^t of a whole t in [-126, 127].
__device__ __forceinline__ float pow2(float t) {
    return __uint_as_float((__float_as_uint(t + 12582912.f) << 23) + 0x3f800000u);  // (the sum's low bits are t)
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
            h = passes == 1 ? w.run : w.run / passes;
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

__device__ __forceinline__ void store2(void* out, int32_t dtype, int64_t i, float x, float y) {
    if (dtype == 0) {
        *reinterpret_cast<float2*>(static_cast<float*>(out) + i) = make_float2(x, y);
    } else if (dtype == 1) {
        *reinterpret_cast<__half2*>(static_cast<__half*>(out) + i) = __floats2half2_rn(x, y);
    } else {
        *reinterpret_cast<__nv_bfloat162*>(static_cast<__nv_bfloat16*>(out) + i) = __floats2bfloat162_rn(x, y);
    }
}

// A warp puts the new token's K and V row of one head into row n - 1 of the cache.
template <int D, bool I8>
__device__ __forceinline__ void append_row(const DecodeArgs& a, const Cache8& c, int s, int h, int n, int lane) {
    constexpr int E = D / 32;  // elements of a lane
    const int Hkv = a.n_head_kv, r0 = (n - 1) / c.page_size * c.page_size, lo = n - 1 - r0;
    const int row = held_back(a.kv, a.err) ? -1 : batch_row(a.kv, s, r0, a.err);
    float x[2][E], was[2];
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        const int64_t i = ((int64_t)s * Hkv + h) * D + lane * E;
        const void* src = v ? a.v_new : a.k_new;
#pragma unroll
        for (int e = 0; e < E; ++e)
            x[v][e] = a.dtype == 0   ? static_cast<const float*>(src)[i + e]
                      : a.dtype == 1 ? __half2float(static_cast<const __half*>(src)[i + e])
                                     : __bfloat162float(static_cast<const __nv_bfloat16*>(src)[i + e]);
        was[v] = row >= 0 && lo > 0 ? (v ? c.v_scale : c.k_scale)[(int64_t)(row / c.page_size) * Hkv + h] : 0.f;
    }
    if (row < 0) return;
#pragma unroll
    for (int v = 0; v < 2; ++v) {
        bool odd = false;
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) m = max(m, magnitude(x[v][e], odd));
        m = __reduce_max_sync(0xffffffffu, m);
        if (odd) report_error(a.err, kDevNotFinite8, 0x94, s);
        uint8_t* dst = (v ? c.v : c.k) + ((int64_t)row * Hkv + h) * D;
        float sc = scale8<I8>(m);
        if (was[v] >= sc) sc = was[v];
        else {
            if (lo > 0) rescale8<I8, 8>(dst, (int64_t)Hkv * D, lo, D, was[v], sc, lane, 32);
            if (lane == 0) (v ? c.v_scale : c.k_scale)[(int64_t)(row / c.page_size) * Hkv + h] = sc;
        }
        const float inv = exact_inverse(sc);
        float y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = tame8<I8>(over(x[v][e], sc, inv));
        const uint32_t q = to8<I8>(y[0], y[1], y[2], y[3]);
        uint8_t* to = dst + (int64_t)lo * Hkv * D + lane * E;
        if constexpr (E == 4) *reinterpret_cast<uint32_t*>(to) = q;
        else *reinterpret_cast<uint16_t*>(to) = (uint16_t)q;
    }
}

// LO: q has remainders (f32).  (P always has: where V's terms cancel, the 11 bits of
// one f16 show in a bf16 output too; 8 sequences of 16 to 32 K rows 47.1 us, with one
// f16 45.2.)  ADD: a unit's sums are added to the accumulators by f32 additions, which
// round, where the products themselves cut: for f32 outputs, which 20 units a warp
// would leave 8e-7 of themselves too small (3 sequences of 29,000 rows; 1.3e-7 with
// it), 256 units and V of one sign 9e-5.  16-bit outputs round off more than that, and
// would pay: batch 61.1 us without, 67.5 with it, 64 K rows 32.0 and 33.8.  JOIN: the
// calls that join_cluster finishes.
template <int D, bool I8, bool LO, bool ADD, bool JOIN>
__global__ void __launch_bounds__(kThreads8 + 32 * kFetchers, 1)
    k10_decode8(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const DecodeArgs a,
                const Cache8 c8, const DecodeSplit sp, const Layout8<D> ly) {
    using LY = Layout8<D>;
    constexpr int kAll = kThreads8 + 32 * kFetchers;
    constexpr int kSteps = D / 16, kCols = D / 8;  // steps of a score; columns of an output that a lane has
    extern __shared__ unsigned char smem_dyn[];
    unsigned char* smem = reinterpret_cast<unsigned char*>(((uintptr_t)smem_dyn + 1023) & ~(uintptr_t)1023);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + ly.off_bar());
    uint64_t* empty = full + LY::kMost;
    uint64_t* q_full = empty + LY::kMost;  // [2] queries are there, and every warp has read them
    uint64_t* q_empty = q_full + 2;
    uint64_t* written = q_empty + 2;       // the warps' sums of a segment are in shared memory,
    uint64_t* merged = written + 1;        // and out of it
    uint64_t* appended = merged + 1;       // the CTA's new rows are in the cache
    int32_t* lens_s = reinterpret_cast<int32_t*>(smem + ly.off_lens());
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int Hkv = a.n_head_kv, G = a.n_head / Hkv, es = a.dtype == 0 ? 4 : 2;
    const int runs = Hkv * sp.passes;

    if (threadIdx.x < ly.stages) {
        tc::mbar_init(&full[threadIdx.x], 2);  // the bytes' announcement, and the scales
        tc::mbar_init(&empty[threadIdx.x], sp.groups);
        tc::fence_mbar_init();
    }
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(&q_full[i], 1);
            tc::mbar_init(&q_empty[i], kWarps8);
        }
        tc::mbar_init(written, kWarps8);
        tc::mbar_init(merged, kWarps8);
        tc::mbar_init(appended, kWarps8);
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
    // the new rows are put into the cache by the CTAs that attend them
    const int lg_whole = a.k_new != nullptr ? __ffs(c8.page_size) - 1 : 0;
    if (JOIN || sp.direct) {
        const int id = blockIdx.x >> (__ffs(C) - 1);
        w0.s = id / runs;
        w0.run = id % runs;
        if (threadIdx.x == 0) lens_s[0] = batch_len(a.kv, w0.s, a.err);
        __syncthreads();
        w0.n = lens_s[0];
        w0.units = units_of(w0.n);
        const int per = (w0.units + C - 1) >> (__ffs(C) - 1);
        w0.whole = lg_whole;
        const int lp = w0.n > 0 ? w0.last_page() : 0;
        auto cut_at = [&](int r) { return r * per > lp ? w0.units : min(r * per, w0.units); };
        w0.u = cut_at(rank);
        w0.left = cut_at(rank + 1) - w0.u;
    } else {
        if (a.kv.n_seq <= kLensOnChip) {
            for (int s = threadIdx.x; s < a.kv.n_seq; s += kAll) lens_s[s] = batch_len(a.kv, s, a.err);
            lens.chip = lens_s;
        }
        __syncthreads();
        w0 = share_of(a, sp, lens, runs, lane);
        w0.whole = lg_whole;
        // (the CTA before has taken the rest of that page)
        if (w0.left > 0 && w0.u > 0 && w0.u > w0.last_page()) w0.advance(a, lens, runs, w0.units - w0.u);
        // sequences without rows, dealt out to the CTAs
        for (int s = blockIdx.x; s < a.kv.n_seq; s += gridDim.x)
            if (lens.at(a, s) == 0) {
                for (int i = threadIdx.x; i < a.n_head * (D / 4); i += kAll)
                    store4(a.out, a.out_dtype, (int64_t)s * a.n_head * D + i * 4, make_float4(0.f, 0.f, 0.f, 0.f));
                if (sp.by_run)
                    for (int i = threadIdx.x; i < runs; i += kAll) sp.cut[s * runs + i] = make_int4(-1, 0, 0, 0);
            }
        if (w0.left <= 0 && !sp.by_run && threadIdx.x == 0) sp.cut[blockIdx.x] = make_int4(-1, 0, 0, 0);
    }
    // (a cluster's CTAs meet whatever their lengths)
    if (w0.left <= 0 && C == 1) {
        if (sp.direct) {  // a sequence without rows
            const int g0 = (w0.run % sp.passes) * sp.pass_heads, n = min(sp.pass_heads, G - g0) * (D / 4);
            const int64_t at = ((int64_t)w0.s * a.n_head + (w0.run / sp.passes) * G + g0) * D;
            for (int i = threadIdx.x; i < n; i += kAll)
                store4(a.out, a.out_dtype, at + i * 4, make_float4(0.f, 0.f, 0.f, 0.f));
        }
        return;
    }
    const uint64_t tmo = a.timeout_ns;
    float2* scale_s = reinterpret_cast<float2*>(smem + ly.off_scale());

    const int groups = sp.groups, streams = kWarps8 / groups;
    // stages of stream i: the first few have one more
    const int base = ly.stages / streams, more = ly.stages % streams;
    auto first_of = [&](int i) { return i * base + min(i, more); };

    if (warp >= kWarps8) {
        // ------------------------------------------------------ fetchers --
        // A lane fetches for one stream whenever a stage of it is free.  Asking for a
        // unit takes a thread some 290 cycles, so that a unit every 220 takes
        // several warps (one warp: 33.0 us for 64 K rows; those that attend do it
        // themselves: 36.4).
        const uint64_t policy = tc::policy_evict_first();  // the cache is read once
        const int lg_page = __ffs(c8.page_size) - 1;
        const Blocks blocks(a.kv.block_rows);
        const int mine = warp - kWarps8 + lane * kFetchers;  // the stream
        const int st0 = first_of(mine), depth = base + (mine < more ? 1 : 0);
        // (the last lane of all: the queries, a segment ahead)
        const bool asks = warp == kWarps8 + kFetchers - 1 && lane == 31;
        Fetch f{w0, w0.run / sp.passes, 0, mine, 0, 0};
        if (mine >= streams && !asks) f.w.left = 0;
        if (!asks) f.find(a, blocks, lens, runs, sp.passes);
        int st = 0, fetched = 0;
        uint32_t phase = 1;  // (a stage's first fill waits for nobody)
        uint64_t since = 0;
        bool more_q = asks && (w0.left > 0 || C > 1), in_cache = a.k_new == nullptr;
        auto left = [&]() { return asks ? more_q : f.more(); };
        for (uint32_t idle = 0; __any_sync(0xffffffffu, left());) {
            const int at = st0 + st;
            bool go = left() && tc::mbar_test(asks ? &q_empty[st] : &empty[at], phase);
            if (go && !in_cache && !asks && f.w.u + f.at - f.before >= f.w.last_page()) {
                go = in_cache = tc::mbar_test(appended, 0);
                // (what was written there by stores is read by copies)
                if (go) asm volatile("fence.proxy.async;" ::: "memory");
            }
            if (go && asks) {
                const int pass = f.w.run % sp.passes;
                const uint32_t bytes = min(sp.pass_heads, G - pass * sp.pass_heads) * D * es;
                tc::mbar_arrive_expect_tx(&q_full[st], bytes);
                tc::bulk_load(smem + ly.off_q() + st * ly.q_bytes,
                              static_cast<const char*>(a.q) +
                                  ((int64_t)f.w.s * a.n_head + (int64_t)(f.w.run / sp.passes) * G + pass * sp.pass_heads) * D * es,
                              bytes, &q_full[st]);
                ++fetched;
                if (++st == 2) st = 0, phase ^= 1;
                if (f.w.left > 0) f.w.advance(a, lens, runs, f.w.segment());
                more_q = f.w.left > 0;
            } else if (go) {
                const int r = f.row(a, blocks), h = f.h;
                unsigned char* to = smem + at * LY::kStage;
                tc::mbar_arrive_expect_tx(&full[at], LY::kStage);
                tc::tma_load_3d(to, &tmK, &full[at], 0, h, r, policy);
                tc::tma_load_3d(to + LY::kHalf, &tmV, &full[at], 0, h, r, policy);
                if (r < a.kv.rows) {
                    const int64_t page = (int64_t)(r >> lg_page) * Hkv + h;
                    tc::copy4_async(&scale_s[at].x, c8.k_scale + page);
                    tc::copy4_async(&scale_s[at].y, c8.v_scale + page);
                    tc::copies_arrive(&full[at]);
                } else {
                    scale_s[at] = make_float2(0.f, 1.f);
                    tc::mbar_arrive(&full[at]);
                }
                ++fetched;
                if (++st == depth) st = 0, phase ^= 1;
                f.at += streams;
                f.find(a, blocks, lens, runs, sp.passes);
            }
            if (__any_sync(0xffffffffu, go)) {
                idle = 0;
            } else if (++idle == 64) {
                since = tc::globaltimer_ns();
            } else if ((idle & 63) == 0 && __any_sync(0xffffffffu, tc::globaltimer_ns() - since > tmo)) {
                if (lane == 0) report_error(a.err, kDevWaitDecode, 0xb1, fetched);
                break;
            }
        }
        // copies still in flight land before the CTA ends
        const int turn = asks ? 2 : depth;
        for (int i = 0; i < min(fetched, turn); ++i) {
            if (--st < 0) st = turn - 1, phase ^= 1;
            tc::mbar_wait(asks ? &q_full[st] : &full[st0 + st], phase ^ 1, tmo);
        }
        return;
    }

    // ---------------------------------------------------------- consumers --
    if (a.k_new != nullptr) {
        // the ends of runs in this CTA's range, dealt out to the warps, which have nothing to attend yet (done by the
        // fetchers: 64 us for 64 sequences of up to 4096 rows, by a kernel before 65, here 60.8)
        Walk x = w0;
        for (int i = 0; x.left > 0;) {
            const int n = x.segment();
            if (x.u + n == x.units && (i++ & (kWarps8 - 1)) == warp) append_row<D, I8>(a, c8, x.s, x.run, x.n, lane);
            x.advance(a, lens, runs, n);
        }
        asm volatile("fence.proxy.async;" ::: "memory");
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(appended);
    }
    const int grp = warp & (groups - 1), stream = warp / groups;
    const int st0 = first_of(stream), depth = base + (stream < more ? 1 : 0);
    bool ok = true;

    float* om = reinterpret_cast<float*>(smem + ly.off_o());
    float* om_w = om + warp * 8 * D;
    float2* ml = reinterpret_cast<float2*>(smem + ly.off_ml());
    float* mps = reinterpret_cast<float*>(smem + ly.off_mp());
    // Place of 16 bytes in a warp's sums of one head: turned by the head, so that
    // lanes of one column block and four heads meet different banks.
    auto chunk = [&](int g, int c) { return c ^ (D == 128 ? g >> 1 & 3 : (g >> 2 & 1) << 2 | (g >> 1 & 1)); };
    // What is left to do of the segment before: its sums are put together once all
    // warps have left theirs, each warp a head (or as many as there are groups),
    // between two units of the next.
    bool pending = false, whole = false;
    int64_t head_row = 0;  // row of the pass's first query head
    int pass_n = 0, part = 0;  // its heads; the segment's slot in the workspace
    int segs = 0;          // segments whose sums this warp has left
    auto merge = [&]() {
        constexpr int kC = D / 32;  // columns of a lane
        for (int g = warp; g < pass_n; g += kWarps8) {
            const int gw = g >> 3, gh = g & 7;
            // lane r: stream r
            const int at = (lane * groups + gw) * 8 + gh;
            const float2 v = lane < streams ? ml[at] : make_float2(-INFINITY, 0.f);
            const float mp = lane < streams ? mps[at] : 0.f;
            const float* from = om + gw * 8 * D + gh * D + chunk(gh, lane * kC / 4) * 4 + lane * kC % 4;
            float t[kWarps8][kC];
#pragma unroll
            for (int r = 0; r < kWarps8; ++r) {
                const float* x = from + (r < streams ? r * groups * 8 * D : 0);
                if constexpr (kC == 4) *reinterpret_cast<float4*>(t[r]) = *reinterpret_cast<const float4*>(x);
                else *reinterpret_cast<float2*>(t[r]) = *reinterpret_cast<const float2*>(x);
            }
            // relative to the power of two that the largest sum is under: what goes on is never beyond V's largest
            float mt = v.x + (float)((int)(__float_as_uint(v.y) >> 23) - 126);
#pragma unroll
            for (int x = 1; x < 8; x <<= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, x));
            mt = __shfl_sync(0xffffffffu, mt, 0);
            const float f = ex2(v.x - mt + mp);
            float lt = v.y * ex2(v.x - mt);
#pragma unroll
            for (int x = 1; x < 8; x <<= 1) lt += __shfl_xor_sync(0xffffffffu, lt, x);
            lt = __shfl_sync(0xffffffffu, lt, 0);
            float acc[kC];
#pragma unroll
            for (int c = 0; c < kC; ++c) acc[c] = 0.f;
#pragma unroll
            for (int r = 0; r < kWarps8; ++r) {
                const float fr = __shfl_sync(0xffffffffu, f, r);
#pragma unroll
                for (int c = 0; c < kC; ++c) acc[c] = r < streams ? fmaf(fr, t[r][c], acc[c]) : acc[c];
            }
            if constexpr (JOIN) {
                // (the ring: this CTA's last copy has landed)
                float* to = reinterpret_cast<float*>(smem) + g * D + lane * kC;
#pragma unroll
                for (int c = 0; c < kC; ++c) to[c] = acc[c];
                if (lane == 0) *reinterpret_cast<float2*>(smem + kPass8 * D * 4 + g * 8) = make_float2(mt, lt);
            } else if (whole) {
                const float inv = 1.f / lt;
                const int64_t to = (head_row + g) * D + lane * kC;
                if constexpr (kC == 4)
                    store4(a.out, a.out_dtype, to, make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv));
                else
                    store2(a.out, a.out_dtype, to, acc[0] * inv, acc[1] * inv);
            } else {
                const int64_t to = (int64_t)part * groups * 8 + g;
                if constexpr (kC == 4)
                    *reinterpret_cast<float4*>(sp.part_o + to * D + lane * kC) = make_float4(acc[0], acc[1], acc[2], acc[3]);
                else
                    *reinterpret_cast<float2*>(sp.part_o + to * D + lane * kC) = make_float2(acc[0], acc[1]);
                if (lane == 0) sp.part_ml[to] = make_float2(mt, lt);
            }
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(merged);
        pending = false;
    };
    // Waits for all warps' sums, then does this one's share.
    auto finish = [&]() {
        if (!pending) return;
        if (ok && !tc::mbar_wait(written, (segs - 1) & 1, tmo)) {
            ok = false;
            report_error(a.err, kDevWaitDecode, 0xb4, segs);
        }
        __syncwarp();
        merge();
    };
    Walk w = w0;
    int it = 0;  // units of the range before the segment
    int st = 0;  // the next stage, and the phase of its barrier
    uint32_t phase = 0;
    for (int seg = 0; w.left > 0 || (C > 1 && seg == 0); ++seg) {
        const int n_seg = w.segment();
        const int h = sp.passes == 1 ? w.run : w.run / sp.passes, pass = w.run - h * sp.passes;
        const int g0 = pass * sp.pass_heads + grp * 8;  // this warp's first query head of the group
        const int64_t q_row = (int64_t)w.s * a.n_head + (int64_t)h * G;
        // lane: row hd of a 16-row tile and of its second half; columns 2 tq + {0, 1}
        const int hd = lane >> 2, tq = lane & 3;
        // columns D / 8 hd + 2 i + {0, 1} of heads 2 tq + {0, 1}: [i][column * 2 + head]
        float o[D / 16][4];
#pragma unroll
        for (int i = 0; i < D / 16; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        // of heads 2 tq + {0, 1}: log2 of what the weights (l: their sum) are relative to, that of P over it (a small whole
        // number, however large the scores), and the factor from the ones to the other
        float m[2] = {kNone8, kNone8}, mp[2] = {0.f, 0.f}, up[2] = {1.f, 1.f}, l[2] = {0.f, 0.f};
        if (ok && !tc::mbar_wait(&q_full[seg & 1], (seg >> 1) & 1, tmo)) {
            ok = false;
            report_error(a.err, kDevWaitDecode, 0xb3, seg);
        }
        __syncwarp();
        // q in f16, dims D / 4 tq + 4 j + {0, 1, 2, 3} for step j
        uint32_t qh[2 * kSteps], ql[LO ? 2 * kSteps : 1];
        float sl[2];  // factor of the scores of heads 2 tq + {0, 1}
        {
            const unsigned char* qs = smem + ly.off_q() + (seg & 1) * ly.q_bytes + ((grp * 8 + hd) * D + D / 4 * tq) * es;
            const bool in = g0 + hd < G;
            float back = a.kq_scale * kLog2e;
            // factor that takes elements of a head whose largest is `top` to 2^14 .. 2^15; `back` takes it back
            auto scaled = [&](float top) {
                const int e = (int)(__float_as_uint(top) >> 23) - 127;
                const int up = e < 128 ? min(14 - e, 126) : 0;  // (at least -113)
                back *= __uint_as_float((uint32_t)(127 - up) << 23);
                return __uint_as_float((uint32_t)(up + 127) << 23);
            };
            if constexpr (LO) {
                float4 x[kSteps];
                float top = 0.f;
#pragma unroll
                for (int j = 0; j < kSteps; ++j) {
                    x[j] = in ? *reinterpret_cast<const float4*>(qs + 16 * j) : make_float4(0.f, 0.f, 0.f, 0.f);
                    top = fmaxf(fmaxf(fmaxf(fabsf(x[j].x), fabsf(x[j].y)), fmaxf(fabsf(x[j].z), fabsf(x[j].w))), top);
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float f = scaled(top);
#pragma unroll
                for (int j = 0; j < kSteps; ++j) {
                    x[j].x *= f, x[j].y *= f, x[j].z *= f, x[j].w *= f;
                    qh[2 * j] = split2<false>(x[j].x, x[j].y);
                    qh[2 * j + 1] = split2<false>(x[j].z, x[j].w);
                    ql[2 * j] = split2<false>(x[j].x, x[j].y);
                    ql[2 * j + 1] = split2<false>(x[j].z, x[j].w);
                }
            } else {
#pragma unroll
                for (int j = 0; j < kSteps / 2; ++j) {
                    const uint4 x = in ? *reinterpret_cast<const uint4*>(qs + 16 * j) : make_uint4(0, 0, 0, 0);
                    qh[4 * j] = x.x, qh[4 * j + 1] = x.y, qh[4 * j + 2] = x.z, qh[4 * j + 3] = x.w;
                }
                if (a.dtype == 2) {
                    // (a pattern without its sign is in the order of the magnitudes)
                    uint32_t t = 0;
#pragma unroll
                    for (int j = 0; j < 2 * kSteps; ++j) t = __vmaxu2(t, qh[j] & 0x7fff7fffu);
                    t = max(t & 0xffffu, t >> 16);
                    t = max(t, __shfl_xor_sync(0xffffffffu, t, 1));
                    t = max(t, __shfl_xor_sync(0xffffffffu, t, 2));
                    const float f = scaled(__uint_as_float(t << 16));
#pragma unroll
                    for (int j = 0; j < 2 * kSteps; ++j) {
                        const __half2 x = __floats2half2_rn(__uint_as_float(qh[j] << 16) * f,
                                                            __uint_as_float(qh[j] & 0xffff0000u) * f);
                        qh[j] = *reinterpret_cast<const uint32_t*>(&x);
                    }
                }
            }
            sl[0] = __shfl_sync(0xffffffffu, back, 8 * tq);
            sl[1] = __shfl_sync(0xffffffffu, back, 8 * tq + 4);
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&q_empty[seg & 1]);
        // first unit of the segment that falls to this stream
        int i = (stream - it) & (streams - 1);
        for (; i < n_seg; i += streams) {
            const int at = st0 + st;
            // (a lane whose wait runs out waits no more; nothing is skipped, so that the lanes stay together)
            if (ok && !tc::mbar_wait(&full[at], phase, tmo)) {
                ok = false;
                report_error(a.err, kDevWaitDecode, 0xb2, it + i);
            }
            __syncwarp();
            if (++st == depth) st = 0, phase ^= 1;
            unsigned char* stage = smem + at * LY::kStage;
            const unsigned char* vb = stage + LY::kHalf;
            const int u = w.u + i, lim = min(kUnit, w.n - u * kUnit);
            const float2 sc = scale_s[at];
            if (!I8 && lim < kUnit) {
                // V rows past the length may hold NaN codes: their P is 0, and 0 * NaN is not 0
                for (int j = lane; j < (kUnit - lim) * (D / 16); j += 32)
                    *reinterpret_cast<uint4*>(stage + LY::kHalf + lim * D + j * 16) = make_uint4(0, 0, 0, 0);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // TMA writes the stage next
                __syncwarp();
            }
            // scores of keys 16 b + hd and 16 b + 8 + hd: [b][half * 2 + head]; the sum of even steps and that of
            // odd ones (each one's products wait for one another)
            float s4[2][4], s5[2][4];
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                uint4 k4[4];
#pragma unroll
                for (int t = 0; t < 4; ++t)
                    k4[t] = *reinterpret_cast<const uint4*>(stage + tile_at<D>(t * 8 + hd, (D / 64) * tq + c));
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int j = 4 * c + e;
                        auto word = [&](const uint4& x) { return e == 0 ? x.x : e == 1 ? x.y : e == 2 ? x.z : x.w; };
                        uint32_t a0, a1, a2, a3;
                        pairs8<I8>(word(k4[2 * b]), a0, a2);
                        pairs8<I8>(word(k4[2 * b + 1]), a1, a3);
                        float(&x)[4] = j & 1 ? s5[b] : s4[b];
                        if (j < 2) mma8_first(x, a0, a1, a2, a3, qh[2 * j], qh[2 * j + 1]);
                        else mma8(x, a0, a1, a2, a3, qh[2 * j], qh[2 * j + 1]);
                        if constexpr (LO) mma8(x, a0, a1, a2, a3, ql[2 * j], ql[2 * j + 1]);
                    }
            }
            // rows 16 b + 8 t + 2 tq + {0, 1} of V, D / 8 columns from D / 8 hd (asked for before they are wanted)
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
            // log2 of V's scale, rounded up (a number's exponent as the low bits of 2^23)
            const float lv = __uint_as_float(0x4b000000u + ((__float_as_uint(sc.y) + 0x7fffffu) >> 23)) - (8388608.f + 127.f);
            float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) s4[b][e] = (s4[b][e] + s5[b][e]) * (sl[e & 1] * sc.x);
            if (lim < kUnit) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (16 * b + 8 * (e >> 1) + hd >= lim) s4[b][e] = -INFINITY;
            }
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx[e & 1] = fmaxf(mx[e & 1], s4[b][e]);
            // (the maximum over the lanes is wanted where one of them is past a running one only)
            auto past = [&](int e) { return mx[e] - m[e] > kMost8 || mx[e] - m[e] + lv > mp[e] + kMost8; };
            if (__any_sync(0xffffffffu, past(0) || past(1))) {
                float alpha[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int x = 4; x < 32; x <<= 1) mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], x));
                    // (each head for itself: no result depends on the other heads)
                    if (!past(e)) mx[e] = -INFINITY;
                    const float to = fmaxf(m[e], floorf(mx[e])), was = mp[e] + (m[e] - to);
                    // (at most 2^127 for the factor: scales below 2^-112 keep fewer bits; 2^-115 at least)
                    const float tp = fmaxf(fmaxf(was, floorf(mx[e] - to + lv) - kUp8), -127.f);
                    l[e] *= ex2(m[e] - to);
                    alpha[e] = ex2(was - tp);
                    m[e] = to, mp[e] = tp, up[e] = pow2(-tp);
                }
#pragma unroll
                for (int j = 0; j < D / 16; ++j)
                    o[j][0] *= alpha[0], o[j][1] *= alpha[1], o[j][2] *= alpha[0], o[j][3] *= alpha[1];
            }
            const float up0 = up[0] * sc.y, up1 = up[1] * sc.y;
            uint32_t ph[2][2], pl[2][2];  // keys 16 b + 8 half + 2 tq + {0, 1} of head hd
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    float x = ex2(s4[b][2 * t] - m[0]), y = ex2(s4[b][2 * t + 1] - m[1]);
                    l[0] += x, l[1] += y;
                    x *= up0, y *= up1;
                    ph[b][t] = turned(split2<false>(x, y));
                    pl[b][t] = turned(split2<false>(x, y));
                }
            // (four tiles of columns at a time: a tile's products wait for one another)
#pragma unroll
            for (int x = 0; x < D / 32; x += 2) {
                float t[4][4];
                float(*to)[4] = ADD ? t : &o[2 * x];
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    uint32_t a0[8], a1[8];  // [tile * 2 + column]
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        pairs8<I8>(prmt(v[b][0][0][x + y], v[b][0][1][x + y], 0x5140), a0[4 * y], a0[4 * y + 1]);
                        pairs8<I8>(prmt(v[b][0][0][x + y], v[b][0][1][x + y], 0x7362), a0[4 * y + 2], a0[4 * y + 3]);
                        pairs8<I8>(prmt(v[b][1][0][x + y], v[b][1][1][x + y], 0x5140), a1[4 * y], a1[4 * y + 1]);
                        pairs8<I8>(prmt(v[b][1][0][x + y], v[b][1][1][x + y], 0x7362), a1[4 * y + 2], a1[4 * y + 3]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if (ADD && b == 0) mma8_first(to[j], a0[2 * j], a0[2 * j + 1], a1[2 * j], a1[2 * j + 1], pl[b][0], pl[b][1]);
                        else mma8(to[j], a0[2 * j], a0[2 * j + 1], a1[2 * j], a1[2 * j + 1], pl[b][0], pl[b][1]);
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma8(to[j], a0[2 * j], a0[2 * j + 1], a1[2 * j], a1[2 * j + 1], ph[b][0], ph[b][1]);
                }
                if constexpr (ADD) {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[2 * x + j][e] += t[j][e];
                }
            }
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&empty[at]);
            if (pending && __all_sync(0xffffffffu, tc::mbar_test(written, (segs - 1) & 1))) merge();
        }

        // Each warp leaves its sums in shared memory and goes on.
        finish();
        if (segs > 0 && ok && !tc::mbar_wait(merged, (segs - 1) & 1, tmo)) {
            ok = false;
            report_error(a.err, kDevWaitDecode, 0xb5, segs);
        }
        __syncwarp();
        if (__any_sync(0xffffffffu, mp[0] < -60.f || mp[1] < -60.f)) {
            // (small scales alone: the factor 2^mp that takes sums of P to those of the weights, over up to 2^42, stays a
            // number)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (mp[e] < -60.f) {
                    mp[e] += 100.f;
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) o[j][e] *= 0x1p-100f, o[j][2 + e] *= 0x1p-100f;
                }
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
            const int g = 2 * tq + e;
            if (hd == 0) {
                ml[warp * 8 + g] = make_float2(m[e], l[e]);
                mps[warp * 8 + g] = mp[e];
            }
#pragma unroll
            for (int j = 0; j < D / 16; j += 2)
                *reinterpret_cast<float4*>(om_w + g * D + chunk(g, kCols / 4 * hd + j / 2) * 4) =
                    make_float4(o[j][e], o[j][2 + e], o[j + 1][e], o[j + 1][2 + e]);
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(written);
        pending = true;
        ++segs;
        whole = w.u == 0 && n_seg == w.units;
        head_row = q_row + pass * sp.pass_heads;
        pass_n = min(min(groups * 8, sp.pass_heads), G - pass * sp.pass_heads);
        part = blockIdx.x * 2 + (w.u == 0 && w.at > w.per * (int)blockIdx.x ? 1 : 0);
        if constexpr (JOIN) {
            finish();
            join_cluster<D, kThreads8, kPass8>(a, sp, smem, om, w, n_seg, head_row, pass_n, h, rank);
            if (C > 1) tc::cluster_sync();  // nobody reads this CTA's part any more
        }
        if (!sp.direct && threadIdx.x == 0) {
            if (w.u == 0) sp.run_start[(int64_t)w.s * runs + w.run] = w.at;
            const int4 c =
                w.u == 0 && n_seg < w.units
                    ? make_int4(w.s, w.run, w.at, lg_whole > 0 ? w.last_page() + 1 : w.units)  // (whose is the last unit?)
                    : make_int4(-1, 0, 0, 0);
            if (!sp.by_run)
                sp.cut[blockIdx.x] = c;  // the CTA's last segment has the last word
            else if (w.u == 0)
                sp.cut[w.s * runs + w.run] = c;
        }
        it += n_seg;
        w.advance(a, lens, runs, n_seg);
    }
    finish();
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
        sp->direct = sp->cluster > 1 && units <= sp->cluster * kClusterMost8;
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

template <int D, bool I8, bool LO, bool ADD, bool JOIN>
cudaError_t launch8_join(DecodeArgs a, const Cache8& c, const DecodeSplit& sp, cudaStream_t s) {
    CUtensorMap mk, mv;
    if (!cache8_map(&mk, c.k, D, a.n_head_kv, a.kv.rows) || !cache8_map(&mv, c.v, D, a.n_head_kv, a.kv.rows))
        return cudaErrorInvalidValue;
    const Layout8<D> ly = Layout8<D>::make(sp.pass_heads, a.dtype == 0 ? 4 : 2);
    const int smem = 232448;  // all there is: the stages take what is left
    int dev = 0;
    cudaGetDevice(&dev);
    // one bit per device ordinal < 32 whose attribute is set
    static std::atomic<unsigned> set_mask{0};
    if (dev >= 32 || !(set_mask.load(std::memory_order_acquire) & (1u << dev))) {
        const cudaError_t e =
            cudaFuncSetAttribute(k10_decode8<D, I8, LO, ADD, JOIN>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
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
    cfg.blockDim = dim3(kThreads8 + 32 * kFetchers);
    cfg.dynamicSmemBytes = ly.bytes() + 1024;
    cfg.numAttrs = sp.cluster > 1 ? 2 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, k10_decode8<D, I8, LO, ADD, JOIN>, mk, mv, a, c, sp, ly);
    if (e != cudaSuccess || sp.direct) return e;
    const int heads = std::min(a.n_head / a.n_head_kv, sp.pass_heads);
    const int64_t grid = (int64_t)sp.joins * heads;
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.dynamicSmemBytes = 0;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k6b_join<D, true>, a, sp, heads, 0);
}

template <int D, bool I8>
cudaError_t launch8_t(const DecodeArgs& a, const Cache8& c, const DecodeSplit& sp, cudaStream_t s) {
    const bool join = sp.cluster > 1;
    if (a.dtype == 0)
        return join ? launch8_join<D, I8, true, true, true>(a, c, sp, s) : launch8_join<D, I8, true, true, false>(a, c, sp, s);
    if (a.out_dtype == 0)
        return join ? launch8_join<D, I8, false, true, true>(a, c, sp, s)
                    : launch8_join<D, I8, false, true, false>(a, c, sp, s);
    return join ? launch8_join<D, I8, false, false, true>(a, c, sp, s)
                : launch8_join<D, I8, false, false, false>(a, c, sp, s);
}

}  // namespace

size_t decode8_ws_bytes(int32_t n_seq, int32_t max_kv_len, int32_t n_head, int32_t n_head_kv, int32_t head_dim,
                        int32_t dtype) {
    DecodeSplit sp{};
    return split8_of(n_seq, max_kv_len, n_head, n_head_kv, head_dim, dtype, nullptr, &sp);
}

cudaError_t launch_decode8(const DecodeArgs& args, const Cache8& c, cudaStream_t s) {
    DecodeArgs a = args;
    DecodeSplit sp{};
    split8_of(a.kv.n_seq, a.kv.max_kv_len, a.n_head, a.n_head_kv, a.head_dim, a.dtype, static_cast<char*>(a.ws), &sp);
    if (a.k_new && sp.passes > 1) {
        // (several runs read the row: no one of them can write it)
        const AppendArgs w{a.kv, a.k_new, a.v_new, c, a.dtype, a.n_head_kv, a.head_dim, a.err};
        const cudaError_t e = launch_append8(w, s);
        if (e != cudaSuccess) return e;
        a.k_new = a.v_new = nullptr;
    }
    if (a.head_dim == 128) return c.i8 ? launch8_t<128, true>(a, c, sp, s) : launch8_t<128, false>(a, c, sp, s);
    return c.i8 ? launch8_t<64, true>(a, c, sp, s) : launch8_t<64, false>(a, c, sp, s);
}

}  // namespace epsp
