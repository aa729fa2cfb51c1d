// k_pack8.cu -- K9: rows into the 8-bit cache and out of it.
//
//   pack    q = round8(x / s), s = scale of the page's rows and KV head
//   unpack  x = q s
//   append  one token's row per sequence (before K10 attends it)
//
// Every element is read once and written once: memory bounds them.
//
// pack: a CTA takes the rows of one page and KV head, of K or of V, into
// registers (16 bytes a load, all in flight before the first is used), so that
// the maximum and the bytes come from one read.  The CTAs of a page's heads
// follow one another, so the whole rows of the source are read at about one
// time.  A page that holds rows before `first` keeps its scale, or has it grown
// and those rows' bytes follow, by the same CTA.  64 K rows (8 heads of 128,
// bf16 to e4m3) 80 us, 5.0 TB/s: the waits within a tile, for its rows and for its
// maximum, bound it (issue slots 50 % busy, 24 warps an SM).
// unpack: tiles of 32 rows, which lie together in both caches, 16 bytes a
// thread.  32 K rows (4 heads of 128, to bf16) 23 us, 4.3 TB/s with the launch.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <climits>

#include "cache8.cuh"
#include "epsp_kernels.h"
#include "tc100.cuh"

namespace epsp {
namespace {

constexpr int kThreads = 256;
constexpr int kOver = 16;  // CTAs per SM that a grid has at most (64 K rows packed: 8 79.3 us, 16 78.9, 32 79.6, 64 87)

// The 4 values of 8 bytes (16-bit types) or 16 bytes (f32).
template <int ET>
__device__ __forceinline__ void values4(const uint32_t* w, float (&x)[4]) {
    if constexpr (ET == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(w[i]);
    } else if constexpr (ET == 1) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[2 * i] = f.x, x[2 * i + 1] = f.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}

// Rows [first, len) of a sequence; an empty range where `first` is none, or no
// rows may be written.
__device__ __forceinline__ int2 span_of(const PackArgs& a, int s) {
    const bool held = held_back(a.dst, a.err);
    const int n = batch_len(a.src, s, a.err), f = a.first ? a.first[s] : 0;
    if (f < 0 || f > n) {
        report_error(a.err, kDevBadLength, 0x92, s);
        return make_int2(0, 0);
    }
    return held ? make_int2(0, 0) : make_int2(f, n);
}

// Largest of the CTA's values.  (Two calls in a row want two boxes: a warp may
// write the second while another still reads the first.)
__device__ __forceinline__ uint32_t cta_max(uint32_t m, uint32_t* box) {
    m = __reduce_max_sync(0xffffffffu, m);
    if ((threadIdx.x & 31) == 0) box[threadIdx.x >> 5] = m;
    __syncthreads();
    m = 0;
    for (int i = 0; i < (int)blockDim.x / 32; ++i) m = max(m, box[i]);
    return m;
}

// Larger of m's values and the magnitudes of w's (f32: one, 16-bit types: two of
// each); a NaN stays.
template <int ET>
__device__ __forceinline__ uint32_t larger(uint32_t m, uint32_t w) {
    if constexpr (ET == 0) {
        return max(m, w & 0x7fffffffu);
    } else if constexpr (ET == 1) {
        const __half2 r = __hmax2_nan(*reinterpret_cast<const __half2*>(&m), __habs2(*reinterpret_cast<const __half2*>(&w)));
        return *reinterpret_cast<const uint32_t*>(&r);
    } else {
        const __nv_bfloat162 r =
            __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&m), __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w)));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
}

// The largest of m's values as f32 bits: patterns of one type are in the order of
// the magnitudes, a NaN's above all.
template <int ET>
__device__ __forceinline__ uint32_t top_of(uint32_t m) {
    if constexpr (ET == 0) return m;
    m = max(m & 0x7fffu, m >> 16 & 0x7fffu);
    if constexpr (ET == 2) return m << 16;
    return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
}

// Four values (8 or 16 bytes) to bytes of scale 1 / inv, all of them finite.
template <int ET, bool I8>
__device__ __forceinline__ uint32_t quantised(const uint32_t* w, float inv) {
    if constexpr (ET == 1 && !I8) {
        // (the product is exact but below 2^-14, where e4m3 has nothing but 0)
        uint32_t r;
        const __half2 f = __float2half2_rn(inv);
        const __half2 x = __hmul2(*reinterpret_cast<const __half2*>(&w[0]), f), y = __hmul2(*reinterpret_cast<const __half2*>(&w[1]), f);
        asm("{\n .reg .b16 l, h;\n cvt.rn.satfinite.e4m3x2.f16x2 l, %1;\n cvt.rn.satfinite.e4m3x2.f16x2 h, %2;\n"
            " mov.b32 %0, {l, h};\n}"
            : "=r"(r)
            : "r"(*reinterpret_cast<const uint32_t*>(&x)), "r"(*reinterpret_cast<const uint32_t*>(&y)));
        return r;
    } else {
        float x[4];
        values4<ET>(w, x);
        return to8<I8>(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    }
}

// C: 16-byte chunks of a page and head per thread, of T threads.  As many threads an
// SM as leave each the registers it needs: with 1024 of C = 8 some are spilled (64 K
// rows 81.6 us, of 768 80.1; a wider rescaling, eight pieces ahead, 154).
template <int ET, bool I8, int C, int T>
__global__ void __launch_bounds__(T, (C == 1 ? 1536 : C == 2 ? 1280 : C == 4 || T > 256 ? 1024 : 768) / T) k9_pack(const PackArgs a) {
    constexpr int kEs = ET == 0 ? 4 : 2, kPer = 16 / kEs;
    __shared__ uint32_t box[4][T / 32];
    __shared__ int2 span_s, place_s[2];
    tc::pdl_wait();
    tc::pdl_launch();
    const int s = blockIdx.y, P = a.c.page_size, d = a.head_dim, Hkv = a.n_head_kv;
    if (threadIdx.x == 0) span_s = span_of(a, s);
    __syncthreads();
    const int f = span_s.x, n = span_s.y;
    if (f >= n) return;
    // Tiles: a page and head of K or of V, the heads of a page one after the other.
    const int lg_page = __ffs(P) - 1, pages = (int)(((int64_t)n + P - 1) >> lg_page), per_page = 2 * Hkv;
    const int lg = __ffs(d * kEs / 16) - 1;  // chunks per row, a power of two
    const int row0 = threadIdx.x >> lg, rows = T >> lg;
    const int64_t stride = (int64_t)Hkv * d, step_src = stride * rows * kEs, step_dst = stride * rows;
    const int64_t first_src = stride * row0 * kEs + (threadIdx.x & ((1 << lg) - 1)) * 16, first_dst = first_src / kEs;
    const int step_page = (int)gridDim.x / per_page, step_part = (int)gridDim.x % per_page;
    int page = (f >> lg_page) + (int)blockIdx.x / per_page, part = (int)blockIdx.x % per_page;
    // A page's place in both caches.  One thread finds the next tile's while this
    // one's rows are on their way (all of them: 883 instructions a thread and tile
    // of 64 elements a thread, half of them for this).
    auto find = [&](int pg, int turn) {
        if (pg < pages)
            place_s[turn] = make_int2(batch_row(a.src, s, pg << lg_page, a.err), batch_row(a.dst, s, pg << lg_page, a.err));
    };
    if (threadIdx.x == 0) find(page, 0);
    __syncthreads();
    for (int turn = 0; page < pages; turn ^= 1) {
        const bool is_v = part & 1;
        const int h = part >> 1, r0 = page << lg_page, from = place_s[turn].x, to = place_s[turn].y;
        const int lo = max(f, r0) - r0, hi = min(n - r0, P);  // rows of the page to write
        const bool there = from >= 0 && to >= 0;
        const char* src = static_cast<const char*>(is_v ? a.v : a.k) + ((int64_t)from * Hkv + h) * d * kEs;
        uint8_t* dst = (is_v ? a.c.v : a.c.k) + ((int64_t)to * Hkv + h) * d;
        float* scale = (is_v ? a.c.v_scale : a.c.k_scale) + (int64_t)(to >> lg_page) * Hkv + h;
        // this thread's chunks: one of every `rows` rows (a page without its ends asks for no comparisons)
        const bool full = there && lo == 0 && hi == P;
        uint4 v[C];
        uint32_t m = 0;
        const char* mine = src + first_src;
#pragma unroll
        for (int j = 0; j < C; ++j, mine += step_src) {
            const int r = row0 + j * rows;
            v[j] = make_uint4(0, 0, 0, 0);
            if (full || (there && r >= lo && r < hi)) v[j] = __ldcs(reinterpret_cast<const uint4*>(mine));
        }
        const float was = there && lo > 0 ? *scale : 0.f;
        page += step_page, part += step_part;
        if (part >= per_page) part -= per_page, ++page;
        if (threadIdx.x == 0) find(page, turn ^ 1);
#pragma unroll
        for (int j = 0; j < C; ++j) {
            const uint32_t* w = reinterpret_cast<const uint32_t*>(&v[j]);
#pragma unroll
            for (int e = 0; e < 4; ++e) m = larger<ET>(m, w[e]);
        }
        m = cta_max(top_of<ET>(m), box[turn]);
        if (!there) continue;
        const bool odd = m >= 0x7f800000u;
        if (odd) {  // (rare) again, without what is not finite
            m = 0;
            bool any = false;
#pragma unroll 1
            for (int i = threadIdx.x; i < (hi - lo) * d; i += T) {
                const char* p = src + ((int64_t)(lo + i / d) * Hkv * d + i % d) * kEs;
                float x;
                if constexpr (ET == 0) x = *reinterpret_cast<const float*>(p);
                else if constexpr (ET == 1) x = __half2float(*reinterpret_cast<const __half*>(p));
                else x = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(p));
                m = max(m, magnitude(x, any));
            }
            m = cta_max(m, box[2 + turn]);
            if (threadIdx.x == 0) report_error(a.err, kDevNotFinite8, 0x93, r0 >> lg_page);
        }
        float sc = scale8<I8>(m);
        if (was >= sc) sc = was;
        else {
            if (lo > 0) rescale8<I8, 1>(dst, (int64_t)Hkv * d, lo, d, was, sc, threadIdx.x, blockDim.x);
            if (threadIdx.x == 0) *scale = sc;
        }
        const float inv = exact_inverse(sc);
        auto store = [&](auto&& four) {
            uint8_t* o = dst + first_dst;
#pragma unroll
            for (int j = 0; j < C; ++j, o += step_dst) {
                const int r = row0 + j * rows;
                if (!full && (r < lo || r >= hi)) continue;
                const uint32_t* w = reinterpret_cast<const uint32_t*>(&v[j]);
                if constexpr (kPer == 8) *reinterpret_cast<uint2*>(o) = make_uint2(four(w), four(w + 2));
                else *reinterpret_cast<uint32_t*>(o) = four(w);
            }
        };
        // f16 holds the inverse of what it can have as a scale, but for scales that a caller made up
        const bool plain = !odd && inv != 0.f && (ET != 1 || I8 || (inv >= 0x1p-14f && inv <= 0x1p15f));
        if (plain) {
            store([&](const uint32_t* w) { return quantised<ET, I8>(w, inv); });
        } else {
            // (rare) from the source again, four values at a time
#pragma unroll 1
            for (int i = threadIdx.x; i < (hi - lo) * d / 4; i += T) {
                const int64_t el = (int64_t)(lo + i * 4 / d) * stride + i * 4 % d;
                uint32_t w[4];
                const uint2* p = reinterpret_cast<const uint2*>(src + el * kEs);
                *reinterpret_cast<uint2*>(w) = p[0];
                if constexpr (kEs == 4) *reinterpret_cast<uint2*>(w + 2) = p[1];
                float x[4];
                values4<ET>(w, x);
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = tame8<I8>(over(x[k], sc, inv));
                *reinterpret_cast<uint32_t*>(dst + el) = to8<I8>(x[0], x[1], x[2], x[3]);
            }
        }
    }
}

// Largest finite value of the context's type.
template <int ET>
__device__ __forceinline__ float largest() {
    return ET == 0 ? 3.402823466e38f : ET == 1 ? 65504.f : __uint_as_float(0x7f7f0000u);
}

constexpr int kTile = 32;   // rows of a tile: a page holds whole ones, so a tile's rows lie together in both caches
constexpr int kUnpack = 2;  // 16-byte chunks of K and of V per thread and turn

template <int ET, bool I8>
__global__ void __launch_bounds__(kThreads) k9_unpack(const PackArgs a) {
    tc::pdl_wait();
    tc::pdl_launch();
    const int s = blockIdx.y, lg_page = __ffs(a.c.page_size) - 1, lg_head = __ffs(a.head_dim / 16) - 1, Hkv = a.n_head_kv;
    const int2 span = span_of(a, s);
    const int f = span.x, n = span.y, per_row = Hkv << lg_head, per_tile = kTile * per_row;
    for (int64_t at = (int64_t)(f / kTile + (int)blockIdx.x) * kTile; at < n; at += (int64_t)gridDim.x * kTile) {
        const int r0 = (int)at, from = batch_row(a.src, s, r0, a.err), to = batch_row(a.dst, s, r0, a.err);
        if (from < 0 || to < 0) continue;
        const uint4* src[2] = {reinterpret_cast<const uint4*>(a.c.k) + (int64_t)from * per_row,
                               reinterpret_cast<const uint4*>(a.c.v) + (int64_t)from * per_row};
        const int64_t page = (int64_t)(from >> lg_page) * Hkv;
        const int lo = max(f - r0, 0) * per_row, hi = min(n - r0, kTile) * per_row;  // chunks of the tile
        for (int i0 = threadIdx.x; i0 < per_tile; i0 += kThreads * kUnpack) {
            uint4 q[2][kUnpack];
            float sc[2][kUnpack];
#pragma unroll
            for (int j = 0; j < kUnpack; ++j) {
                const int i = i0 + j * kThreads;
                if (i < lo || i >= hi) continue;
                q[0][j] = __ldcs(src[0] + i);
                q[1][j] = __ldcs(src[1] + i);
                const int h = (int)((uint32_t)i % (uint32_t)per_row) >> lg_head;
                sc[0][j] = a.c.k_scale[page + h];
                sc[1][j] = a.c.v_scale[page + h];
            }
#pragma unroll
            for (int kv = 0; kv < 2; ++kv)
#pragma unroll
                for (int j = 0; j < kUnpack; ++j) {
                    const int i = i0 + j * kThreads;
                    if (i < lo || i >= hi) continue;
                    const uint32_t* w = reinterpret_cast<const uint32_t*>(&q[kv][j]);
                    void* out = const_cast<void*>(kv ? a.v : a.k);
                    const int64_t el = ((int64_t)to * per_row + i) * 16;
                    uint32_t o[8];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x[4];
                        from8<I8>(w[e], x);
#pragma unroll
                        for (int k = 0; k < 4; ++k) x[k] *= sc[kv][j];
                        if (sc[kv][j] > largest<ET>() / (I8 ? 128.f : 448.f)) {
                            // (rare) a value near the type's largest may have been rounded past it; a NaN stays
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                if (fabsf(x[k]) > largest<ET>()) x[k] = copysignf(largest<ET>(), x[k]);
                        }
                        if constexpr (ET == 0) {
                            reinterpret_cast<float4*>(static_cast<float*>(out) + el)[e] = make_float4(x[0], x[1], x[2], x[3]);
                        } else if constexpr (ET == 1) {
                            const __half2 p = __floats2half2_rn(x[0], x[1]), r = __floats2half2_rn(x[2], x[3]);
                            o[2 * e] = *reinterpret_cast<const uint32_t*>(&p);
                            o[2 * e + 1] = *reinterpret_cast<const uint32_t*>(&r);
                        } else {
                            const __nv_bfloat162 p = __floats2bfloat162_rn(x[0], x[1]), r = __floats2bfloat162_rn(x[2], x[3]);
                            o[2 * e] = *reinterpret_cast<const uint32_t*>(&p);
                            o[2 * e + 1] = *reinterpret_cast<const uint32_t*>(&r);
                        }
                    }
                    if constexpr (ET != 0) {
                        uint4* p = reinterpret_cast<uint4*>(static_cast<uint16_t*>(out) + el);
                        p[0] = make_uint4(o[0], o[1], o[2], o[3]);
                        p[1] = make_uint4(o[4], o[5], o[6], o[7]);
                    }
                }
        }
    }
}

// One CTA of 128 threads per (sequence, KV head, K or V), an element per thread.
// Latency bounds it: the length, then the block table, then the page's scale.
template <int ET, bool I8>
__global__ void __launch_bounds__(128) k9_append(const AppendArgs a) {
    __shared__ uint32_t box[4];
    __shared__ int n_s;
    tc::pdl_wait();
    tc::pdl_launch();
    const int P = a.c.page_size, d = a.head_dim, Hkv = a.n_head_kv;
    const bool is_v = blockIdx.x & 1;
    const int s = (int)(blockIdx.x >> 1) / Hkv, h = (int)(blockIdx.x >> 1) % Hkv, t = threadIdx.x;
    float x = 0.f;
    if (t < d) {
        const int64_t i = ((int64_t)s * Hkv + h) * d + t;
        const void* src = is_v ? a.v_new : a.k_new;
        if constexpr (ET == 0) x = static_cast<const float*>(src)[i];
        else if constexpr (ET == 1) x = __half2float(static_cast<const __half*>(src)[i]);
        else x = __bfloat162float(static_cast<const __nv_bfloat16*>(src)[i]);
    }
    if (t == 0) n_s = batch_len(a.kv, s, a.err);
    __syncthreads();
    const int n = n_s;
    if (n == 0) return;
    const int r0 = (n - 1) / P * P, lo = n - 1 - r0;
    const int row = held_back(a.kv, a.err) ? -1 : batch_row(a.kv, s, r0, a.err);
    bool odd = false;
    uint32_t m = magnitude(x, odd);
    float* scale = (is_v ? a.c.v_scale : a.c.k_scale) + (int64_t)(max(row, 0) / P) * Hkv + h;
    const float was = row >= 0 && lo > 0 ? *scale : 0.f;
    m = cta_max(m, box);
    odd = __syncthreads_or(odd);
    if (row < 0) return;
    if (odd && t == 0) report_error(a.err, kDevNotFinite8, 0x94, s);
    uint8_t* dst = (is_v ? a.c.v : a.c.k) + ((int64_t)row * Hkv + h) * d;
    float sc = scale8<I8>(m);
    if (was >= sc) sc = was;
    else {
        if (lo > 0) rescale8<I8, 8>(dst, (int64_t)Hkv * d, lo, d, was, sc, threadIdx.x, blockDim.x);
        if (t == 0) *scale = sc;
    }
    if (t < d) dst[(int64_t)lo * Hkv * d + t] = (uint8_t)to8<I8>(tame8<I8>(over(x, sc, exact_inverse(sc))), 0.f, 0.f, 0.f);
}

// Kernels here may start before what precedes them on the stream has ended:
// they wait for it on the device.
template <class... P, class... A>
cudaError_t go(void (*kernel)(P...), dim3 grid, int threads, cudaStream_t s, A... args) {
    cudaLaunchAttribute at{};
    at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.stream = s;
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// CTAs for `work` pieces per sequence.
unsigned grid_x(int64_t work, int32_t n_seq) {
    const int64_t most = std::max<int64_t>(1, 148 * kOver / n_seq);
    return (unsigned)std::min(work, most);
}

template <int ET, bool I8>
cudaError_t pack_t(const PackArgs& a, cudaStream_t s) {
    const int64_t pages = (a.src.max_kv_len + (int64_t)a.c.page_size - 1) / a.c.page_size;
    const dim3 grid(grid_x(pages * a.n_head_kv * 2, a.src.n_seq), a.src.n_seq);
    // (8 chunks a thread: 80 us for 64 K rows in pages of 128; 4, of twice the threads, 94; 16, of half of them, 93)
    const int chunks = a.c.page_size * a.head_dim * (ET == 0 ? 4 : 2) / (16 * kThreads);
    switch (chunks) {
        case 1: return go(k9_pack<ET, I8, 1, 256>, grid, 256, s, a);
        case 2: return go(k9_pack<ET, I8, 2, 256>, grid, 256, s, a);
        case 4: return go(k9_pack<ET, I8, 4, 256>, grid, 256, s, a);
        case 8: return go(k9_pack<ET, I8, 8, 256>, grid, 256, s, a);
        default: return go(k9_pack<ET, I8, 8, 512>, grid, 512, s, a);
    }
}

template <int ET, bool I8>
cudaError_t unpack_t(const PackArgs& a, cudaStream_t s) {
    const int64_t tiles = (a.src.max_kv_len + (int64_t)kTile - 1) / kTile + 1;  // (from `first` rounded down)
    const dim3 grid(grid_x(tiles, a.src.n_seq), a.src.n_seq);
    return go(k9_unpack<ET, I8>, grid, kThreads, s, a);
}

template <int ET, bool I8>
cudaError_t append_t(const AppendArgs& a, cudaStream_t s) {
    const int64_t ctas = (int64_t)a.kv.n_seq * a.n_head_kv * 2;
    if (ctas > INT_MAX) return cudaErrorInvalidValue;
    return go(k9_append<ET, I8>, dim3((unsigned)ctas), 128, s, a);
}

#define EPSP_BY_TYPES(fn, a, s)                                             \
    switch ((a).dtype) {                                                    \
        case 0: return (a).c.i8 ? fn<0, true>(a, s) : fn<0, false>(a, s);   \
        case 1: return (a).c.i8 ? fn<1, true>(a, s) : fn<1, false>(a, s);   \
        default: return (a).c.i8 ? fn<2, true>(a, s) : fn<2, false>(a, s);  \
    }

}  // namespace

cudaError_t launch_pack(const PackArgs& a, cudaStream_t s) { EPSP_BY_TYPES(pack_t, a, s) }
cudaError_t launch_unpack(const PackArgs& a, cudaStream_t s) { EPSP_BY_TYPES(unpack_t, a, s) }
cudaError_t launch_append8(const AppendArgs& a, cudaStream_t s) { EPSP_BY_TYPES(append_t, a, s) }

}  // namespace epsp
