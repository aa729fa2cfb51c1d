// cache8.cuh -- the arithmetic of the 8-bit cache, one place for every kernel
// that writes it.
//
// A page's scale is 2^e, e the least integer with amax <= M 2^e (M = 448 for
// e4m3, 127 for integers) and at least -100, and a value's byte the nearest to
// x / 2^e, ties to even.  A power of two costs e4m3 nothing (its steps are
// relative), half a bit of an integer's on average; it makes x / s exact, so
// that the rounding to 8 bits is the only one, that every order of the same
// work gives the same bytes, and that a page whose scale grows under appended
// rows loses only what falls below the new last place.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

#include "epsp_kernels.h"

namespace epsp {
namespace {

constexpr int kLeastExp8 = -100;  // exponent of the smallest scale

// Scale of a page whose largest finite magnitude has these f32 bits.
template <bool I8>
__device__ __forceinline__ float scale8(uint32_t amax_bits) {
    constexpr uint32_t top = I8 ? 0x42fe0000u : 0x43e00000u;  // 127, 448
    // both are m 2^x with x = 6, 8: the exponents' difference, one more where amax's mantissa is the larger
    const int e = (int)(amax_bits >> 23) - (int)(top >> 23) + ((amax_bits & 0x7fffffu) > (top & 0x7fffffu) ? 1 : 0);
    return __uint_as_float((uint32_t)(max(e, kLeastExp8) + 127) << 23);
}

// 1 / s where that is exact (a power of two), else 0.
__device__ __forceinline__ float exact_inverse(float s) {
    const uint32_t b = __float_as_uint(s), e = b >> 23;
    return (b & 0x7fffffu) == 0 && e >= 1 && e <= 253 ? __uint_as_float((254 - e) << 23) : 0.f;
}

// Four values, already divided by their scale and at most its M, to bytes.  The
// integers are the low bits of a sum with 1.5 * 2^23, which rounds as wanted.
template <bool I8>
__device__ __forceinline__ uint32_t to8(float x0, float x1, float x2, float x3) {
    if constexpr (I8) {
        auto q = [](float x) { return __float_as_uint(x + 12582912.f); };
        return __byte_perm(__byte_perm(q(x0), q(x1), 0x0040), __byte_perm(q(x2), q(x3), 0x0040), 0x5410);
    } else {
        uint32_t r;
        asm("{\n .reg .b16 l, h;\n cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n"
            " mov.b32 %0, {l, h};\n}"
            : "=r"(r)
            : "f"(x0), "f"(x1), "f"(x2), "f"(x3));
        return r;
    }
}

// What a value that is not finite goes into the cache as, already divided: an
// infinity as the largest magnitude, a NaN as 0.
template <bool I8>
__device__ __forceinline__ float tame8(float x) {
    constexpr float top = I8 ? 127.f : 448.f;
    return x == x ? fminf(fmaxf(x, -top), top) : 0.f;
}

// Four bytes to the numbers they hold, exactly.
template <bool I8>
__device__ __forceinline__ void from8(uint32_t w, float (&x)[4]) {
    if constexpr (I8) {
        // b + 128 as the low bits of 2^23
        const uint32_t u = w ^ 0x80808080u;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(__byte_perm(u, 0x4b000000u, 0x7440 + i)) - 8388736.f;
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * i)), __NV_E4M3);
            const float2 f = __half22float2(__half2(h));
            x[2 * i] = f.x;
            x[2 * i + 1] = f.y;
        }
    }
}

// x / s: by its exact inverse where it has one.
__device__ __forceinline__ float over(float x, float s, float inv) { return inv != 0.f ? x * inv : x / s; }

// The bytes of rows [0, rows) of one head at `p` follow their page's scale from
// `was` to `s`: thread `first` of `step` threads, A 16-byte pieces of each on
// their way at a time.  (A warp wants eight: a step of 64 sequences in which every
// page grows takes 88 us; by 4 bytes, one row after the other, 264.)
template <bool I8, int A>
__device__ __forceinline__ void rescale8(uint8_t* p, int64_t stride, int rows, int d, float was, float s, int first, int step) {
    const float f = was / s;
    const int lg = __ffs(d / 16) - 1, n = rows << lg;
    auto at = [&](int i) { return reinterpret_cast<uint4*>(p + (int64_t)(i >> lg) * stride + (i & ((1 << lg) - 1)) * 16); };
    for (int i0 = first; i0 < n; i0 += A * step) {
        uint4 w[A];
#pragma unroll
        for (int j = 0; j < A; ++j)
            if (i0 + j * step < n) w[j] = *at(i0 + j * step);
#pragma unroll
        for (int j = 0; j < A; ++j) {
            if (i0 + j * step >= n) break;
            uint32_t* q = reinterpret_cast<uint32_t*>(&w[j]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x[4];
                from8<I8>(q[e], x);
                q[e] = to8<I8>(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
            }
            *at(i0 + j * step) = w[j];
        }
    }
}

// f32 bits of |x| where x is finite, else 0; `odd` is set where it is not.
__device__ __forceinline__ uint32_t magnitude(float x, bool& odd) {
    const uint32_t b = __float_as_uint(x) & 0x7fffffffu;
    if (b < 0x7f800000u) return b;
    odd = true;
    return 0;
}

}  // namespace
}  // namespace epsp
