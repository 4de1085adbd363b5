// e4m3 values with one f32 scale per block of 128: the arithmetic shared by
// the activation quantiser, the weight preparation and the products.
//
// Block scale: s = fl(amax * fl(1 / 448)), at least 2^-126 so that it is a
// normal number; 1 for a block of zeros.  Value: q = e4m3(fl(x / s)), round to
// nearest even; |x / s| <= 448 (1 + 2^-21), which rounds to at most 448, so
// nothing saturates.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

namespace rk {

constexpr int kF8Block = 128;

__device__ __forceinline__ float f8_scale(float amax) {
    return amax == 0.0f ? 1.0f : fmaxf(__fmul_rn(amax, 1.0f / 448.0f), 1.17549435e-38f);
}

// Two f32 -> two e4m3 bytes (a in the low byte).
__device__ __forceinline__ uint32_t f8_pack2(float a, float b) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}

__device__ __forceinline__ uint32_t f8_pack4(float a, float b, float c, float d) {
    return f8_pack2(a, b) | (f8_pack2(c, d) << 16);
}

// A quotient whose e4m3 rounding is that of fl(x / s): one step of Markstein's
// method (IBM J. Res. Dev. 34, 1990) from x y, y = RN(1 / s).  x y is off by
// at most 2^-23 of it, the step's remainder and y by 2^-24 of theirs, so q is
// the rounding of a number within 2^-46 of x / s, and differs from fl(x / s)
// only if x / s is that near to the middle of two neighbouring floats.  The
// e4m3 codes then differ only if one of those floats is the middle of two
// e4m3 values.  With s = S 2^i and x = X 2^j (24-bit S, X) and the floats'
// middle C 2^l, C = 2^20 M +- 1 (25 bits, M of 5; 2^21 M - 1 below a power of
// two), that is X 2^k - S C = N, |N| <= 2^49 2^-46 = 8, k >= 23: S is within 8
// of a multiple of 2^20.  N = 0 cannot be, C is odd and longer than X.  For
// such S but the multiples themselves (16 of 2^20) f8_codes() divides.
// Neither a quotient that matters (2^-11 and more; smaller ones are 0 in
// e4m3) nor its remainder, a multiple of 2^-34 2^-23 s, underflows for
// s >= 2^-90; for a smaller s, in no real tensor, f8_codes() divides too.
// Three operations where the IEEE division takes about thirty; the signs are
// such that a quotient of -0 stays one.
__device__ __forceinline__ float f8_quotient(float x, float s, float y) {
    const float q = __fmul_rn(x, y);
    return __fmaf_rn(-y, __fmaf_rn(q, s, -x), q);
}

// Whether f8_quotient serves a block of this scale.
__device__ __forceinline__ bool f8_quick(float s) {
    const uint32_t near = (__float_as_uint(s) + 8u) & 0xFFFFFu;
    return s >= 8.0779357e-28f && (near > 16u || near == 8u);
}

// e4m3 codes of a thread's values of one block (N a multiple of 4), four per
// word.  The rare scale is decided once for all of them.
template <int N>
__device__ __forceinline__ void f8_codes(const float (&v)[N], float s, uint32_t (&code)[N / 4]) {
    float q[N];
    if (f8_quick(s)) {
        const float y = __frcp_rn(s);
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = f8_quotient(v[i], s, y);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) q[i] = __fdiv_rn(v[i], s);
    }
#pragma unroll
    for (int i = 0; i < N / 4; ++i) code[i] = f8_pack4(q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]);
}

// Largest magnitude as an integer: f32 bits without the sign order like the
// magnitudes, infinities and NaN above every finite value, so one maximum
// both finds the scale and shows a non-finite value.
__device__ __forceinline__ uint32_t mag_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
__device__ __forceinline__ bool mag_finite(uint32_t m) { return m < 0x7F800000u; }

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
    return __half2float(v);
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
    return __bfloat162float(v);
}

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
    return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}

// Eight consecutive values as they lie in memory.
template <class T>
struct Raw8 {
    static constexpr int kWords = sizeof(T) * 2;
    uint32_t w[kWords];
    // p at a 16-byte boundary
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) {
            const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0u;
    }
    // up to n of them, at any boundary; 0 behind
    __device__ __forceinline__ void load_some(const T* p, int n) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint32_t b = 0u;
            if (i < n) {
                if constexpr (sizeof(T) == 4)
                    b = __float_as_uint(p[i]);
                else
                    b = reinterpret_cast<const unsigned short*>(p)[i];
            }
            if constexpr (sizeof(T) == 4)
                w[i] = b;
            else
                w[i / 2] = (i & 1) ? (w[i / 2] | (b << 16)) : b;
        }
    }
    // the largest magnitude, as f32 bits (mag_bits); 16-bit types two at a time
    __device__ __forceinline__ uint32_t mag_max() const {
        if constexpr (sizeof(T) == 4) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
            return m;
        } else {
            uint32_t m = w[0] & 0x7FFF7FFFu;
#pragma unroll
            for (int i = 1; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
            const unsigned short b = static_cast<unsigned short>(max(m & 0xFFFFu, m >> 16));
            T x;
            memcpy(&x, &b, 2);
            return __float_as_uint(to_f32<T>(x));
        }
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(w[i]);
            } else {
                const unsigned short b = static_cast<unsigned short>((i & 1) ? w[i / 2] >> 16 : w[i / 2] & 0xFFFFu);
                T x;
                memcpy(&x, &b, 2);
                v[i] = to_f32<T>(x);
            }
        }
    }
};

}  // namespace rk
