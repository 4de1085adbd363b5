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

// Eight consecutive values at a 16-byte boundary.
template <class T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
        v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            T lo, hi;
            const unsigned short l = static_cast<unsigned short>(w[i] & 0xFFFFu),
                                 h = static_cast<unsigned short>(w[i] >> 16);
            if constexpr (sizeof(T) == 2) {
                memcpy(&lo, &l, 2);
                memcpy(&hi, &h, 2);
            }
            v[2 * i] = to_f32<T>(lo);
            v[2 * i + 1] = to_f32<T>(hi);
        }
    }
}

}  // namespace rk
