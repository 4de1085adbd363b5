// ggml K-quant superblocks (Q4_K / Q5_K / Q6_K) -> f32 values on the device,
// shared by the int8 (quant.cu) and e4m3 (quant_f8.cu) weight preparations.
#pragma once

#include <cuda_fp16.h>

#include <cstdint>

#include "kernels.h"
#include "quant_math.cuh"

namespace rk {

__device__ __forceinline__ uint32_t ld32(const uint8_t* p) { return *reinterpret_cast<const uint32_t*>(p); }
__device__ __forceinline__ uint32_t ld16(const uint8_t* p) { return *reinterpret_cast<const uint16_t*>(p); }

__device__ __forceinline__ float half_bits_to_float(uint32_t bits) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(bits & 0xFFFFu)));
}

// Byte i (0..11) of the 12 scale bytes held in three little-endian words.
__device__ __forceinline__ int scale_byte(const uint32_t (&s)[3], int i) {
    const uint32_t w = i < 4 ? s[0] : (i < 8 ? s[1] : s[2]);
    return static_cast<int>((w >> (8 * (i & 3))) & 0xFFu);
}

// 6-bit scale/min pair j of a Q4_K/Q5_K superblock (ggml's K-quant scale
// packing: j < 4 in the low 6 bits of bytes j / j+4, j >= 4 split between
// the nibbles of byte j+4 and the top bits of bytes j-4 / j).
__device__ __forceinline__ void scale_min_k4(int j, const uint32_t (&s)[3], int& sc, int& m) {
    if (j < 4) {
        sc = scale_byte(s, j) & 63;
        m = scale_byte(s, j + 4) & 63;
    } else {
        sc = (scale_byte(s, j + 4) & 0x0F) | ((scale_byte(s, j - 4) >> 6) << 4);
        m = (scale_byte(s, j + 4) >> 4) | ((scale_byte(s, j) >> 6) << 4);
    }
}

// Dequantise the 8 values that thread `l` (0..31) owns in one superblock and
// hand them to `put(slot, index_in_block, value)`; slot 0..7 is a fixed
// per-lane order (Q4_K/Q5_K: slots 0-3 are 4 consecutive values at
// 64g + 4(l%8), slots 4-7 the 4 at 32 further; Q6_K: slots t and 4 + t are the
// 2 consecutive values at 128h + 2(l%16) + 32t).  Value formulas follow the
// llama-gguf dequantisers the reference calls (capi/src/lib.rs:732-733,
// 986-988): Q4_K/Q5_K (d*sc)*q - (dmin*m), Q6_K (d*sc)*(q-32), f32 each step.
template <int KIND, class Put>
__device__ __forceinline__ void dequant8(const uint8_t* blk, int l, Put&& put) {
    if constexpr (KIND == kQ4K || KIND == kQ5K) {
        const uint32_t dd = ld32(blk);
        const float d = half_bits_to_float(dd), dmin = half_bits_to_float(dd >> 16);
        const uint32_t s[3] = {ld32(blk + 4), ld32(blk + 8), ld32(blk + 12)};
        const int g = l >> 3, i4 = (l & 7) * 4;
        int sc, mn;
        scale_min_k4(2 * g, s, sc, mn);
        const float d1 = __fmul_rn(d, static_cast<float>(sc)), m1 = __fmul_rn(dmin, static_cast<float>(mn));
        scale_min_k4(2 * g + 1, s, sc, mn);
        const float d2 = __fmul_rn(d, static_cast<float>(sc)), m2 = __fmul_rn(dmin, static_cast<float>(mn));
        const uint32_t q = ld32(blk + (KIND == kQ4K ? 16 : 48) + 32 * g + i4);
        uint32_t h = 0;
        if constexpr (KIND == kQ5K) h = ld32(blk + 16 + i4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int lo = (q >> (8 * i)) & 0x0F, hi = (q >> (8 * i + 4)) & 0x0F;
            if constexpr (KIND == kQ5K) {
                const uint32_t hb = (h >> (8 * i)) & 0xFF;
                lo |= ((hb >> (2 * g)) & 1) << 4;
                hi |= ((hb >> (2 * g + 1)) & 1) << 4;
            }
            put(i, 64 * g + i4 + i, __fsub_rn(__fmul_rn(d1, small_uint_to_float(lo)), m1));
            put(4 + i, 64 * g + 32 + i4 + i, __fsub_rn(__fmul_rn(d2, small_uint_to_float(hi)), m2));
        }
    } else {
        const float d = half_bits_to_float(ld16(blk + 208));
        const int h = l >> 4, lp = (l & 15) * 2;
        const uint32_t qa = ld16(blk + 64 * h + lp);
        const uint32_t qb = ld16(blk + 64 * h + 32 + lp);
        const uint32_t qh = ld16(blk + 128 + 32 * h + lp);
        const int8_t* sc = reinterpret_cast<const int8_t*>(blk + 192);
        float ds[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) ds[t] = __fmul_rn(d, static_cast<float>(sc[8 * h + 2 * t + (lp >> 4)]));
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t a = (qa >> (8 * e)) & 0xFF, b = (qb >> (8 * e)) & 0xFF, hb = (qh >> (8 * e)) & 0xFF;
            // q - 32 as an exact float: (2^23 + q) - (2^23 + 32)
            const uint32_t q0 = (a & 0x0F) | ((hb & 3) << 4);
            const uint32_t q1 = (b & 0x0F) | (((hb >> 2) & 3) << 4);
            const uint32_t q2 = (a >> 4) | (((hb >> 4) & 3) << 4);
            const uint32_t q3 = (b >> 4) | (((hb >> 6) & 3) << 4);
            const int base = 128 * h + lp + e;
            put(4 * e + 0, base, __fmul_rn(ds[0], __fsub_rn(__uint_as_float(0x4B000000u | q0), 8388640.0f)));
            put(4 * e + 1, base + 32, __fmul_rn(ds[1], __fsub_rn(__uint_as_float(0x4B000000u | q1), 8388640.0f)));
            put(4 * e + 2, base + 64, __fmul_rn(ds[2], __fsub_rn(__uint_as_float(0x4B000000u | q2), 8388640.0f)));
            put(4 * e + 3, base + 96, __fmul_rn(ds[3], __fsub_rn(__uint_as_float(0x4B000000u | q3), 8388640.0f)));
        }
    }
}

}  // namespace rk
