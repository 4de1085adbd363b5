// e4m3 quantisation with one scale per block of 128 (f8.cuh): activation
// rows (a scale per row and 128 columns) and weights (a scale per 128 x 128
// block), dense or from ggml K-quant superblocks.
//
// All are byte streams bound by HBM: each value is read once, held in
// registers while its block's largest magnitude is found (warp shuffles, for
// a 128 x 128 block also shared memory), and its code written once.
#include <algorithm>

#include "f8.cuh"
#include "kernels.h"
#include "kquant.cuh"
#include "ptx.cuh"

namespace rk {
namespace {

constexpr int kRowsThreads = 256;
constexpr int kUnroll = 4;  // blocks of 128 that a half-warp has in flight

__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// Values col..col+7 of a row that ends at k; 0 behind it.
template <class T, bool VEC>
__device__ __forceinline__ void row_load8(const T* row, int col, int k, float (&v)[8]) {
    if (VEC && col + 8 <= k) {
        load8(row + col, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = col + i < k ? to_f32<T>(row[col + i]) : 0.0f;
}

template <bool VEC>
__device__ __forceinline__ void row_store8(uint8_t* row, int col, int k, const float (&v)[8], float s) {
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = __fdiv_rn(v[i], s);
    const uint32_t lo = f8_pack4(q[0], q[1], q[2], q[3]), hi = f8_pack4(q[4], q[5], q[6], q[7]);
    if (VEC && col + 8 <= k) {
        *reinterpret_cast<uint2*>(row + col) = make_uint2(lo, hi);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (col + i < k) row[col + i] = static_cast<uint8_t>((i < 4 ? lo : hi) >> (8 * (i & 3)));
}

// A half-warp per block, 8 consecutive values per lane, kUnroll blocks per
// half-warp with all their loads in flight.  Triggers the dependent product
// at its start: that reads nothing of this kernel's before its own wait.
template <class T, bool VEC>
__global__ void __launch_bounds__(kRowsThreads) rows_f8_kernel(const T* __restrict__ a, int k, long long lda,
                                                               unsigned kb, unsigned blocks,
                                                               uint8_t* __restrict__ out, long long ld8,
                                                               float* __restrict__ scales, long long lds, int* err) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const unsigned half = (blockIdx.x * kRowsThreads + threadIdx.x) >> 4;
    const unsigned halves = gridDim.x * (kRowsThreads / 16);
    const int lane = threadIdx.x & 15;
    float v[kUnroll][8];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const unsigned b = half + u * halves;
        const unsigned r = b / kb;
        if (b < blocks) {
            row_load8<T, VEC>(a + r * lda, static_cast<int>(b - r * kb) * kF8Block + lane * 8, k, v[u]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[u][i] = 0.0f;
        }
    }
    bool finite = true;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const unsigned b = half + u * halves;
        const unsigned r = b / kb, c = b - r * kb;
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            amax = fmaxf(amax, fabsf(v[u][i]));
            finite &= isfinite(v[u][i]);
        }
        const float s = f8_scale(half_warp_max(amax));
        if (b < blocks) {
            row_store8<VEC>(out + r * ld8, static_cast<int>(c) * kF8Block + lane * 8, k, v[u], s);
            if (lane == 0) scales[r * lds + c] = s;
        }
    }
    if (!finite) atomicExch(err, kErrNonFinite);
}

template <class T>
int rows_f8(const T* a, int m, int k, long long lda, uint8_t* out, long long ld8, float* scales, long long lds,
            int* err, cudaStream_t s) {
    const unsigned kb = static_cast<unsigned>((k + kF8Block - 1) / kF8Block);
    const unsigned long long total = static_cast<unsigned long long>(m) * kb;
    if (total > 0xF0000000ull) return cudaErrorInvalidValue;
    const unsigned per = kRowsThreads / 16 * kUnroll;
    const unsigned grid = static_cast<unsigned>((total + per - 1) / per);
    const bool vec = (reinterpret_cast<uintptr_t>(a) % 16 == 0) && (lda * sizeof(T)) % 16 == 0 &&
                     (reinterpret_cast<uintptr_t>(out) % 8 == 0) && ld8 % 8 == 0;
    auto kern = vec ? rows_f8_kernel<T, true> : rows_f8_kernel<T, false>;
    // the max-shared carveout, so that the dependent product's CTA (about
    // 200 KB of shared memory) becomes resident beside these
    static bool carve[64][2] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !carve[dev][vec]) {
        cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        carve[dev][vec] = true;
    }
    kern<<<grid, kRowsThreads, 0, s>>>(a, k, lda, kb, static_cast<unsigned>(total), out, ld8, scales, lds, err);
    return cudaGetLastError();
}

// ---- 128 x 128 weight blocks ----------------------------------------------

constexpr int kPrepThreads = 256;

template <int THREADS>
__device__ __forceinline__ float cta_max(float v, float* red) {
    v = warp_max(v);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    float r = red[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) r = fmaxf(r, red[w]);
    return r;
}

// One CTA per block: 16 lanes of 8 values per row, 16 rows per pass, 8 passes
// held in registers.
template <class T, bool VEC>
__global__ void __launch_bounds__(kPrepThreads) prep_f8_dense_kernel(const T* __restrict__ w, int n, int k,
                                                                     long long ldw, unsigned nb, unsigned kb,
                                                                     uint8_t* __restrict__ out, long long ld8,
                                                                     float* __restrict__ scales, int* err) {
    __shared__ float red[kPrepThreads / 32];
    const unsigned per = nb * kb;
    const unsigned mat = blockIdx.x / per, b = blockIdx.x - mat * per;
    const unsigned rb = b / kb, cb = b - rb * kb;
    const int col = static_cast<int>(cb) * kF8Block + (threadIdx.x & 15) * 8;
    const int row0 = static_cast<int>(rb) * kF8Block + (threadIdx.x >> 4);
    w += static_cast<long long>(mat) * n * ldw;
    out += static_cast<long long>(mat) * n * ld8;
    float v[8][8];
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int r = row0 + 16 * p;
        if (r < n) {
            row_load8<T, VEC>(w + r * ldw, col, k, v[p]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[p][i] = 0.0f;
        }
    }
    float amax = 0.0f;
    bool finite = true;
#pragma unroll
    for (int p = 0; p < 8; ++p)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            amax = fmaxf(amax, fabsf(v[p][i]));
            finite &= isfinite(v[p][i]);
        }
    if (!finite) atomicExch(err, kErrNonFinite);
    const float s = f8_scale(cta_max<kPrepThreads>(amax, red));
    if (threadIdx.x == 0) scales[blockIdx.x] = s;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const int r = row0 + 16 * p;
        if (r < n) row_store8<VEC>(out + r * ld8, col, k, v[p], s);
    }
}

constexpr int kKqThreads = 1024;

// K-quant superblocks: one CTA per 128 rows of one superblock column (two
// 128 x 128 blocks).  A warp dequantises 4 superblocks, 8 values per lane;
// lanes 0-15 own the first 128 values of a superblock, lanes 16-31 the rest.
template <int KIND>
__global__ void __launch_bounds__(kKqThreads) prep_f8_kq_kernel(const uint8_t* __restrict__ blocks, int n,
                                                                unsigned sb, uint8_t* __restrict__ out,
                                                                long long ld8, float* __restrict__ scales, int* err) {
    constexpr int kBytes = KIND == kQ4K ? 144 : KIND == kQ5K ? 176 : 210;
    __shared__ float red[2][kKqThreads / 32];
    const unsigned rb = blockIdx.x / sb, cb = blockIdx.x - rb * sb;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    float v[4][8];
    float amax = 0.0f;
    bool finite = true;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const long long r = static_cast<long long>(rb) * kF8Block + warp * 4 + p;
        if (r < n) {
            dequant8<KIND>(blocks + (r * sb + cb) * kBytes, lane, [&](int slot, int, float x) {
                v[p][slot] = x;
                amax = fmaxf(amax, fabsf(x));
                finite &= isfinite(x);
            });
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[p][i] = 0.0f;
        }
    }
    if (!finite) atomicExch(err, kErrNonFinite);
    amax = half_warp_max(amax);
    static_assert(kKqThreads / 32 == 32, "two maxima per lane below");
    if ((lane & 15) == 0) red[lane >> 4][warp] = amax;
    __syncthreads();
    // two reads of 16 maxima by each half-warp, then a shuffle
    const float s = f8_scale(half_warp_max(fmaxf(red[lane >> 4][lane & 15], red[lane >> 4][16 + (lane & 15)])));
    if (warp == 0 && (lane & 15) == 0)
        scales[static_cast<long long>(rb) * 2 * sb + 2 * cb + (lane >> 4)] = s;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const long long r = static_cast<long long>(rb) * kF8Block + warp * 4 + p;
        if (r >= n) continue;
        uint8_t* dst = out + r * ld8 + cb * 256;
        float q[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = __fdiv_rn(v[p][i], s);
        if constexpr (KIND == kQ6K) {
            const int base = 128 * (lane >> 4) + (lane & 15) * 2;
#pragma unroll
            for (int t = 0; t < 4; ++t)
                *reinterpret_cast<uint16_t*>(dst + base + 32 * t) = static_cast<uint16_t>(f8_pack2(q[t], q[4 + t]));
        } else {
            const int base = 64 * (lane >> 3) + (lane & 7) * 4;
            *reinterpret_cast<uint32_t*>(dst + base) = f8_pack4(q[0], q[1], q[2], q[3]);
            *reinterpret_cast<uint32_t*>(dst + base + 32) = f8_pack4(q[4], q[5], q[6], q[7]);
        }
    }
}

template <class T>
int prep_dense(const T* w, int n, int k, long long ldw, int count, uint8_t* out, long long ld8, float* scales,
               int* err, cudaStream_t s) {
    const unsigned nb = (n + kF8Block - 1) / kF8Block, kb = (k + kF8Block - 1) / kF8Block;
    const unsigned long long grid = static_cast<unsigned long long>(nb) * kb * count;
    if (grid > 0x7fffffffull) return cudaErrorInvalidValue;
    const bool vec = (reinterpret_cast<uintptr_t>(w) % 16 == 0) && (ldw * sizeof(T)) % 16 == 0 &&
                     (reinterpret_cast<uintptr_t>(out) % 8 == 0) && ld8 % 8 == 0;
    auto kern = vec ? prep_f8_dense_kernel<T, true> : prep_f8_dense_kernel<T, false>;
    kern<<<static_cast<unsigned>(grid), kPrepThreads, 0, s>>>(w, n, k, ldw, nb, kb, out, ld8, scales, err);
    return cudaGetLastError();
}

}  // namespace

int launch_quant_rows_f8(int type, const void* a, int m, int k, long long lda, uint8_t* out, long long ld8,
                         float* scales, long long lds, int* err, cudaStream_t s) {
    switch (type) {
        case kTypeF32: return rows_f8(static_cast<const float*>(a), m, k, lda, out, ld8, scales, lds, err, s);
        case kTypeF16: return rows_f8(static_cast<const __half*>(a), m, k, lda, out, ld8, scales, lds, err, s);
        case kTypeBF16: return rows_f8(static_cast<const __nv_bfloat16*>(a), m, k, lda, out, ld8, scales, lds, err, s);
        default: return cudaErrorInvalidValue;
    }
}

int launch_prep_f8(int type, const void* w, int n, int k, long long ldw, int count, uint8_t* out, long long ld8,
                   float* scales, int* err, cudaStream_t s) {
    switch (type) {
        case kTypeF32: return prep_dense(static_cast<const float*>(w), n, k, ldw, count, out, ld8, scales, err, s);
        case kTypeF16: return prep_dense(static_cast<const __half*>(w), n, k, ldw, count, out, ld8, scales, err, s);
        case kTypeBF16:
            return prep_dense(static_cast<const __nv_bfloat16*>(w), n, k, ldw, count, out, ld8, scales, err, s);
        default: return cudaErrorInvalidValue;
    }
}

int launch_prep_f8_kq(int kind, const uint8_t* blocks, int n, int k, uint8_t* out, long long ld8, float* scales,
                      int* err, cudaStream_t s) {
    const unsigned sb = static_cast<unsigned>(k / 256), nb = (n + kF8Block - 1) / kF8Block;
    const unsigned long long grid = static_cast<unsigned long long>(nb) * sb;
    if (grid > 0x7fffffffull) return cudaErrorInvalidValue;
    const unsigned g = static_cast<unsigned>(grid);
    switch (kind) {
        case kQ4K: prep_f8_kq_kernel<kQ4K><<<g, kKqThreads, 0, s>>>(blocks, n, sb, out, ld8, scales, err); break;
        case kQ5K: prep_f8_kq_kernel<kQ5K><<<g, kKqThreads, 0, s>>>(blocks, n, sb, out, ld8, scales, err); break;
        case kQ6K: prep_f8_kq_kernel<kQ6K><<<g, kKqThreads, 0, s>>>(blocks, n, sb, out, ld8, scales, err); break;
        default: return cudaErrorInvalidValue;
    }
    return cudaGetLastError();
}

}  // namespace rk
