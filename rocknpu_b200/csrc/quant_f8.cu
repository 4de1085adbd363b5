// e4m3 quantisation with one scale per block of 128 (f8.cuh): activation
// rows (a scale per row and 128 columns) and weights (a scale per 128 x 128
// block), dense or from ggml K-quant superblocks.
//
// All are byte streams: each value is read once, held in registers while its
// block's largest magnitude is found (warp shuffles, for a 128 x 128 block
// also shared memory), and its code written once.  What bounds them is the
// arithmetic of a code (an SM issues in about three of four cycles): maximum,
// quotient, conversion, and for K-quants the decoding.
#include <algorithm>

#include "f8.cuh"
#include "kernels.h"
#include "kquant.cuh"
#include "ptx.cuh"

namespace rk {
namespace {

constexpr int kRowsThreads = 256;
constexpr int kRowsUnroll = 2;  // blocks of 128 per half-warp and step
constexpr int kRowsCtas = 4;  // per SM (bf16 16384 x 8192: 4 84 us, 5 85)

__device__ __forceinline__ uint32_t half_warp_max(uint32_t v) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

template <int N>
__device__ __forceinline__ uint32_t mag_max(const float (&v)[N]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, mag_bits(v[i]));
    return m;
}

// Values col..col+7 of a row that ends at k; 0 behind it.
template <class T, bool VEC>
__device__ __forceinline__ void row_load8(const T* row, int col, int k, Raw8<T>& v) {
    if (VEC && col + 8 <= k)
        v.load(row + col);
    else
        v.load_some(row + col, k - col);
}

template <bool VEC>
__device__ __forceinline__ void row_store8(uint8_t* row, int col, int k, const float (&v)[8], float s) {
    uint32_t code[2];
    f8_codes(v, s, code);
    if (VEC && col + 8 <= k) {
        *reinterpret_cast<uint2*>(row + col) = make_uint2(code[0], code[1]);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (col + i < k) row[col + i] = static_cast<uint8_t>(code[i / 4] >> (8 * (i & 3)));
}

// Block b of the walk: column block c of row r.
struct At {
    unsigned b, r, c;
    __device__ __forceinline__ void set(unsigned to, unsigned kb) {
        b = to;
        r = to / kb;
        c = to - r * kb;
    }
    __device__ __forceinline__ void on(const At& by, unsigned kb) {
        b += by.b;
        r += by.r;
        c += by.c;
        if (c >= kb) {
            c -= kb;
            ++r;
        }
    }
};

// A half-warp per kRowsUnroll consecutive blocks, 8 consecutive values per
// lane and block; a step's loads are issued before the step before it is
// quantised.  Triggers the dependent product at its start: that reads nothing
// of this kernel's before its own wait.  VEC, VOUT: rows can be read
// 16 bytes, codes written 8 bytes at a time.  WHOLE (and both): k is a multiple of
// kRowsUnroll blocks, so a step's blocks are whole and neighbours in a row, with one
// address for all: the kernel is bound by its instructions (bf16 16384 x 8192
// 84 us, 4.9 TB/s; 97 with an address and bounds for each block).
template <class T, bool VEC, bool VOUT, bool WHOLE>
__global__ void __launch_bounds__(kRowsThreads, kRowsCtas)
    rows_f8_kernel(const T* __restrict__ a, int k, long long lda, unsigned kb, unsigned blocks,
                   uint8_t* __restrict__ out, long long ld8, float* __restrict__ scales, long long lds, int* err) {
    constexpr int U = kRowsUnroll;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 15;
    At at, step, one;
    one.set(1, kb);
    step.set(gridDim.x * (kRowsThreads / 16) * U, kb);
    at.set((blockIdx.x * (kRowsThreads / 16) + (threadIdx.x >> 4)) * U, kb);
    auto load = [&](At p, Raw8<T>(&v)[U]) {
        if constexpr (WHOLE) {
            const T* row = a + p.r * lda + p.c * kF8Block + lane * 8;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (p.b < blocks)
                    v[u].load(row + u * kF8Block);
                else
                    v[u].clear();
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (p.b < blocks)
                    row_load8<T, VEC>(a + p.r * lda, static_cast<int>(p.c) * kF8Block + lane * 8, k, v[u]);
                else
                    v[u].clear();
                p.on(one, kb);
            }
        }
    };
    Raw8<T> cur[U];
    load(at, cur);
    const unsigned odd = (threadIdx.x >> 4 & 1) * U;  // the two halves of a warp take the same steps
    uint32_t most = 0;
    while (at.b - odd < blocks) {
        Raw8<T> next[U];
        At then = at;
        then.on(step, kb);
        load(then, next);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float v[8];
            cur[u].values(v);
            const uint32_t m = half_warp_max(cur[u].mag_max());
            most = max(most, m);
            const float s = f8_scale(__uint_as_float(m));
            if constexpr (WHOLE) {
                uint32_t code[2];
                f8_codes(v, s, code);
                if (at.b < blocks) {
                    *reinterpret_cast<uint2*>(out + at.r * ld8 + at.c * kF8Block + lane * 8 + u * kF8Block) =
                        make_uint2(code[0], code[1]);
                    if (lane == 0) scales[at.r * lds + at.c + u] = s;
                }
            } else {
                if (at.b < blocks) {
                    row_store8<VOUT>(out + at.r * ld8, static_cast<int>(at.c) * kF8Block + lane * 8, k, v, s);
                    if (lane == 0) scales[at.r * lds + at.c] = s;
                }
                at.on(one, kb);
            }
            cur[u] = next[u];
        }
        at = then;
    }
    if (!mag_finite(most)) report(err, kErrNonFinite);
}

template <class T>
int rows_f8(const T* a, int m, int k, long long lda, uint8_t* out, long long ld8, float* scales, long long lds,
            int* err, cudaStream_t s) {
    const unsigned kb = static_cast<unsigned>((k + kF8Block - 1) / kF8Block);
    const unsigned long long total = static_cast<unsigned long long>(m) * kb;
    if (total > 0xF0000000ull) return cudaErrorInvalidValue;
    const unsigned per = kRowsThreads / 16 * kRowsUnroll;
    const unsigned grid = static_cast<unsigned>(std::min<unsigned long long>((total + per - 1) / per, sm_count() * kRowsCtas));
    // rows of odd lengths still have aligned codes
    const bool vout = reinterpret_cast<uintptr_t>(out) % 8 == 0 && ld8 % 8 == 0;
    const bool vec = reinterpret_cast<uintptr_t>(a) % 16 == 0 && (lda * sizeof(T)) % 16 == 0 && vout;
    const int kind = !vout ? 0 : !vec ? 1 : k % (kRowsUnroll * kF8Block) ? 2 : 3;
    auto kern = kind == 0   ? rows_f8_kernel<T, false, false, false>
                : kind == 1 ? rows_f8_kernel<T, false, true, false>
                : kind == 2 ? rows_f8_kernel<T, true, true, false>
                            : rows_f8_kernel<T, true, true, true>;
    // the max-shared carveout, so that the dependent product's CTA (about
    // 200 KB of shared memory) becomes resident beside these; a long run is no
    // slower with it
    static bool carve[64][4] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && !carve[dev][kind]) {
        cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        carve[dev][kind] = true;
    }
    kern<<<grid, kRowsThreads, 0, s>>>(a, k, lda, kb, static_cast<unsigned>(total), out, ld8, scales, lds, err);
    return cudaGetLastError();
}

// ---- 128 x 128 weight blocks ----------------------------------------------

constexpr int kPrepThreads = 256;
constexpr int kPrepRows = kPrepThreads / 16, kPrepPasses = kF8Block / kPrepRows;

template <int THREADS>
__device__ __forceinline__ uint32_t cta_max(uint32_t v, uint32_t* red) {
    v = __reduce_max_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    uint32_t r = red[0];
#pragma unroll
    for (int w = 1; w < THREADS / 32; ++w) r = max(r, red[w]);
    return r;
}

// One CTA per block: 16 lanes of 8 values per row, kPrepRows rows per pass, all
// passes held in registers.
// VEC, VOUT: rows can be read 16 bytes, codes written 8 bytes at a time.
// WHOLE (and both): every block is, and nothing is asked of bounds (bf16, 8 of
// 5632 x 2048: 55 us, 5.0 TB/s; 58.6 without).  CTAs per SM as the registers
// hold the passes: WHOLE with four spills, 69 us; two of 512 threads 63.
template <class T, bool VEC, bool VOUT, bool WHOLE>
__global__ void __launch_bounds__(kPrepThreads, sizeof(T) == 4 ? 2 : WHOLE ? 3 : 4)
    prep_f8_dense_kernel(const T* __restrict__ w, int n, int k, long long ldw, unsigned nb, unsigned kb,
                         uint8_t* __restrict__ out, long long ld8, float* __restrict__ scales, int* err) {
    __shared__ uint32_t red[kPrepThreads / 32];
    const unsigned per = nb * kb;
    const unsigned mat = blockIdx.x / per, b = blockIdx.x - mat * per;
    const unsigned rb = b / kb, cb = b - rb * kb;
    const int col = static_cast<int>(cb) * kF8Block + (threadIdx.x & 15) * 8;
    const int row0 = static_cast<int>(rb) * kF8Block + (threadIdx.x >> 4);
    w += static_cast<long long>(mat) * n * ldw;
    out += static_cast<long long>(mat) * n * ld8;
    Raw8<T> raw[kPrepPasses];
#pragma unroll
    for (int p = 0; p < kPrepPasses; ++p) {
        const int r = row0 + kPrepRows * p;
        if constexpr (WHOLE)
            raw[p].load(w + r * ldw + col);
        else if (r < n)
            row_load8<T, VEC>(w + r * ldw, col, k, raw[p]);
        else
            raw[p].clear();
    }
    uint32_t m = 0;
#pragma unroll
    for (int p = 0; p < kPrepPasses; ++p) m = max(m, raw[p].mag_max());
    m = cta_max<kPrepThreads>(m, red);
    const float s = f8_scale(__uint_as_float(m));
    if (threadIdx.x == 0) {
        if (!mag_finite(m)) report(err, kErrNonFinite);
        scales[blockIdx.x] = s;
    }
#pragma unroll
    for (int p = 0; p < kPrepPasses; ++p) {
        const int r = row0 + kPrepRows * p;
        float v[8];
        raw[p].values(v);
        if constexpr (WHOLE) {
            uint32_t code[2];
            f8_codes(v, s, code);
            *reinterpret_cast<uint2*>(out + r * ld8 + col) = make_uint2(code[0], code[1]);
        } else {
            if (r < n) row_store8<VOUT>(out + r * ld8, col, k, v, s);
        }
    }
}

constexpr int kKqThreads = 512;

// The values of half a superblock in four rows that a lane owns, 8 each, in
// dequant8's order; `at` is the lane's place there (0..15 the first 128
// values, 16..31 the rest).  A half-warp has a row, rows 2 p and 2 p + 1 of the
// warp's eight are a warp's step p.  The sub-blocks' scales and mins of all eight
// rows, four each, are decoded once per warp, one per lane, and handed out by shuffles;
// dequant8 decodes them in every lane.  The same values, one rounding each.
template <int KIND>
__device__ __forceinline__ void dequant4x8(const uint8_t* const (&blk)[4], const bool (&live)[4], const uint8_t* mine,
                                           bool on, int lane, int at, float (&v)[4][8]) {
    if constexpr (KIND == kQ4K || KIND == kQ5K) {
        const int g = at >> 3, i4 = (at & 7) * 4;
        uint32_t q[4], h[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            q[p] = live[p] ? ld32(blk[p] + (KIND == kQ4K ? 16 : 48) + 32 * g + i4) : 0u;
            h[p] = KIND == kQ5K && live[p] ? ld32(blk[p] + 16 + i4) : 0u;
        }
        float dj = 0.0f, mj = 0.0f;
        if (on) {
            const uint32_t dd = ld32(mine);
            const uint32_t s[3] = {ld32(mine + 4), ld32(mine + 8), ld32(mine + 12)};
            int sc, mn;
            scale_min_k4((at & 16) / 4 + (lane & 3), s, sc, mn);
            dj = __fmul_rn(half_bits_to_float(dd), static_cast<float>(sc));
            mj = __fmul_rn(half_bits_to_float(dd >> 16), static_cast<float>(mn));
        }
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int from = 4 * (2 * p + (lane >> 4)) + 2 * (g & 1) + half;
                const float d = __shfl_sync(0xffffffffu, dj, from), m = __shfl_sync(0xffffffffu, mj, from);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t c = (q[p] >> (8 * i + 4 * half)) & 0x0Fu;
                    if constexpr (KIND == kQ5K) c |= ((h[p] >> (8 * i + 2 * g + half)) & 1u) << 4;
                    v[p][4 * half + i] = __fsub_rn(__fmul_rn(d, small_uint_to_float(c)), m);
                }
            }
    } else {
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            if (live[p]) {
                dequant8<KIND>(blk[p], at, [&](int slot, int, float x) { v[p][slot] = x; });
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[p][i] = 0.0f;
            }
        }
    }
}

// K-quant superblocks: one CTA per 128 x 128 block, 128 rows of half a
// superblock column.  Bound by its arithmetic, with HBM waiting (5632 x 2048:
// Q4_K 10.8 us, Q5_K 13.1, Q6_K 13.3), so several CTAs share an SM and some
// compute while others load; one of 1024 threads per superblock column was
// alone there and took 15.4, 17.3 and 18.6.  Three CTAs spill: faster for Q6_K
// only (n not a multiple of 128: 14.9, two 16.3).
// WHOLE: n is a multiple of 128.
template <int KIND, bool WHOLE>
__global__ void __launch_bounds__(kKqThreads, KIND == kQ6K ? 3 : 2)
    prep_f8_kq_kernel(const uint8_t* __restrict__ blocks, int n, unsigned sb, uint8_t* __restrict__ out, long long ld8,
                      float* __restrict__ scales, int* err) {
    constexpr int kBytes = KIND == kQ4K ? 144 : KIND == kQ5K ? 176 : 210;
    __shared__ uint32_t red[kKqThreads / 32];
    const unsigned rb = blockIdx.x / (2 * sb), half_col = blockIdx.x - rb * 2 * sb, cb = half_col >> 1;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int at = static_cast<int>(half_col & 1) * 16 + (lane & 15);
    const long long r0 = static_cast<long long>(rb) * kF8Block + warp * 8;
    const uint8_t* blk[4];
    bool live[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const long long r = r0 + 2 * p + (lane >> 4);
        live[p] = WHOLE || r < n;
        blk[p] = blocks + (r * sb + cb) * kBytes;
    }
    const long long rs = r0 + (lane >> 2);
    float v[4][8];
    dequant4x8<KIND>(blk, live, blocks + (rs * sb + cb) * kBytes, WHOLE || rs < n, lane, at, v);
    uint32_t m = 0;
#pragma unroll
    for (int p = 0; p < 4; ++p) m = max(m, mag_max(v[p]));
    m = cta_max<kKqThreads>(m, red);
    const float s = f8_scale(__uint_as_float(m));
    if (threadIdx.x == 0) {
        if (!mag_finite(m)) report(err, kErrNonFinite);
        scales[blockIdx.x] = s;
    }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        if (!live[p]) continue;
        uint8_t* dst = out + (r0 + 2 * p + (lane >> 4)) * ld8 + cb * 256;
        uint32_t code[2];
        f8_codes(v[p], s, code);
        if constexpr (KIND == kQ6K) {
            // slots t and 4 + t are neighbours
            const int base = 128 * (at >> 4) + (at & 15) * 2;
#pragma unroll
            for (int t = 0; t < 4; ++t)
                *reinterpret_cast<uint16_t*>(dst + base + 32 * t) =
                    static_cast<uint16_t>(__byte_perm(code[0], code[1], t | ((4 + t) << 4)));
        } else {
            const int base = 64 * (at >> 3) + (at & 7) * 4;
            *reinterpret_cast<uint32_t*>(dst + base) = code[0];
            *reinterpret_cast<uint32_t*>(dst + base + 32) = code[1];
        }
    }
}

template <class T>
int prep_dense(const T* w, int n, int k, long long ldw, int count, uint8_t* out, long long ld8, float* scales,
               int* err, cudaStream_t s) {
    const unsigned nb = (n + kF8Block - 1) / kF8Block, kb = (k + kF8Block - 1) / kF8Block;
    const unsigned long long grid = static_cast<unsigned long long>(nb) * kb * count;
    if (grid > 0x7fffffffull) return cudaErrorInvalidValue;
    const bool vout = reinterpret_cast<uintptr_t>(out) % 8 == 0 && ld8 % 8 == 0;
    const bool vec = reinterpret_cast<uintptr_t>(w) % 16 == 0 && (ldw * sizeof(T)) % 16 == 0 && vout;
    auto kern = !vout                          ? prep_f8_dense_kernel<T, false, false, false>
                : !vec                         ? prep_f8_dense_kernel<T, false, true, false>
                : n % kF8Block || k % kF8Block ? prep_f8_dense_kernel<T, true, true, false>
                                               : prep_f8_dense_kernel<T, true, true, true>;
    kern<<<static_cast<unsigned>(grid), kPrepThreads, 0, s>>>(w, n, k, ldw, nb, kb, out, ld8, scales, err);
    return cudaGetLastError();
}

template <int KIND>
int prep_kq(const uint8_t* blocks, int n, unsigned sb, unsigned grid, uint8_t* out, long long ld8, float* scales, int* err,
            cudaStream_t s) {
    auto kern = n % kF8Block == 0 ? prep_f8_kq_kernel<KIND, true> : prep_f8_kq_kernel<KIND, false>;
    kern<<<grid, kKqThreads, 0, s>>>(blocks, n, sb, out, ld8, scales, err);
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
    const unsigned long long grid = static_cast<unsigned long long>(nb) * sb * 2;
    if (grid > 0x7fffffffull) return cudaErrorInvalidValue;
    const unsigned g = static_cast<unsigned>(grid);
    switch (kind) {
        case kQ4K: return prep_kq<kQ4K>(blocks, n, sb, g, out, ld8, scales, err, s);
        case kQ5K: return prep_kq<kQ5K>(blocks, n, sb, g, out, ld8, scales, err, s);
        case kQ6K: return prep_kq<kQ6K>(blocks, n, sb, g, out, ld8, scales, err, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace rk
