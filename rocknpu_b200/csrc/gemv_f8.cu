// The block-scaled e4m3 product for a few tokens; gemm_f8.cu says what is
// computed.
//
// With up to 8 tokens the product is a stream of the weights from HBM, and a
// short one is over in microseconds, so here the weights go from memory to
// registers, 32 bytes per load, with no stage, barrier or tile exchange in
// between: 1 x 2048 x 5632 f32 takes 5.6 us, 10.9 by the quantiser and
// gemm_f8.cu; 1 x 8192 x 28672 44 us (5.3 TB/s), 57 by those.  Four blocks are on
// their way per warp (three or two: the long one 47 us; six spill, 58).
//
// A warp multiplies 16 weight rows by a block of 128 at a time: e4m3 -> f16
// (exact) into mma.sync m16n8k16, tokens as the 8 columns; f32 sums of a
// block times the two scales are added to f32 totals.  The sum over k may run
// in any order, so thread (g, t) takes the 32 consecutive bytes 32 t .. of
// rows g and g + 8, and the activations lie in shared memory in the order in
// which the threads then need them, as f16, a padded 320 bytes per token and
// block (an odd multiple of 64: two tokens' 64-byte reads fall into different banks).
//
// Tiles of 16 rows are dealt evenly to the CTAs, one per SM.  The warps of a
// CTA share a tile's blocks of k (as many as there are blocks, up to all 16;
// neighbours in k, so that a row is read in long pieces) and add their totals
// through shared memory in a fixed order; tiles are not cut across CTAs.
//
// Activations are e4m3 codes or, for short rows (every CTA then does all of
// it), dense values that each CTA quantises itself, which saves a launch.
#include <algorithm>

#include "f8.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace rk {
namespace {

constexpr int kWarps = 16;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;       // weight rows of a tile
constexpr int kAhead = 4;       // blocks on their way per warp
constexpr int kActBytes = 320;  // 128 f16 values, their f32 scale, padding
constexpr int kPitch = 20;      // floats per token of a warp's totals (bank spread)
constexpr int kMaxItems = 256;  // blocks of activations

struct GemvParams {
    const void* a;  // codes or dense values
    long long lda;
    const float* a_scale;  // codes only
    long long ld_as;
    const uint8_t* w;
    long long ldw;
    const float* w_scale;
    void* out;
    long long ldo;
    int out_type, m, n, k, num_kb, tiles, ways;
    int wide;  // dense rows can be read 16 bytes at a time
    int* err;
};

constexpr int kPartBytes = 2 * kWarps * 8 * kPitch * 4;

// 32 consecutive bytes at a 32-byte boundary.
__device__ __forceinline__ void load32(const uint8_t* p, uint32_t (&w)[8]) {
    asm volatile("ld.global.nc.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                 : "l"(p));
}

// Two e4m3 bytes -> two f16, exactly.
__device__ __forceinline__ uint32_t half2_of(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(two)));
    return r;
}

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// All activations to shared memory, [block][token]: a half-warp per token and
// block, 8 values per lane.  Byte of value k in a row: thread t = k / 32 reads
// its four 16-byte chunks j = (k % 32) / 8 at (4 j + t) * 16.  One item per
// step: several with overlapping loads were 1 us faster with 8 tokens, but 0.4 us
// slower with one, for a kernel that is fetched cold each time.
template <class A>
__device__ __forceinline__ void fill(const GemvParams& p, uint8_t* act) {
    const int l = threadIdx.x & 15, half = threadIdx.x >> 4, items = p.m * p.num_kb;
    uint32_t most = 0;
    // the two halves of a warp take the same steps
    for (int i = half; i - (half & 1) < items; i += kThreads / 16) {
        const int kb = i < items ? i / p.m : p.num_kb, tok = i < items ? i - kb * p.m : 0, col = kb * kF8Block + l * 8;
        uint32_t code[2] = {0u, 0u};
        float s = 0.0f;
        if constexpr (sizeof(A) == 1) {
            // k is a multiple of 32, rows start at multiples of 16 bytes
            if (col < p.k) {
                const uint2 v =
                    __ldg(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(p.a) + tok * p.lda + col));
                code[0] = v.x, code[1] = v.y;
            }
            if (i < items && l == 0) s = __ldg(p.a_scale + tok * p.ld_as + kb);
        } else {
            const A* row = static_cast<const A*>(p.a) + tok * p.lda;
            Raw8<A> raw;
            if (p.wide && col < p.k)
                raw.load(row + col);
            else
                raw.load_some(row + col, p.k - col);
            float v[8];
            raw.values(v);
            uint32_t m = raw.mag_max();
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            most = max(most, m);
            s = f8_scale(__uint_as_float(m));
            f8_codes(v, s, code);
        }
        if (i < items) {
            uint8_t* row = act + i * kActBytes;
            *reinterpret_cast<uint4*>(row + ((l & 3) * 4 + (l >> 2)) * 16) =
                make_uint4(half2_of(code[0] & 0xFFFFu), half2_of(code[0] >> 16), half2_of(code[1] & 0xFFFFu),
                           half2_of(code[1] >> 16));
            if (l == 0) *reinterpret_cast<float*>(row + 256) = s;
        }
    }
    if (!mag_finite(most) && blockIdx.x == 0) report(p.err, kErrNonFinite);
}

template <class T>
__device__ __forceinline__ void store(const GemvParams& p, int tok, int row, float v) {
    static_cast<T*>(p.out)[tok * p.ldo + row] = from_f32<T>(v);
}

// A: uint8_t (codes) or the dense type.
template <class A>
__global__ void __launch_bounds__(kThreads, 1) gemv_f8_kernel(const __grid_constant__ GemvParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    float* part = reinterpret_cast<float*>(smem);
    uint8_t* act = smem + kPartBytes;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int teams = kWarps / p.ways, team = warp / p.ways, way = warp - team * p.ways;
    const int t0 = static_cast<int>(static_cast<long long>(blockIdx.x) * p.tiles / gridDim.x);
    const int t1 = static_cast<int>((static_cast<long long>(blockIdx.x) + 1) * p.tiles / gridDim.x);
    const int nb = (p.num_kb - way + p.ways - 1) / p.ways;  // this warp's blocks of a tile

    // weights on their way, and the next to ask for
    uint32_t lo[kAhead][8], hi[kAhead][8];
    float sw[kAhead];
    int ask_tile = t0 + team, ask_kb = way;
    auto ask = [&](uint32_t(&l)[8], uint32_t(&h)[8], float& s) {
        const int col = ask_kb * kF8Block + t * 32;
        if (ask_tile < t1 && col < p.k) {
            // rows behind the last repeat it; nothing of them is kept
            const int row = ask_tile * kRows + g;
            load32(p.w + min(row, p.n - 1) * p.ldw + col, l);
            load32(p.w + min(row + 8, p.n - 1) * p.ldw + col, h);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) l[i] = h[i] = 0u;
        }
        if (ask_tile < t1) s = __ldg(p.w_scale + static_cast<long long>(ask_tile / (kF8Block / kRows)) * p.num_kb + ask_kb);
        ask_kb += p.ways;
        if (ask_kb >= p.num_kb) {
            ask_kb = way;
            ask_tile += teams;
        }
    };
#pragma unroll
    for (int d = 0; d < kAhead; ++d) ask(lo[d], hi[d], sw[d]);
    fill<A>(p, act);
    __syncthreads();

    // this lane's token's row of a block, and its two columns' scales; columns
    // behind the last token repeat it, nothing of them is kept
    const int at = min(g, p.m - 1) * kActBytes + t * 16;
    const int at0 = min(2 * t, p.m - 1) * kActBytes + 256, at1 = min(2 * t + 1, p.m - 1) * kActBytes + 256;
    float acc[4] = {};
    int tile = t0 + team, done = 0, buf = 0;
    while (tile < t1) {
#pragma unroll
        for (int d = 0; d < kAhead; ++d) {
            if (tile >= t1) break;
            const uint8_t* rows = act + (way + done * p.ways) * p.m * kActBytes;
            float sums[2][4] = {};  // two chains of MMAs
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t a[2][4];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t l = lo[d][2 * c + j], h = hi[d][2 * c + j];
                    a[j][0] = half2_of(l & 0xFFFFu);
                    a[j][1] = half2_of(h & 0xFFFFu);
                    a[j][2] = half2_of(l >> 16);
                    a[j][3] = half2_of(h >> 16);
                }
                const uint4 b = *reinterpret_cast<const uint4*>(rows + at + c * 64);
                mma(sums[0], a[0][0], a[0][1], a[0][2], a[0][3], b.x, b.y);
                mma(sums[1], a[1][0], a[1][1], a[1][2], a[1][3], b.z, b.w);
            }
            const float s0 = *reinterpret_cast<const float*>(rows + at0) * sw[d];
            const float s1 = *reinterpret_cast<const float*>(rows + at1) * sw[d];
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = fmaf(sums[0][i] + sums[1][i], i & 1 ? s1 : s0, acc[i]);
            ask(lo[d], hi[d], sw[d]);
            if (++done < nb) continue;
            // The tile's totals.  Two sets of places: whoever writes one again
            // has passed the barrier of the tile between, which the readers
            // of this one reach after reading.
            float* mine = part + (buf * kWarps + warp) * 8 * kPitch;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                mine[(2 * t + (i & 1)) * kPitch + g + 8 * (i >> 1)] = acc[i];
                acc[i] = 0.0f;
            }
            if (p.ways > 1)
                asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "r"(p.ways * 32) : "memory");
            else
                __syncwarp();
            const float* first = part + (buf * kWarps + team * p.ways) * 8 * kPitch;
            for (int i = way * 32 + lane; i < kRows * p.m; i += p.ways * 32) {
                const int r = i & (kRows - 1), tok = i / kRows, row = tile * kRows + r;
                float v = 0.0f;
                for (int w = 0; w < p.ways; ++w) v += first[(w * 8 + tok) * kPitch + r];
                if (row < p.n) {
                    if (p.out_type == kTypeF32)
                        store<float>(p, tok, row, v);
                    else if (p.out_type == kTypeF16)
                        store<__half>(p, tok, row, v);
                    else
                        store<__nv_bfloat16>(p, tok, row, v);
                }
            }
            done = 0;
            buf ^= 1;
            tile += teams;
        }
    }
}

// Launched without programmatic dependence: beside the quantiser's CTAs this
// kernel's would get their carveout, nearly all of it shared memory, and the
// loads on their way need the L1 cache (1.4 times the time at 8192 x 28672).
template <class A>
int launch_cfg(const GemvParams& p, cudaStream_t s) {
    auto kern = gemv_f8_kernel<A>;
    static bool attr_done[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             kPartBytes + kMaxItems * kActBytes);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    kern<<<std::min(p.tiles, sm_count()), kThreads, kPartBytes + p.m * p.num_kb * kActBytes, s>>>(p);
    return cudaGetLastError();
}

}  // namespace

// Few enough activations that the L1 cache keeps room for the loads (rows of
// 8192: 4 tokens 48 us, 57 us by gemm_f8.cu; 8 tokens, past the limit, 54 and 57 for
// 28672 columns, 14 and 13 for 1024).
bool gemv_f8_fits(const GemmF8& g) {
    return g.m <= 8 && g.k <= kMaxItems * kF8Block && g.m * ((g.k + kF8Block - 1) / kF8Block) <= kMaxItems &&
           g.k % 32 == 0 && g.ldw % 32 == 0 && reinterpret_cast<uintptr_t>(g.w) % 32 == 0;
}

// Up to 128 blocks, four per half-warp, cost less in every CTA than in a launch of
// their own (4096 x 14336: 4 tokens 19.1 us, with a launch 20.4; 8 tokens 23.5 and 21.8).
bool gemv_f8_quantizes(const GemmF8& g) { return g.m * ((g.k + kF8Block - 1) / kF8Block) <= 128; }

int launch_gemv_f8(const GemmF8& g, const void* dense, int type, long long ld, int* err, cudaStream_t s) {
    GemvParams p{};
    p.a = dense ? dense : g.a;
    p.lda = dense ? ld : g.lda;
    p.a_scale = g.a_scale;
    p.ld_as = g.ld_as;
    p.w = g.w;
    p.ldw = g.ldw;
    p.w_scale = g.w_scale;
    p.out = g.out;
    p.ldo = g.ldo;
    p.out_type = g.out_type;
    p.m = g.m;
    p.n = g.n;
    p.k = g.k;
    p.num_kb = (g.k + kF8Block - 1) / kF8Block;
    p.tiles = (g.n + kRows - 1) / kRows;
    p.ways = 1;
    while (p.ways < kWarps && 2 * p.ways <= p.num_kb) p.ways *= 2;
    p.err = err;
    if (!dense) return launch_cfg<uint8_t>(p, s);
    const size_t es = type == kTypeF32 ? 4 : 2;
    p.wide = reinterpret_cast<uintptr_t>(dense) % 16 == 0 && ld * es % 16 == 0;
    switch (type) {
        case kTypeF32: return launch_cfg<float>(p, s);
        case kTypeF16: return launch_cfg<__half>(p, s);
        case kTypeBF16: return launch_cfg<__nv_bfloat16>(p, s);
        default: return cudaErrorInvalidValue;
    }
}

}  // namespace rk
