// out[m, n] = sum_b a_s[m, b] * w_s[n / 128, b] * sum_{k in block b} a[m, k] * w[n, k]
// with e4m3 a and w and blocks of 128 along k: the product of activations with
// a scale per row and block and weights with a scale per 128 x 128 block.
//
// A block of 128 e4m3 values is one 128-byte swizzle row, so one pipeline
// stage is one scale block: four kind::f8f6f4 MMAs (K = 32) give its exact
// products summed in f32 in TMEM, and the epilogue warps add that sum, times
// the two scales, to f32 accumulators in registers while the tensor core
// works on the next block in another TMEM buffer.
//
// Orientation as in the int8 GEMM: the MMA's M side is 128 weight rows
// (lane = output column, so stores are whole 128-byte lines), its N side BT
// tokens; a tile's 128 weight rows share one weight scale per block.
//
// Work: tiles of 128 x BT, either whole tiles per CTA, or ("stream") the
// blocks of all tiles in one line cut evenly over the CTAs.  A tile cut by a
// range border is summed by the CTA that finishes it last, from the
// contributors' f32 partial tiles in the order of the blocks: the result does
// not depend on which CTA that is.
//
// Launch: programmatic dependent launch behind the quantiser.  Every wait is
// bounded as in the int8 GEMM.
//
// Measured: 16 x 8192 x 28672 bf16 56 us with the quantiser, 4.2 TB/s of weights
// in boxes of 128-byte rows (a flat copy of cold memory: 5.2).
#include <algorithm>

#include "gemm_f8.cuh"

namespace rk {
namespace {

using f8_detail::F8Params;
using f8_detail::fail;

constexpr int kEpiWarps = 8;
constexpr int kEpiThreads = kEpiWarps * 32;
constexpr int kThreads = (3 + kEpiWarps) * 32;
constexpr int kWRows = 128;
constexpr int kWBox = kWRows * kF8Block;

template <int BT>
struct F8Cfg {
    static constexpr int kABox = BT * kF8Block;
    static constexpr int kStage = kWBox + kABox;
    static constexpr int kStages = std::min(12, (200 * 1024) / kStage);
    static constexpr int kBufs = 512 / BT < 4 ? 512 / BT : 4;
    static constexpr int kCols = BT / 2;  // columns per epilogue warp
    static constexpr int kBarOffset = kStages * kStage;
    static constexpr int kNumBars = 2 * kStages + 2 * kBufs + 1;
    static constexpr int kScaleOffset = (kBarOffset + kNumBars * 8 + 32 + 15) & ~15;
    static constexpr int kBytes = kScaleOffset + kEpiWarps * 2 * kCols * 4 + 1024;  // + alignment slack
    static constexpr uint32_t kTmemCols = kBufs * BT;
    static_assert(kTmemCols >= 32 && kTmemCols <= 512 && (kTmemCols & (kTmemCols - 1)) == 0, "TMEM");
    static_assert(kBytes <= 232448, "shared memory");
};

struct Seg {
    int tile, n0, m0, kb0, kb1;
};

// First block of CTA c's range of the line.
__device__ __forceinline__ int range_start(const F8Params& p, int c) {
    return static_cast<int>(static_cast<long long>(c) * p.total / static_cast<int>(gridDim.x));
}

// The CTA whose range holds block x of the line.
__device__ __forceinline__ int range_of(const F8Params& p, int x) {
    return static_cast<int>(((static_cast<long long>(x) + 1) * static_cast<int>(gridDim.x) - 1) / p.total);
}

template <int BT>
struct Walk {
    int cur, end;
    __device__ __forceinline__ explicit Walk(const F8Params& p) {
        cur = p.stream ? range_start(p, blockIdx.x) : static_cast<int>(blockIdx.x);
        end = p.stream ? range_start(p, blockIdx.x + 1) : p.total;
    }
    __device__ __forceinline__ bool next(const F8Params& p, Seg& s) {
        if (cur >= end) return false;
        if (p.stream) {
            s.tile = cur / p.num_kb;
            s.kb0 = cur - s.tile * p.num_kb;
            s.kb1 = min(p.num_kb, s.kb0 + (end - cur));
            cur += s.kb1 - s.kb0;
        } else {
            s.tile = cur;
            s.kb0 = 0;
            s.kb1 = p.num_kb;
            cur += gridDim.x;
        }
        // group_m token tiles advance together, so that a wave's tiles stay in L2
        const int per_group = p.group_m * p.tiles_n;
        const int g = s.tile / per_group;
        const int first_m = g * p.group_m;
        const int gsz = min(p.group_m, p.tiles_m - first_m);
        const int local = s.tile - g * per_group;
        s.m0 = (first_m + local % gsz) * BT;
        s.n0 = (local / gsz) * kWRows;
        return true;
    }
};

// The epilogue warps' barrier; whether any of their threads passed true.
__device__ __forceinline__ bool epi_any(bool v) {
    uint32_t r;
    asm volatile(
        "{\n"
        " .reg .pred p, q;\n"
        " setp.ne.u32 p, %1, 0;\n"
        " bar.red.or.pred q, 1, %2, p;\n"
        " selp.u32 %0, 1, 0, q;\n"
        "}\n"
        : "=r"(r)
        : "r"(v ? 1u : 0u), "n"(kEpiThreads)
        : "memory");
    return r != 0;
}

__device__ __forceinline__ void epi_bar() { asm volatile("bar.sync 1, %0;" ::"n"(kEpiThreads) : "memory"); }

template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t* r) {
    if constexpr (N == 8) {
        tmem_ld8(addr, r);
    } else if constexpr (N == 16) {
        tmem_ld16(addr, *reinterpret_cast<uint32_t(*)[16]>(r));
    } else {
        tmem_ld32(addr, r);
    }
}

// This thread's output column of a tile: kCols tokens from m0.
template <int COLS, class T>
__device__ __forceinline__ void store_cols(const F8Params& p, const float (&acc)[COLS], int m0, int col) {
    if (col >= p.n) return;
    T* o = static_cast<T*>(p.out) + static_cast<long long>(m0) * p.ldo + col;
    if (m0 + COLS <= p.m) {
#pragma unroll
        for (int c = 0; c < COLS; ++c) o[c * p.ldo] = from_f32<T>(acc[c]);
    } else {
#pragma unroll
        for (int c = 0; c < COLS; ++c)
            if (m0 + c < p.m) o[c * p.ldo] = from_f32<T>(acc[c]);
    }
}

template <int COLS>
__device__ __forceinline__ void store_tile(const F8Params& p, const float (&acc)[COLS], int m0, int col) {
    if (p.out_type == kTypeF32)
        store_cols<COLS, float>(p, acc, m0, col);
    else if (p.out_type == kTypeF16)
        store_cols<COLS, __half>(p, acc, m0, col);
    else
        store_cols<COLS, __nv_bfloat16>(p, acc, m0, col);
}

template <int BT>
__global__ void __launch_bounds__(kThreads, 1) gemm_f8_kernel(const __grid_constant__ F8Params p) {
    using C = F8Cfg<BT>;
    constexpr int S = C::kStages, B = C::kBufs, COLS = C::kCols;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOffset);
    uint64_t* empty = full + S;
    uint64_t* tfull = empty + S;
    uint64_t* tempty = tfull + B;
    uint64_t* drain = tempty + B;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    uint32_t* last_flag = tmem_slot + 1;
    volatile uint32_t* abort = tmem_slot + 2;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 2);
            mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < B; ++b) {
            mbar_init(&tfull[b], 1);
            mbar_init(&tempty[b], kEpiWarps);
        }
        mbar_init(drain, 1);
        *abort = 0u;
        fence_mbar_init();
        prefetch_tmap(&p.tmap_w);
        prefetch_tmap(&p.tmap_a);
    }
    if (warp == 2) {
        tmem_alloc(tmem_slot, C::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    if (warp == 0 || warp == 1) {
        if (lane == 0) {
            // ---- producers: warp 0 weights, warp 1 activations ----
            const bool is_w = warp == 0;
            const CUtensorMap* map = is_w ? &p.tmap_w : &p.tmap_a;
            const uint32_t box = is_w ? kWBox : C::kABox;
            const int off = is_w ? 0 : kWBox;
            if (!is_w || !p.early_weights) griddep_wait();
            Walk<BT> walk(p);
            Seg t;
            int g = 0;
            bool ok = true;
            while (ok && walk.next(p, t)) {
                const int row = is_w ? t.n0 : t.m0;
                for (int kb = t.kb0; kb < t.kb1; ++kb, ++g) {
                    const int s = g % S;
                    if (g >= S && !wait_or_abort(&empty[s], ((g / S) & 1) ^ 1, abort)) {
                        if (!*abort) fail(p.err, abort, kErrTimeoutEmpty);
                        ok = false;
                        break;
                    }
                    mbar_arrive_expect_tx(&full[s], box);
                    tma_load_2d(smem + s * C::kStage + off, map, &full[s], kb * kF8Block, row);
                }
            }
            // copies in flight must land before the CTA exits
            for (int i = max(0, g - S); i < g; ++i) {
                if (!mbar_wait(&full[i % S], (i / S) & 1)) {
                    report(p.err, kErrTimeoutDrain);
                    break;
                }
            }
        }
    } else if (warp == 2) {
        if (lane == 0) {
            // ---- MMA issuer: one TMEM buffer per block ----
            constexpr uint32_t idesc = make_idesc<2>(kWRows, BT);
            Walk<BT> walk(p);
            Seg t;
            int g = 0;
            bool ok = true;
            while (ok && walk.next(p, t)) {
                for (int kb = t.kb0; kb < t.kb1; ++kb, ++g) {
                    const int s = g % S, b = g % B;
                    if (g >= B && !wait_or_abort(&tempty[b], ((g / B) & 1) ^ 1, abort)) {
                        if (!*abort) fail(p.err, abort, kErrTimeoutAccum);
                        ok = false;
                        break;
                    }
                    if (!wait_or_abort(&full[s], (g / S) & 1, abort)) {
                        if (!*abort) fail(p.err, abort, kErrTimeoutFull);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t wa = smem_u32(smem + s * C::kStage);
#pragma unroll
                    for (int ks = 0; ks < kF8Block / 32; ++ks)
                        tc_mma<2>(tmem_base + b * BT, smem_desc_k128(wa + ks * 32),
                                  smem_desc_k128(wa + kWBox + ks * 32), idesc, ks != 0 ? 1u : 0u);
                    tc_commit(&empty[s]);
                    tc_commit(&tfull[b]);
                }
            }
            // our MMAs must finish before TMEM is released
            tc_commit(drain);
            if (!mbar_wait(drain, 0)) report(p.err, kErrTimeoutDrain);
        }
        __syncwarp();
    } else {
        // ---- epilogue warps 3..10 ----
        const int e = warp - 3;
        const int q = warp & 3;   // TMEM lane quarter this warp may access
        const int half = e >> 2;  // which half of the tile's tokens
        const int etid = threadIdx.x - 96;
        constexpr int kPer = (COLS + 31) / 32;  // token scales per lane
        constexpr int kChunk = COLS < 32 ? COLS : 32;
        float* slice = reinterpret_cast<float*>(smem + C::kScaleOffset) + e * 2 * COLS;
        griddep_wait();
        Walk<BT> walk(p);
        Seg t;
        int g = 0;
        bool ok = true;
        while (walk.next(p, t)) {
            const float* ws = p.w_scale + static_cast<long long>(t.n0 / kWRows) * p.num_kb;
            const int m0 = t.m0 + half * COLS;
            const float* as[kPer];
#pragma unroll
            for (int i = 0; i < kPer; ++i) as[i] = p.a_scale + static_cast<long long>(min(m0 + lane + 32 * i, p.m - 1)) * p.ld_as;
            // the next block's scales are loaded one block ahead
            float sa[kPer], sw = ld_global(ws + t.kb0);
#pragma unroll
            for (int i = 0; i < kPer; ++i) sa[i] = ld_global(as[i] + t.kb0);
            float acc[COLS];
#pragma unroll
            for (int c = 0; c < COLS; ++c) acc[c] = 0.0f;
            for (int kb = t.kb0; ok && kb < t.kb1; ++kb, ++g) {
                const int b = g % B;
                float* sc = slice + (g & 1) * COLS;
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    if (lane + 32 * i < COLS) sc[lane + 32 * i] = sa[i] * sw;
                const int nkb = min(kb + 1, t.kb1 - 1);
                sw = ld_global(ws + nkb);
#pragma unroll
                for (int i = 0; i < kPer; ++i) sa[i] = ld_global(as[i] + nkb);
                __syncwarp();
                int ready = 0;
                if (lane == 0) ready = wait_or_abort(&tfull[b], (g / B) & 1, abort) ? 1 : 0;
                ready = __shfl_sync(0xffffffffu, ready, 0);
                if (!ready) {
                    if (lane == 0 && !*abort) fail(p.err, abort, kErrTimeoutAccum);
                    ok = false;  // this warp stores nothing more, but joins the others' barriers
                    break;
                }
                tc_fence_after();
                const uint32_t base = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + b * BT + half * COLS;
#pragma unroll
                for (int c0 = 0; c0 < COLS; c0 += kChunk) {
                    uint32_t r[kChunk];
                    tmem_ld<kChunk>(base + c0, r);
                    tmem_ld_wait();
#pragma unroll
                    for (int c = 0; c < kChunk; c += 4) {
                        const float4 s4 = *reinterpret_cast<const float4*>(sc + c0 + c);
                        acc[c0 + c] = fmaf(__uint_as_float(r[c]), s4.x, acc[c0 + c]);
                        acc[c0 + c + 1] = fmaf(__uint_as_float(r[c + 1]), s4.y, acc[c0 + c + 1]);
                        acc[c0 + c + 2] = fmaf(__uint_as_float(r[c + 2]), s4.z, acc[c0 + c + 2]);
                        acc[c0 + c + 3] = fmaf(__uint_as_float(r[c + 3]), s4.w, acc[c0 + c + 3]);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&tempty[b]);
            }
            const int col = t.n0 + q * 32 + lane;
            if (t.kb1 - t.kb0 == p.num_kb) {
                if (ok) store_tile<COLS>(p, acc, m0, col);
                continue;
            }
            // a cut tile: this CTA's partial sums, then the last contributor adds all
            constexpr int kPart = COLS * kEpiThreads;
            float* mine = p.part + (2ll * blockIdx.x + (t.kb0 == 0 ? 1 : 0)) * kPart + etid;
#pragma unroll
            for (int c = 0; c < COLS; ++c) __stcg(mine + c * kEpiThreads, acc[c]);
            const int x0 = t.tile * p.num_kb;
            const int first = range_of(p, x0), last = range_of(p, x0 + p.num_kb - 1);
            __threadfence();
            if (epi_any(!ok)) {
                ok = false;
                continue;
            }
            if (etid == 0) {
                // a tile that is cut is the last of its first CTA
                const unsigned prev = atomicAdd(p.counters + first, 1u);
                *last_flag = prev == static_cast<unsigned>(last - first) ? 1u : 0u;
                if (*last_flag) p.counters[first] = 0u;
            }
            epi_bar();
            if (*last_flag) {
                __threadfence();
#pragma unroll
                for (int c = 0; c < COLS; ++c) acc[c] = 0.0f;
                for (int cta = first; cta <= last; ++cta) {
                    const float* theirs = p.part + (2ll * cta + (cta == first ? 1 : 0)) * kPart + etid;
#pragma unroll
                    for (int c = 0; c < COLS; ++c) acc[c] += __ldcg(theirs + c * kEpiThreads);
                }
                store_tile<COLS>(p, acc, m0, col);
            }
        }
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem_base, C::kTmemCols);
    }
}

struct F8Plan {
    int bt = 16, grid = 1, tiles = 1;
    bool stream = false, pair = false;
    size_t scratch = 0;
};

// Tile height and distribution, by costs in one unit.  They are fitted so that
// the faster form is chosen and are not the cycles a form takes (a pair's
// block is priced 600 and takes about 890 of them).  A block costs a CTA the
// larger of its MMAs (four of at least 55, and about 150 of barriers and
// commits) and its bytes from L2 at about 60 per unit.  Whole tiles take
// ceil(tiles / SMs) rounds; cut evenly the blocks divide without a remainder,
// but a CTA then writes (and its neighbour reads) up to two partial tiles at
// about 30 bytes per unit.
F8Plan plan_f8(int m, int n, int k) {
    F8Plan pl;
    const int kb = (k + kF8Block - 1) / kF8Block, sms = sm_count();
    double best = 1e300;
    for (int bt : {16, 32, 64, 128}) {
        if (bt > 16 && bt / 2 >= m) break;
        const long long tiles =  // more are refused at the launch
            std::min<long long>(static_cast<long long>((n + kWRows - 1) / kWRows) * ((m + bt - 1) / bt), 0x7fffffff);
        const double block = std::max(4.0 * std::max(55.0, bt / 2.0) + 150.0, (kWRows + bt) * 128 / 60.0);
        const double whole = static_cast<double>((tiles + sms - 1) / sms) * kb * block;
        const long long total = tiles * kb;
        const double cut = static_cast<double>((total + sms - 1) / sms) * block + 1500.0 + kWRows * bt * 8 / 30.0;
        const bool can_cut = total < 0x7fffffffll && tiles % sms != 0;
        const bool stream = can_cut && cut < whole;
        const double cost = stream ? cut : whole;
        if (cost < best) {
            best = cost;
            pl.bt = bt;
            pl.stream = stream;
            pl.tiles = static_cast<int>(tiles);
            pl.grid = static_cast<int>(std::min<long long>(stream ? total : tiles, sms));
            pl.scratch = stream ? static_cast<size_t>(pl.grid) * 2 * kWRows * bt * sizeof(float) : 0;
        }
    }
    // two-SM tiles: 512 cycles of MMAs per block and 256 x 256 outputs; 4000 for
    // a tile's start and its stores
    const long long pairs = static_cast<long long>((n + 255) / 256) * ((m + 255) / 256);
    const int slots = m > 128 ? f8_detail::pair_slots() : 0;
    if (slots > 0) {
        const double cost = static_cast<double>((pairs + slots - 1) / slots) * (kb * 600.0 + 4000.0);
        if (cost < best) {
            pl = F8Plan{};
            pl.pair = true;
            pl.bt = 256;
            pl.tiles = static_cast<int>(std::min<long long>(pairs, 0x7fffffff));
            pl.grid = static_cast<int>(std::min<long long>(pairs, slots));
        }
    }
    return pl;
}

template <int BT>
int launch_cfg(const F8Params& p, int grid, cudaStream_t s) {
    using C = F8Cfg<BT>;
    auto kern = gemm_f8_kernel<BT>;
    static bool attr_done[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(grid), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

}  // namespace

size_t gemm_f8_scratch_bytes(int m, int n, int k) { return plan_f8(m, n, k).scratch; }

int launch_gemm_f8(const GemmF8& g, int* err, cudaStream_t s) {
    if (gemv_f8_fits(g)) return launch_gemv_f8(g, nullptr, 0, 0, err, s);
    F8Plan pl = plan_f8(g.m, g.n, g.k);
    if (pl.stream && (!g.counters || !g.scratch || g.scratch_bytes < pl.scratch)) {
        pl.stream = false;
        pl.grid = std::min(pl.tiles, sm_count());
    }
    F8Params p{};
    p.w_scale = g.w_scale;
    p.a_scale = g.a_scale;
    p.ld_as = g.ld_as;
    p.out = g.out;
    p.ldo = g.ldo;
    p.out_type = g.out_type;
    p.m = g.m;
    p.n = g.n;
    p.num_kb = (g.k + kF8Block - 1) / kF8Block;
    const int wt = pl.pair ? 256 : kWRows;
    p.tiles_n = (g.n + wt - 1) / wt;
    p.tiles_m = (g.m + pl.bt - 1) / pl.bt;
    if (static_cast<long long>(p.tiles_n) * p.tiles_m > 0x7fffffffll) return cudaErrorInvalidValue;
    p.group_m = std::min(p.tiles_m, 8);
    p.stream = pl.stream ? 1 : 0;
    p.total = pl.stream ? pl.tiles * p.num_kb : pl.tiles;
    p.early_weights = g.early_weights ? 1 : 0;
    p.part = static_cast<float*>(g.scratch);
    p.counters = g.counters;
    p.err = err;
    if (pl.pair) {
        // each CTA of a pair loads 128 rows of either operand
        if (!make_kmajor_map(&p.tmap_w, g.w, 1, g.k, g.n, g.ldw, 128) ||
            !make_kmajor_map(&p.tmap_a, g.a, 1, g.k, g.m, g.lda, 128))
            return cudaErrorInvalidValue;
        return f8_detail::launch_pair(p, pl.grid, s);
    }
    if (!make_kmajor_map(&p.tmap_w, g.w, 1, g.k, g.n, g.ldw, kWRows)) return cudaErrorInvalidValue;
    if (!make_kmajor_map(&p.tmap_a, g.a, 1, g.k, g.m, g.lda, pl.bt)) return cudaErrorInvalidValue;
    switch (pl.bt) {
        case 16: return launch_cfg<16>(p, pl.grid, s);
        case 32: return launch_cfg<32>(p, pl.grid, s);
        case 64: return launch_cfg<64>(p, pl.grid, s);
        default: return launch_cfg<128>(p, pl.grid, s);
    }
}

}  // namespace rk
