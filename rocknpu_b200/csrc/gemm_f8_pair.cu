// The block-scaled e4m3 product on two-SM pairs (tcgen05 cta_group::2), for
// shapes with many output tiles; gemm_f8.cu says what is computed.
//
// A cluster of two CTAs computes a 256-token x 256-column tile.  Here the
// MMA's M side is tokens: CTA r holds tokens [m0 + 128 r, +128) and weight
// rows [n0 + 128 r, +128) of each block in shared memory (32 KB per CTA and
// block, 64 bytes per cycle at the MMA's rate), one thread of the even CTA
// issues the M = 256, N = 256 MMAs, and each CTA's TMEM receives its 128
// tokens x 256 columns, in one of two buffers.
//
// Tokens are the TMEM lanes, so the scale of a block is one number per thread
// (its token's times its 128 columns', one weight scale block): an epilogue
// thread adds 128 columns with 64 two-wide multiply-adds and reads no shared
// memory, which the MMA's operands fill to half.  Two-wide, because plain f32
// multiply-adds slow the tensor core (measured: an MMA of 128 cycles takes 223
// beside a stream of them, 128 beside two-wide ones).  The totals are 128 registers
// per thread, so the epilogue warps take registers from the others
// (setmaxnreg: 384 threads x 168 = 128 x 40 + 256 x 232).  At a tile's end each warp
// turns its 32 tokens through shared memory, 128 bytes of columns at a time,
// and stores whole lines.
//
// MMA issue.  Whatever a warp reads from shared memory, a barrier included, it
// gets only after the tensor core has accepted the MMAs it issued before
// (about 200 cycles per look, measured with 4 MMAs between looks: 720 cycles
// per block instead of 512), so one warp that waits and issues in turn starves
// the tensor core.  Two warps take turns: one waits for its block's operands
// and TMEM buffer while the other's MMAs run, then for its turn.  One barrier
// per stage, done[s], says both that a block's operands may be overwritten and
// that its sums are in TMEM; the epilogue is never more than the two TMEM
// buffers behind, less than the stages, so it cannot miss a phase.
//
// Measured: 4096 x 8192 x 28672 bf16 1030 us with the quantiser, 1.9 PFLOP/s, at
// the power limit's clocks; 910 us and 2.1 PFLOP/s for a call after idling.  A block
// takes about 890 cycles where its MMAs take 512: an epilogue warp has one TMEM
// load in flight, waits for four of them, and frees the buffer after the last.
//
// Bounded waits as in the int8 pair kernel (gemm_pair.cu).
#include <algorithm>

#include "gemm_f8.cuh"

namespace rk {
namespace f8_detail {
namespace {

constexpr int kTile = 256;
constexpr int kEpiWarps = 8;
constexpr int kThreads = (4 + kEpiWarps) * 32;
constexpr int kBox = 128 * kF8Block;  // 128 rows of either operand, one block
constexpr int kStage = 2 * kBox;
constexpr int kStages = 5;
constexpr int kRowPitch = 144;  // staging: 128 bytes of columns + 16 (bank spread)
constexpr int kStaging = 32 * kRowPitch;
constexpr int kBarOffset = kStages * kStage;
constexpr int kNumBars = 2 * kStages + 5;
constexpr int kStageOffset = (kBarOffset + kNumBars * 8 + 32 + 127) / 128 * 128;
constexpr int kBytes = kStageOffset + kEpiWarps * kStaging + 1024;  // + alignment slack
static_assert(kBytes <= 232448, "shared memory");

struct Tile {
    int n0, m0;
    __device__ __forceinline__ Tile(const F8Params& p, int u) {
        // group_m token tiles advance together, so that a wave's tiles stay in L2
        const int per_group = p.group_m * p.tiles_n;
        const int g = u / per_group, first = g * p.group_m, gsz = min(p.group_m, p.tiles_m - first);
        const int local = u - g * per_group;
        m0 = (first + local % gsz) * kTile;
        n0 = (local / gsz) * kTile;
    }
};

// A warp's 32 tokens x 128 columns (one token per lane) to memory.
template <class T>
__device__ __forceinline__ void store_rows(const F8Params& p, const float2 (&acc2)[64], int m0, int n0, uint8_t* staging,
                                           int lane) {
    float acc[128];
#pragma unroll
    for (int c = 0; c < 64; ++c) acc[2 * c] = acc2[c].x, acc[2 * c + 1] = acc2[c].y;
    constexpr int kPer = 128 / sizeof(T);  // columns per 128-byte piece
    T* out = static_cast<T*>(p.out);
    const bool whole = reinterpret_cast<uintptr_t>(out) % 16 == 0 && p.ldo * sizeof(T) % 16 == 0;
#pragma unroll
    for (int c0 = 0; c0 < 128; c0 += kPer) {
        __syncwarp();
        uint4* mine = reinterpret_cast<uint4*>(staging + lane * kRowPitch);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint32_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(T) == 4) {
                    w[j] = __float_as_uint(acc[c0 + 4 * i + j]);
                } else {
                    T pair[2] = {from_f32<T>(acc[c0 + 8 * i + 2 * j]), from_f32<T>(acc[c0 + 8 * i + 2 * j + 1])};
                    memcpy(&w[j], pair, 4);
                }
            }
            mine[i] = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        if (whole && n0 + c0 + kPer <= p.n) {
            // 8 lanes per 128-byte line, 4 tokens per step
#pragma unroll
            for (int r = 0; r < 32; r += 4) {
                const int tok = r + (lane >> 3);
                const uint4 v = *reinterpret_cast<const uint4*>(staging + tok * kRowPitch + (lane & 7) * 16);
                if (m0 + tok < p.m)
                    *reinterpret_cast<uint4*>(out + static_cast<long long>(m0 + tok) * p.ldo + n0 + c0 +
                                              (lane & 7) * (16 / static_cast<int>(sizeof(T)))) = v;
            }
        } else {
            for (int r = 0; r < 32 && m0 + r < p.m; ++r)
                for (int c = lane; c < kPer; c += 32)
                    if (n0 + c0 + c < p.n)
                        out[static_cast<long long>(m0 + r) * p.ldo + n0 + c0 + c] =
                            reinterpret_cast<const T*>(staging + r * kRowPitch)[c];
        }
    }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gemm_f8_pair_kernel(const __grid_constant__ F8Params p) {
    constexpr int S = kStages;
    extern __shared__ uint8_t smem_raw[];
    // same offset in both CTAs: the MMA addresses the peer's half by it
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + kBarOffset);
    uint64_t* done = full + S;
    uint64_t* tempty = done + S;
    uint64_t* turn = tempty + 2;
    uint64_t* drain = turn + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile uint32_t* abort = tmem_slot + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 2);  // the leader's two producers
            mbar_init(&done[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&turn[b], 1);
            mbar_init(&tempty[b], 2 * kEpiWarps);  // epilogue warps of both CTAs
        }
        mbar_init(drain, 2);  // the two issuers
        *abort = 0u;
        fence_mbar_init();
        prefetch_tmap(&p.tmap_w);
        prefetch_tmap(&p.tmap_a);
    }
    if (warp == 2) {
        tmem_alloc_pair(tmem_slot, 2 * kTile);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    cluster_sync();  // both CTAs' barriers initialised and TMEM allocated
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const int pair = static_cast<int>(blockIdx.x >> 1), npairs = static_cast<int>(gridDim.x >> 1);

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        if (warp < 2 && lane == 0) {
            // ---- producers: warp 0 this CTA's weight rows, warp 1 its tokens ----
            const bool is_w = warp == 0;
            const CUtensorMap* map = is_w ? &p.tmap_w : &p.tmap_a;
            const int off = is_w ? kBox : 0;
            if (!is_w || !p.early_weights) griddep_wait();
            int g = 0;
            bool ok = true;
            for (int u = pair; ok && u < p.total; u += npairs) {
                const Tile t(p, u);
                const int row = (is_w ? t.n0 : t.m0) + 128 * static_cast<int>(rank);
                for (int kb = 0; kb < p.num_kb; ++kb, ++g) {
                    const int s = g % S;
                    if (g >= S && !wait_or_abort(&done[s], ((g / S) & 1) ^ 1, abort)) {
                        if (!*abort) fail(p.err, abort, kErrTimeoutEmpty);
                        ok = false;
                        break;
                    }
                    // the leader expects both CTAs' bytes of this operand
                    if (leader) mbar_arrive_expect_tx(&full[s], 2 * kBox);
                    tma_load_2d_pair(smem + s * kStage + off, map, map_cluster(smem_u32(&full[s]), 0), kb * kF8Block,
                                     row);
                }
            }
            // every stage filled here must be consumed (so its copy has landed) before the CTA leaves
            for (int i = max(0, g - S); i < g; ++i) {
                if (!mbar_wait(&done[i % S], (i / S) & 1)) {
                    report(p.err, kErrTimeoutDrain);
                    break;
                }
            }
        } else if (warp >= 2 && lane == 0 && leader) {
            // ---- MMA issuers (even CTA), taking turns: warp 2 the even blocks
            // with TMEM buffer 0, warp 3 the odd ones with buffer 1 ----
            constexpr uint32_t idesc = make_idesc<2>(kTile, kTile);
            const int b = warp - 2;
            const int blocks = (p.total - pair + npairs - 1) / npairs * p.num_kb;
            for (int g = b; g < blocks; g += 2) {
                const int s = g % S;
                if (!wait_or_abort(&full[s], (g / S) & 1, abort)) {
                    if (!*abort) fail(p.err, abort, kErrTimeoutFull);
                    break;
                }
                // the other warp has issued block g - 1
                if (g > 0 && !wait_or_abort(&turn[b], ((g - 1) >> 1) & 1, abort)) {
                    if (!*abort) fail(p.err, abort, kErrTimeoutFull);
                    break;
                }
                // the last of the three to come: this buffer has been read out
                if (g >= 2 && !wait_or_abort(&tempty[b], ((g >> 1) & 1) ^ 1, abort)) {
                    if (!*abort) fail(p.err, abort, kErrTimeoutAccum);
                    break;
                }
                tc_fence_after();
                const uint32_t ta = smem_u32(smem + s * kStage);
#pragma unroll
                for (int ks = 0; ks < kF8Block / 32; ++ks)
                    tc_mma_pair<2>(tmem_base + b * kTile, smem_desc_k128(ta + ks * 32),
                                   smem_desc_k128(ta + kBox + ks * 32), idesc, ks != 0 ? 1u : 0u);
                mbar_arrive(&turn[b ^ 1]);
                tc_commit_pair(&done[s], 0x3);
            }
            // the pair's MMAs must finish before either CTA releases TMEM
            tc_commit_pair(drain, 0x3);
            if (!mbar_wait(drain, 0)) report(p.err, kErrTimeoutDrain);
        } else if (warp == 2 && lane == 0) {
            // odd CTA: the leader's MMAs write this CTA's TMEM too
            if (!mbar_wait(drain, 0)) report(p.err, kErrTimeoutDrain);
        }
        __syncwarp();
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        // ---- epilogue warps 4..11 ----
        const int e = warp - 4, q = warp & 3, half = e >> 2;
        uint8_t* staging = smem + kStageOffset + e * kStaging;
        const uint32_t tempty_leader = map_cluster(smem_u32(&tempty[0]), 0);
        griddep_wait();
        int g = 0;
        bool ok = true;
        for (int u = pair; u < p.total; u += npairs) {
            const Tile t(p, u);
            const int m0 = t.m0 + 128 * static_cast<int>(rank) + q * 32, n0 = t.n0 + half * 128;
            // columns past n read a scale that exists; their sums are not stored
            const float* ws = p.w_scale + static_cast<long long>(min(n0, p.n - 1) / kF8Block) * p.num_kb;
            const float* as = p.a_scale + static_cast<long long>(min(m0 + lane, p.m - 1)) * p.ld_as;
            float2 acc[64];
#pragma unroll
            for (int c = 0; c < 64; ++c) acc[c] = make_float2(0.0f, 0.0f);
            // A block's 128 columns in four pieces; the next piece is on its way
            // while one is added, the next block's first piece included.
            auto ready = [&](int i) {
                if (!wait_or_abort(&done[i % S], (i / S) & 1, abort)) {
                    if (!*abort) fail(p.err, abort, kErrTimeoutAccum);
                    ok = false;  // of this lane; the others' may still have come
                }
                __syncwarp();
                tc_fence_after();
            };
            const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(half * 128);
            auto add = [&](int c, const uint32_t(&r)[32], float s) {
                const float2 ss = make_float2(s, s);
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    acc[c * 16 + j] = __ffma2_rn(make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1])), ss,
                                                 acc[c * 16 + j]);
            };
            // scales two blocks ahead
            const int last = p.num_kb - 1;
            float s = ld_global(as) * ld_global(ws), a1 = ld_global(as + min(1, last)), w1 = ld_global(ws + min(1, last));
            uint32_t r0[32], r1[32];
            ready(g);
            tmem_ld32(lane_base + (g & 1) * kTile, r0);
            // unrolled, so that the carried piece stays in place (1089 -> 1015 us at
            // 4096 x 28672 x 8192)
#pragma unroll 4
            for (int kb = 0; kb < p.num_kb; ++kb, ++g) {
                const float a2 = ld_global(as + min(kb + 2, last)), w2 = ld_global(ws + min(kb + 2, last));
                const uint32_t base = lane_base + (g & 1) * kTile;
                tmem_ld_wait();
                tmem_ld32(base + 32, r1);
                add(0, r0, s);
                tmem_ld_wait();
                tmem_ld32(base + 64, r0);
                add(1, r1, s);
                tmem_ld_wait();
                tmem_ld32(base + 96, r1);
                add(2, r0, s);
                tmem_ld_wait();
                // read out: this CTA's half of the buffer is free
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (leader)
                        mbar_arrive(&tempty[g & 1]);
                    else
                        mbar_arrive_remote_relaxed(tempty_leader + (g & 1) * 8);
                }
                if (kb < last) {
                    ready(g + 1);
                    tmem_ld32(lane_base + ((g + 1) & 1) * kTile, r0);
                }
                add(3, r1, s);
                s = a1 * w1;
                a1 = a2;
                w1 = w2;
            }
            ok = __all_sync(0xffffffffu, ok);  // the stores have barriers of the warp
            if (ok) {
                if (p.out_type == kTypeF32)
                    store_rows<float>(p, acc, m0, n0, staging, lane);
                else if (p.out_type == kTypeF16)
                    store_rows<__half>(p, acc, m0, n0, staging, lane);
                else
                    store_rows<__nv_bfloat16>(p, acc, m0, n0, staging, lane);
            }
        }
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    // neither CTA leaves (or releases TMEM) while the pair may still touch
    // its shared memory, barriers or TMEM
    cluster_sync();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 2 * kTile);
    }
}

}  // namespace

int pair_slots() {
    static int slots[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && slots[dev] > 0) return slots[dev];
    int n = 0;
    if (cudaFuncSetAttribute(gemm_f8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes) == cudaSuccess) {
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(2 * 74, 1, 1);
        cfg.blockDim = dim3(kThreads, 1, 1);
        cfg.dynamicSmemBytes = kBytes;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 2;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&n, gemm_f8_pair_kernel, &cfg) != cudaSuccess) n = 0;
    }
    cudaGetLastError();
    if (n <= 0) n = sm_count() / 2 - 4;  // conservative when the query fails
    if (dev >= 0 && dev < 64) slots[dev] = n;
    return n;
}

int launch_pair(const F8Params& p, int npairs, cudaStream_t s) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(2 * npairs), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = kBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, gemm_f8_pair_kernel, p);
}

}  // namespace f8_detail
}  // namespace rk
