// A whole mixture-of-experts layer for a few tokens in one launch, over
// expert weights in e4m3 with a scale per 128 x 128 block:
//
//   l = x R^T;  top-k experts of each token, softmax weights p
//   h = silu(x Wg_e^T) * (x Wu_e^T);  y = sum over slots of p * (h Wd_e^T)
//
// With a few tokens the layer is a stream of the chosen experts' weights from
// HBM; everything here serves that stream.
//
// Products.  Weights go from TMA stages (128-byte swizzle) to registers,
// e4m3 -> f16 (exact), into mma.sync m16n8k16 with tokens as the 8 columns.
// Activations are not quantised: a block of 128 is scaled by a power of two
// so that its largest magnitude is in [2^14, 2^15) and held in f16; for f32
// calls a second f16 holds the remainder (22 bits in all), for f16 / bf16
// calls the inputs fit one f16 and the hidden values are rounded to 11 bits,
// finer than the result's own rounding for bf16, the same for f16.  Sums are
// f32: 128 products per block in the MMA's accumulator, times the weight
// scale and the activation's power of two, added to f32 totals.
//
// k order.  The sum over k may run in any order, so thread (g, t) of a warp
// takes 32 consecutive bytes 32 t .. of weight row g (two 16-byte reads that
// the swizzle spreads over all banks) and the activations are laid out in
// memory in the order in which the threads then need them.
//
// Work.  A tile is 256 weight rows (128 gate + 128 up rows, or 256 down
// rows); the blocks of all tiles of all chosen experts form one line that is
// cut evenly over the CTAs, one per SM, so no SM idles for a whole tile.  A
// tile cut by a border is finished by the CTA that arrives last on it, from
// the contributors' f32 partial tiles in line order (the result does not
// depend on who that is); the last of a column tile's experts sums the slots
// in slot order.
//
// Phases: (0) router products and the activations' layout; grid barrier; (1)
// every CTA picks the experts for itself, gate / up products, SiLU; grid
// barrier; (2) down products, weighted sum.  The weight copies of phase 2
// start before its barrier.  The launch is cooperative, so all CTAs are
// resident; every wait is bounded all the same.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "f8.cuh"
#include "kernels.h"
#include "ptx.cuh"
#include "quant_math.cuh"

namespace rk {
namespace {

constexpr int kConsumers = 8;                      // warps
constexpr int kConsThreads = kConsumers * 32;
constexpr int kThreads = kConsThreads + 32;        // + the producer warp
constexpr int kBoxRows = 128;
constexpr int kBoxBytes = kBoxRows * kF8Block;
constexpr int kMaxPairs = kMoeMaxTokens * kMoeMaxTop;
constexpr int kRouterTokens = 4;                   // tokens per router task

// Words of the zeroed header.
constexpr int kCut1 = 0, kCut2 = 1024, kBarrier = 2048, kExit = 2049, kCombine = 4096;

struct MoeParams {
    CUtensorMap tm_gate, tm_up, tm_down;  // (k, rows, expert), box 128 B x 128 rows
    const float *gate_s, *up_s, *down_s;
    long long gate_ss, up_ss, down_ss;  // scales of one expert
    const void* x;
    void* out;
    const void* router;
    long long ldx, ldo, ld_router;
    int type, router_type;
    int* ids;
    float* weights;
    int t, h, f, e, top, renorm;
    int kb_h, kb_f, tiles_f, tiles_h;
    unsigned* ctrl;
    float* logits;    // [t][e]
    uint8_t* xq;      // [t][kb_h] activation blocks
    uint8_t* hq;      // [pair][kb_f] activation blocks
    float* part;      // [CTA][2][8 NG][kConsThreads] partial tiles
    float* pair_out;  // [pair][h]
    int* err;
};

// An activation block of 128 values: f16 values (and remainders) in the
// order of the MMA operands, then the f32 power of two.
template <bool LO>
struct ActBlock {
    static constexpr int kScaleAt = LO ? 512 : 256;
    static constexpr int kBytes = kScaleAt + 16;
    // distance of two rows in shared memory: an odd multiple of 64 bytes, so
    // that two rows' 64-byte reads fall into different banks
    static constexpr int kPitch = LO ? 576 : 320;
};

template <int NG, bool LO>
struct MoeCfg {
    using Act = ActBlock<LO>;
    static constexpr int kAct = (NG * 8 * Act::kPitch + 1023) / 1024 * 1024;
    static constexpr int kStage = 2 * kBoxBytes + kAct;
    static constexpr int kStages = (212 * 1024) / kStage;
    static constexpr int kBarOffset = kStages * kStage;
    static constexpr int kTables = kBarOffset + (2 * kStages * 8 + 32 + 15) / 16 * 16;
    static constexpr int kTableBytes = kMaxPairs * (4 + 2 + 2 + 4) + kMoeMaxExperts * 4 + 16 +
                                       kConsumers * kMoeMaxTokens * 4;
    static constexpr int kBytes = kTables + kTableBytes + 1024;  // + alignment slack
    static_assert(kBytes <= 232448, "shared memory");
};

// Routing tables of a CTA, in shared memory.
struct Tables {
    float* pair_w;       // [pair] weight of slot (token * top + slot)
    short* pair_e;       // [pair] its expert, -1: empty
    short* order;        // pairs sorted by expert, then token
    int* entry;          // [entries] expert << 16 | first position in order
    int* count;          // [expert] pairs
    int* info;           // [0] entries, [1] positions
    float* red;          // [kConsumers][kMoeMaxTokens]
};

__device__ __forceinline__ void fail(int* err, volatile uint32_t* abort, int code) {
    atomicCAS(err, 0, code);
    *abort = 1u;
}

__device__ __forceinline__ unsigned ld_acquire(const unsigned* p) {
    unsigned v;
    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

// All threads' earlier writes (ordered before by a CTA barrier) are visible
// to whoever sees the count.
__device__ __forceinline__ void grid_arrive(unsigned* bar) {
    __threadfence();
    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(bar) : "memory");
}

__device__ __forceinline__ bool grid_wait(const unsigned* bar, unsigned need, volatile uint32_t* abort) {
    const uint64_t t0 = globaltimer_ns();
    while (ld_acquire(bar) < need) {
        if (*abort) return false;
        if (globaltimer_ns() - t0 > kWaitLimitNs) return false;
    }
    return true;
}

__device__ __forceinline__ void cons_bar() { asm volatile("bar.sync 2, %0;" ::"n"(kConsThreads) : "memory"); }

// The same barrier; whether any consumer thread passed true.
__device__ __forceinline__ bool cons_any(bool v) {
    uint32_t r;
    asm volatile(
        "{\n"
        " .reg .pred p, q;\n"
        " setp.ne.u32 p, %1, 0;\n"
        " bar.red.or.pred q, 2, %2, p;\n"
        " selp.u32 %0, 1, 0, q;\n"
        "}\n"
        : "=r"(r)
        : "r"(v ? 1u : 0u), "n"(kConsThreads)
        : "memory");
    return r != 0;
}

__device__ __forceinline__ float load_dense(const void* p, int type, long long i) {
    if (type == kTypeF32) return __ldg(static_cast<const float*>(p) + i);
    if (type == kTypeF16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void store_dense(void* p, int type, long long i, float v) {
    if (type == kTypeF32)
        static_cast<float*>(p)[i] = v;
    else if (type == kTypeF16)
        static_cast<__half*>(p)[i] = __float2half_rn(v);
    else
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// Power of two s with amax / s in [2^14, 2^15) (1 for a block of zeros, at
// least 2^-126), and its exact reciprocal.
__device__ __forceinline__ float act_scale(float amax, float& inv) {
    const uint32_t ex = (__float_as_uint(amax) >> 23) & 0xFFu;
    const uint32_t se = amax == 0.0f ? 127u : (ex > 15u ? ex - 14u : 1u);
    inv = __uint_as_float((254u - se) << 23);
    return __uint_as_float(se << 23);
}

// Byte of value k (0..127) in an activation block: thread t = k / 32 reads
// 16-byte chunk j = (k % 32) / 8 at (4 j + t) * 16.
__device__ __forceinline__ int act_at(int k) { return (((k >> 3) & 3) * 4 + (k >> 5)) * 16 + (k & 7) * 2; }

__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    uint32_t r;
    memcpy(&r, &v, 4);
    return r;
}

// ---- phase 0: activation blocks of x, router products ----------------------

template <bool LO>
__device__ __forceinline__ void layout_x(const MoeParams& p, int warp, int warps, int lane) {
    bool finite = true;
    for (int task = warp; task < p.t * p.kb_h; task += warps) {
        const int tok = task / p.kb_h, kb = task - tok * p.kb_h;
        float v[4], amax = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = kb * kF8Block + lane * 4 + i;
            v[i] = k < p.h ? load_dense(p.x, p.type, tok * p.ldx + k) : 0.0f;
            finite &= isfinite(v[i]);
            amax = fmaxf(amax, fabsf(v[i]));
        }
        float inv;
        const float s = act_scale(warp_max(amax), inv);
        uint8_t* blk = p.xq + static_cast<long long>(task) * ActBlock<LO>::kBytes;
        float hi[4], lo[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            hi[i] = __half2float(__float2half_rn(v[i] * inv));
            lo[i] = v[i] * inv - hi[i];
        }
        *reinterpret_cast<uint2*>(blk + act_at(lane * 4)) = make_uint2(pack_half2(hi[0], hi[1]), pack_half2(hi[2], hi[3]));
        if constexpr (LO)
            *reinterpret_cast<uint2*>(blk + 256 + act_at(lane * 4)) =
                make_uint2(pack_half2(lo[0], lo[1]), pack_half2(lo[2], lo[3]));
        if (lane == 0) *reinterpret_cast<float*>(blk + ActBlock<LO>::kScaleAt) = s;
    }
    if (!finite) atomicExch(p.err, kErrNonFinite);
}

// Partial sums over k0..k1 of one expert's row with kRouterTokens tokens.
__device__ __forceinline__ void router_dot(const MoeParams& p, int ex, int tok0, int k0, int k1, int lane,
                                           float (&s)[kRouterTokens]) {
#pragma unroll
    for (int i = 0; i < kRouterTokens; ++i) s[i] = 0.0f;
#pragma unroll 4
    for (int k = k0 + lane; k < k1; k += 32) {
        const float r = load_dense(p.router, p.router_type, ex * p.ld_router + k);
#pragma unroll
        for (int i = 0; i < kRouterTokens; ++i)
            if (tok0 + i < p.t) s[i] = fmaf(r, load_dense(p.x, p.type, (tok0 + i) * p.ldx + k), s[i]);
    }
#pragma unroll
    for (int i = 0; i < kRouterTokens; ++i)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s[i] += __shfl_xor_sync(0xffffffffu, s[i], o);
}

// Few tasks: a CTA's consumer warps share a task's k range; many: a warp each.
__device__ __forceinline__ void router_products(const MoeParams& p, const Tables& tb, int warp, int lane) {
    const int groups = (p.t + kRouterTokens - 1) / kRouterTokens, tasks = p.e * groups;
    float s[kRouterTokens];
    if (tasks <= 2 * static_cast<int>(gridDim.x)) {
        const int per = (p.h + kConsumers - 1) / kConsumers;
        for (int task = blockIdx.x; task < tasks; task += gridDim.x) {
            const int ex = task / groups, tok0 = (task - ex * groups) * kRouterTokens;
            if (warp < kConsumers) {
                router_dot(p, ex, tok0, warp * per, min(p.h, (warp + 1) * per), lane, s);
                if (lane == 0)
#pragma unroll
                    for (int i = 0; i < kRouterTokens; ++i) tb.red[warp * kRouterTokens + i] = s[i];
            }
            __syncthreads();
            if (threadIdx.x < kRouterTokens && tok0 + static_cast<int>(threadIdx.x) < p.t) {
                float sum = 0.0f;
                for (int w = 0; w < kConsumers; ++w) sum += tb.red[w * kRouterTokens + threadIdx.x];
                __stcg(p.logits + (tok0 + threadIdx.x) * p.e + ex, sum);
            }
            __syncthreads();
        }
    } else {
        const int warps = gridDim.x * (kThreads / 32);
        for (int task = blockIdx.x * (kThreads / 32) + warp; task < tasks; task += warps) {
            const int ex = task / groups, tok0 = (task - ex * groups) * kRouterTokens;
            router_dot(p, ex, tok0, 0, p.h, lane, s);
            if (lane == 0)
#pragma unroll
                for (int i = 0; i < kRouterTokens; ++i)
                    if (tok0 + i < p.t) __stcg(p.logits + (tok0 + i) * p.e + ex, s[i]);
        }
    }
}

// ---- routing ---------------------------------------------------------------

// Order-preserving integer of a logit, above 0; NaN sorts last.
__device__ __forceinline__ uint32_t sort_key(float v) {
    const uint32_t b = __float_as_uint(v);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 1u;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// One token: its `top` largest logits, ties to the lower expert.
__device__ __forceinline__ void choose(const MoeParams& p, const Tables& tb, int tok, int lane) {
    constexpr int kPer = kMoeMaxExperts / 32;
    float v[kPer];
    uint32_t key[kPer];
    float vmax = -INFINITY;
    bool finite = true;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int ex = lane + 32 * j;
        v[j] = ex < p.e ? __ldcg(p.logits + tok * p.e + ex) : -INFINITY;
        finite &= ex >= p.e || isfinite(v[j]);
        key[j] = ex < p.e ? sort_key(v[j]) : 0u;
        vmax = fmaxf(vmax, v[j]);
    }
    if (!finite) atomicExch(p.err, kErrNonFinite);
    vmax = warp_max(vmax);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kPer; ++j) sum += lane + 32 * j < p.e ? expf(v[j] - vmax) : 0.0f;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    float chosen = 0.0f, mine = 0.0f;  // lane k keeps slot k
    int mine_e = 0;
    for (int k = 0; k < p.top; ++k) {
        uint32_t best = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) best = max(best, key[j]);
        best = __reduce_max_sync(0xffffffffu, best);
        uint32_t at = 0xffffffffu;
#pragma unroll
        for (int j = kPer - 1; j >= 0; --j)
            if (key[j] == best) at = lane + 32 * j;
        at = __reduce_min_sync(0xffffffffu, at);
        float ev = 0.0f;
#pragma unroll
        for (int j = 0; j < kPer; ++j)
            if (static_cast<uint32_t>(lane + 32 * j) == at) {
                ev = expf(v[j] - vmax);
                key[j] = 0u;
            }
        ev = __shfl_sync(0xffffffffu, ev, at & 31);
        chosen += ev;
        if (lane == k) {
            mine = ev;
            mine_e = static_cast<int>(at);
        }
    }
    if (lane < p.top) {
        const float w = mine / (p.renorm ? chosen : sum);
        const int pair = tok * p.top + lane;
        tb.pair_w[pair] = w;
        tb.pair_e[pair] = static_cast<short>(mine_e);
        if (blockIdx.x == 0) {
            p.ids[pair] = mine_e;
            p.weights[pair] = w;
        }
    }
}

// Pairs sorted by expert (then token); experts with pairs become entries of
// at most `cap` pairs each.
__device__ __forceinline__ void build_tables(const MoeParams& p, const Tables& tb, int cap) {
    const int pairs = p.t * p.top;
    for (int ex = threadIdx.x; ex < p.e; ex += kThreads) {
        int n = 0;
        for (int i = 0; i < pairs; ++i) n += tb.pair_e[i] == ex;
        tb.count[ex] = n;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int pos = 0, ents = 0;
        for (int e0 = 0; e0 < p.e; e0 += 32) {
            const int ex = e0 + lane, n = ex < p.e ? tb.count[ex] : 0, ne = (n + cap - 1) / cap;
            int sp = n, se = ne;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int a = __shfl_up_sync(0xffffffffu, sp, o), b = __shfl_up_sync(0xffffffffu, se, o);
                if (lane >= o) sp += a, se += b;
            }
            for (int i = 0; i < ne; ++i) tb.entry[ents + se - ne + i] = (ex << 16) | (pos + sp - n + i * cap);
            if (ex < p.e) tb.count[ex] = pos + sp - n;  // now the expert's first position
            pos += __shfl_sync(0xffffffffu, sp, 31);
            ents += __shfl_sync(0xffffffffu, se, 31);
        }
        if (lane == 0) tb.info[0] = ents, tb.info[1] = pos;
    }
    __syncthreads();
    for (int ex = threadIdx.x; ex < p.e; ex += kThreads) {
        int at = tb.count[ex];
        for (int i = 0; i < pairs; ++i)
            if (tb.pair_e[i] == ex) tb.order[at++] = static_cast<short>(i);
    }
    __syncthreads();
}

// First position and number of pairs of entry i.
__device__ __forceinline__ void entry_pairs(const Tables& tb, int i, int cap, int& first, int& n) {
    const int w = tb.entry[i];
    first = w & 0xFFFF;
    int end = tb.info[1];
    if (i + 1 < tb.info[0]) end = tb.entry[i + 1] & 0xFFFF;
    n = min(cap, end - first);
}

// ---- the line of blocks ----------------------------------------------------

struct Line {
    int tiles, nkb, total;  // tiles per entry, blocks per tile, blocks in all
    int parts;              // CTAs that share it: all, or one per block
    __device__ __forceinline__ Line(int entries, int tiles_, int nkb_)
        : tiles(tiles_), nkb(nkb_), total(entries * tiles_ * nkb_), parts(min(static_cast<int>(gridDim.x), total)) {}
    // First block of CTA cta's part; the CTA whose part holds block x.
    __device__ __forceinline__ int start(int cta) const {
        return static_cast<int>(static_cast<long long>(cta) * total / parts);
    }
    __device__ __forceinline__ int owner(int x) const {
        return static_cast<int>(((static_cast<long long>(x) + 1) * parts - 1) / total);
    }
};

struct Seg {
    int entry, tile, kb0, kb1, x0;  // x0: the tile's first block in the line
};

struct Walk {
    int cur, end;
    __device__ __forceinline__ explicit Walk(const Line& l) : cur(0), end(0) {
        if (static_cast<int>(blockIdx.x) < l.parts) {
            cur = l.start(blockIdx.x);
            end = l.start(blockIdx.x + 1);
        }
    }
    __device__ __forceinline__ bool next(const Line& l, Seg& s) {
        if (cur >= end) return false;
        const int ft = cur / l.nkb;
        s.x0 = ft * l.nkb;
        s.kb0 = cur - s.x0;
        s.kb1 = min(l.nkb, s.kb0 + (end - cur));
        s.entry = ft / l.tiles;
        s.tile = ft - s.entry * l.tiles;
        cur += s.kb1 - s.kb0;
        return true;
    }
};

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
        "[%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// Untiled copy: both addresses and the size are multiples of 16 bytes.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                     smem_u32(dst)),
                 "l"(src), "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two e4m3 bytes -> two f16, exactly.
__device__ __forceinline__ uint32_t e4m3_to_half2(uint32_t two) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(static_cast<uint16_t>(two)));
    return r;
}

// ---- the kernel ------------------------------------------------------------

template <int NG, bool LO>
struct Consumer {
    using C = MoeCfg<NG, LO>;
    using Act = ActBlock<LO>;
    // gate / up (or the two halves of 256 down rows) x token groups x fragment
    float acc[2][NG][4];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int n = 0; n < NG; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[b][n][i] = 0.0f;
    }

    // One block of 128: this warp's 16 rows of both boxes times ng token groups.
    __device__ __forceinline__ void block(const uint8_t* stage, int warp, int lane, int ng, float s0, float s1) {
        const int g = lane >> 2, t = lane & 3;
        uint32_t a[2][8][4];  // box, k step, fragment
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const uint8_t* row = stage + b * kBoxBytes + (warp * 16 + g) * kF8Block;
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int at = ((2 * t + c) ^ g) * 16;
                const uint4 lo = *reinterpret_cast<const uint4*>(row + at);
                const uint4 hi = *reinterpret_cast<const uint4*>(row + 8 * kF8Block + at);
                const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[b][4 * c + i][0] = e4m3_to_half2(wl[i] & 0xFFFFu);
                    a[b][4 * c + i][1] = e4m3_to_half2(wh[i] & 0xFFFFu);
                    a[b][4 * c + i][2] = e4m3_to_half2(wl[i] >> 16);
                    a[b][4 * c + i][3] = e4m3_to_half2(wh[i] >> 16);
                }
            }
        }
        const uint8_t* act = stage + 2 * kBoxBytes;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            if (n >= ng) break;
            const uint8_t* row = act + (n * 8 + g) * Act::kPitch + t * 16;
            float d[2][4] = {};
#pragma unroll
            for (int part = 0; part < (LO ? 2 : 1); ++part)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint4 v = *reinterpret_cast<const uint4*>(row + part * 256 + j * 64);
                    mma_f16(d[0], a[0][2 * j], v.x, v.y);
                    mma_f16(d[1], a[1][2 * j], v.x, v.y);
                    mma_f16(d[0], a[0][2 * j + 1], v.z, v.w);
                    mma_f16(d[1], a[1][2 * j + 1], v.z, v.w);
                }
            // columns 2t and 2t + 1
            const uint8_t* sc = act + (n * 8 + 2 * t) * Act::kPitch + Act::kScaleAt;
            const float x0 = *reinterpret_cast<const float*>(sc), x1 = *reinterpret_cast<const float*>(sc + Act::kPitch);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float xs = (i & 1) ? x1 : x0;
                acc[0][n][i] = fmaf(d[0][i], s0 * xs, acc[0][n][i]);
                acc[1][n][i] = fmaf(d[1][i], s1 * xs, acc[1][n][i]);
            }
        }
    }

    __device__ __forceinline__ void put_part(float* to, int ng) const {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int n = 0; n < NG; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n < ng) __stcg(to + ((n * 2 + b) * 4 + i) * kConsThreads, acc[b][n][i]);
    }

    __device__ __forceinline__ void add_part(const float* from, int ng) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int n = 0; n < NG; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (n < ng) acc[b][n][i] += __ldcg(from + ((n * 2 + b) * 4 + i) * kConsThreads);
    }
};

template <int NG, bool LO>
__global__ void __launch_bounds__(kThreads, 1) moe_f8_kernel(const __grid_constant__ MoeParams p) {
    using C = MoeCfg<NG, LO>;
    using Act = ActBlock<LO>;
    constexpr int S = C::kStages, kCap = NG * 8;
    constexpr int kPart = 8 * NG * kConsThreads;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOffset);
    uint64_t* empty = full + S;
    volatile uint32_t* abort = reinterpret_cast<uint32_t*>(empty + S);
    uint32_t* last_flag = reinterpret_cast<uint32_t*>(empty + S) + 1;
    Tables tb;
    tb.pair_w = reinterpret_cast<float*>(smem + C::kTables);
    tb.entry = reinterpret_cast<int*>(tb.pair_w + kMaxPairs);
    tb.count = tb.entry + kMaxPairs;
    tb.info = tb.count + kMoeMaxExperts;
    tb.red = reinterpret_cast<float*>(tb.info + 4);
    tb.pair_e = reinterpret_cast<short*>(tb.red + kConsumers * kMoeMaxTokens);
    tb.order = tb.pair_e + kMaxPairs;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const unsigned grid = gridDim.x;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], 2);  // weights, activations
            mbar_init(&empty[s], kConsumers);
        }
        *abort = 0u;
        fence_mbar_init();
        prefetch_tmap(&p.tm_gate);
        prefetch_tmap(&p.tm_up);
        prefetch_tmap(&p.tm_down);
    }

    // ---- phase 0 ----
    layout_x<LO>(p, blockIdx.x * (kThreads / 32) + warp, grid * (kThreads / 32), lane);
    if (p.router) router_products(p, tb, warp, lane);
    asm volatile("fence.proxy.async.global;" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) {
        grid_arrive(p.ctrl + kBarrier);
        if (!grid_wait(p.ctrl + kBarrier, grid, abort)) fail(p.err, abort, kErrTimeoutGrid);
    }
    if (!__syncthreads_or(threadIdx.x == 0 && *abort != 0u)) {
        // ---- routing, by every CTA for itself ----
        if (p.router) {
            for (int tok = warp; tok < p.t; tok += kThreads / 32) choose(p, tb, tok, lane);
        } else {
            for (int i = threadIdx.x; i < p.t * p.top; i += kThreads) {
                int ex = p.ids[i];
                if (ex >= p.e) {
                    if (blockIdx.x == 0) atomicCAS(p.err, 0, kErrBadIndex);
                    ex = -1;
                }
                tb.pair_e[i] = static_cast<short>(ex < 0 ? -1 : ex);
                tb.pair_w[i] = p.weights[i];
            }
        }
        __syncthreads();
        build_tables(p, tb, kCap);
        const int entries = tb.info[0];
        const Line line1(entries, p.tiles_f, p.kb_h), line2(entries, p.tiles_h, p.kb_f);

        if (entries == 0) {
            // no slot names an expert: the sums are empty
            for (long long i = blockIdx.x * kThreads + threadIdx.x; i < static_cast<long long>(p.t) * p.h;
                 i += grid * kThreads)
                store_dense(p.out, p.type, i / p.h * p.ldo + i % p.h, 0.0f);
        } else if (warp == kConsumers) {
            // ---- producer warp ----
            asm volatile("fence.proxy.async.global;" ::: "memory");
            int gw = 0, ga = 0;  // stages whose weights / activations were issued
            bool ok = true;
            auto issue_w = [&](int phase, const Seg& s, int kb) {
                const int st = gw % S;
                if (lane == 0) {
                    if (gw >= S && !wait_or_abort(&empty[st], ((gw / S) & 1) ^ 1, abort)) {
                        if (!*abort) fail(p.err, abort, kErrTimeoutEmpty);
                        ok = false;
                    } else {
                        uint8_t* dst = smem + st * C::kStage;
                        const int ex = tb.entry[s.entry] >> 16;
                        mbar_arrive_expect_tx(&full[st], 2 * kBoxBytes);
                        if (phase == 1) {
                            tma_load_3d(dst, &p.tm_gate, &full[st], kb * kF8Block, s.tile * kBoxRows, ex);
                            tma_load_3d(dst + kBoxBytes, &p.tm_up, &full[st], kb * kF8Block, s.tile * kBoxRows, ex);
                        } else {
                            tma_load_3d(dst, &p.tm_down, &full[st], kb * kF8Block, s.tile * 2 * kBoxRows, ex);
                            tma_load_3d(dst + kBoxBytes, &p.tm_down, &full[st], kb * kF8Block,
                                        s.tile * 2 * kBoxRows + kBoxRows, ex);
                        }
                    }
                }
                ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                if (ok) ++gw;
            };
            auto issue_a = [&](int phase, const Seg& s, int kb) {
                const int st = ga % S;
                int first, n;
                entry_pairs(tb, s.entry, kCap, first, n);
                uint8_t* dst = smem + st * C::kStage + 2 * kBoxBytes;
                if (lane == 0) mbar_arrive_expect_tx(&full[st], n * Act::kBytes);
                __syncwarp();
                for (int i = lane; i < n; i += 32) {
                    const uint8_t* src =
                        phase == 1
                            ? p.xq + (static_cast<long long>(tb.order[first + i] / p.top) * p.kb_h + kb) * Act::kBytes
                            : p.hq + (static_cast<long long>(first + i) * p.kb_f + kb) * Act::kBytes;
                    bulk_load(dst + i * Act::kPitch, src, Act::kBytes, &full[st]);
                }
                ++ga;
            };
            Seg s;
            {
                Walk walk(line1);
                while (ok && walk.next(line1, s))
                    for (int kb = s.kb0; ok && kb < s.kb1; ++kb) {
                        issue_w(1, s, kb);
                        if (ok) issue_a(1, s, kb);
                    }
            }
            // phase 2: up to S stages of weights ahead of the barrier
            {
                Walk walk(line2), walk_a(line2);
                Seg sa;
                bool more = walk.next(line2, s), more_a = walk_a.next(line2, sa);
                int kb = more ? s.kb0 : 0, kba = more_a ? sa.kb0 : 0;
                auto step_w = [&] {
                    issue_w(2, s, kb);
                    if (ok && ++kb == s.kb1) {
                        more = walk.next(line2, s);
                        kb = s.kb0;
                    }
                };
                for (int i = 0; ok && more && i < S; ++i) step_w();
                if (ok && more_a) {
                    if (lane == 0 && !grid_wait(p.ctrl + kBarrier, 2 * grid, abort)) {
                        if (!*abort) fail(p.err, abort, kErrTimeoutGrid);
                        ok = false;
                    }
                    ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                    asm volatile("fence.proxy.async.global;" ::: "memory");
                }
                while (ok && more_a) {
                    if (ga == gw) step_w();  // past the weights issued ahead
                    if (!ok) break;
                    issue_a(2, sa, kba);
                    if (++kba == sa.kb1) {
                        more_a = walk_a.next(line2, sa);
                        kba = sa.kb0;
                    }
                }
            }
            // copies in flight must land before the CTA exits
            if (lane == 0)
                for (int i = max(0, gw - S); i < gw; ++i)
                    if (!mbar_wait(&full[i % S], (i / S) & 1)) {
                        atomicCAS(p.err, 0, kErrTimeoutDrain);
                        break;
                    }
            __syncwarp();
        } else {
            // ---- consumer warps ----
            const int g = lane >> 2, t = lane & 3;
            Consumer<NG, LO> c;
            int stage = 0;
            bool ok = true;
            for (int phase = 1; ok && phase <= 2; ++phase) {
                const Line& line = phase == 1 ? line1 : line2;
                Walk walk(line);
                Seg s;
                while (ok && walk.next(line, s)) {
                    int first, n;
                    entry_pairs(tb, s.entry, kCap, first, n);
                    const int ng = (n + 7) / 8, ex = tb.entry[s.entry] >> 16;
                    const float *s0, *s1;
                    if (phase == 1) {
                        s0 = p.gate_s + ex * p.gate_ss + static_cast<long long>(s.tile) * p.kb_h;
                        s1 = p.up_s + ex * p.up_ss + static_cast<long long>(s.tile) * p.kb_h;
                    } else {
                        // the last tile's second half may not exist: any scale, its rows are zero
                        const int rb = 2 * s.tile, last = (p.h + kF8Block - 1) / kF8Block - 1;
                        s0 = p.down_s + ex * p.down_ss + static_cast<long long>(rb) * p.kb_f;
                        s1 = p.down_s + ex * p.down_ss + static_cast<long long>(min(rb + 1, last)) * p.kb_f;
                    }
                    c.clear();
                    float w0 = __ldg(s0 + s.kb0), w1 = __ldg(s1 + s.kb0);
                    for (int kb = s.kb0; kb < s.kb1; ++kb, ++stage) {
                        const int st = stage % S;
                        const int nk = min(kb + 1, s.kb1 - 1);
                        const float n0 = __ldg(s0 + nk), n1 = __ldg(s1 + nk);
                        int ready = 0;
                        if (lane == 0) ready = wait_or_abort(&full[st], (stage / S) & 1, abort) ? 1 : 0;
                        ready = __shfl_sync(0xffffffffu, ready, 0);
                        if (!ready) {
                            if (lane == 0 && !*abort) fail(p.err, abort, kErrTimeoutFull);
                            ok = false;
                            break;
                        }
                        c.block(smem + st * C::kStage, warp, lane, ng, w0, w1);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&empty[st]);
                        w0 = n0;
                        w1 = n1;
                    }
                    // one decision for all consumer warps
                    if (cons_any(!ok)) {
                        ok = false;
                        break;
                    }
                    if (s.kb1 - s.kb0 != line.nkb) {
                        // a cut tile
                        float* mine = p.part + (2ll * blockIdx.x + (s.kb0 == 0 ? 1 : 0)) * kPart + threadIdx.x;
                        c.put_part(mine, ng);
                        const int a = line.owner(s.x0), b = line.owner(s.x0 + line.nkb - 1);
                        __threadfence();
                        cons_bar();
                        if (threadIdx.x == 0) {
                            // a tile that is cut is the last of its first CTA
                            unsigned* cut = p.ctrl + (phase == 1 ? kCut1 : kCut2) + a;
                            *last_flag = atomicAdd(cut, 1u) == static_cast<unsigned>(b - a) ? 1u : 0u;
                            if (*last_flag) *cut = 0u;
                        }
                        cons_bar();
                        if (!*last_flag) continue;
                        __threadfence();
                        c.clear();
                        for (int cta = a; cta <= b; ++cta)
                            c.add_part(p.part + (2ll * cta + (cta == a ? 1 : 0)) * kPart + threadIdx.x, ng);
                    }
                    if (phase == 1) {
                        // hidden values of 128 rows; rows behind f are zero (zero weights)
                        float hv[NG][4], am[NG][2];
#pragma unroll
                        for (int i = 0; i < NG; ++i) {
                            if (i >= ng) break;
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float gate = c.acc[0][i][j];
                                hv[i][j] = gate / (1.0f + expf(-gate)) * c.acc[1][i][j];
                            }
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                float m = fmaxf(fabsf(hv[i][j]), fabsf(hv[i][j + 2]));
#pragma unroll
                                for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                                am[i][j] = m;
                                if (g == 0) tb.red[warp * kMoeMaxTokens + i * 8 + 2 * t + j] = m;
                            }
                        }
                        cons_bar();
#pragma unroll
                        for (int i = 0; i < NG; ++i) {
                            if (i >= ng) break;
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const int col = i * 8 + 2 * t + j;
                                float m = 0.0f, inv;
                                for (int w = 0; w < kConsumers; ++w) m = fmaxf(m, tb.red[w * kMoeMaxTokens + col]);
                                const float sc = act_scale(m, inv);
                                if (col < n) {
                                    uint8_t* blk = p.hq + (static_cast<long long>(first + col) * p.kb_f + s.tile) * Act::kBytes;
#pragma unroll
                                    for (int r = 0; r < 2; ++r) {
                                        const float v = hv[i][j + 2 * r] * inv;
                                        const __half hi = __float2half_rn(v);
                                        const int at = act_at(warp * 16 + g + 8 * r);
                                        *reinterpret_cast<__half*>(blk + at) = hi;
                                        if constexpr (LO)
                                            *reinterpret_cast<__half*>(blk + 256 + at) = __float2half_rn(v - __half2float(hi));
                                    }
                                    if (warp == 0 && g == 0) *reinterpret_cast<float*>(blk + Act::kScaleAt) = sc;
                                }
                            }
                        }
                        cons_bar();  // red is free again
                    } else {
                        // this expert's rows of its slots, then the last expert of the column tile sums them
                        const int row0 = s.tile * 2 * kBoxRows + warp * 16 + g;
#pragma unroll
                        for (int i = 0; i < NG; ++i) {
                            if (i >= ng) break;
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const int col = i * 8 + 2 * t + j;
                                if (col < n) {
                                    float* o = p.pair_out + static_cast<long long>(tb.order[first + col]) * p.h;
#pragma unroll
                                    for (int b = 0; b < 2; ++b)
#pragma unroll
                                        for (int r = 0; r < 2; ++r) {
                                            const int row = row0 + b * kBoxRows + 8 * r;
                                            if (row < p.h) __stcg(o + row, c.acc[b][i][j + 2 * r]);
                                        }
                                }
                            }
                        }
                        __threadfence();
                        cons_bar();
                        if (threadIdx.x == 0) {
                            unsigned* cnt = p.ctrl + kCombine + s.tile;
                            *last_flag = atomicAdd(cnt, 1u) == static_cast<unsigned>(entries - 1) ? 1u : 0u;
                            if (*last_flag) *cnt = 0u;
                        }
                        cons_bar();
                        if (*last_flag) {
                            __threadfence();
                            const int row = s.tile * 2 * kBoxRows + threadIdx.x;
                            if (row < p.h) {
#pragma unroll 4
                                for (int tok = 0; tok < p.t; ++tok) {
                                    float y = 0.0f;
                                    for (int k = 0; k < p.top; ++k) {
                                        const int pair = tok * p.top + k;
                                        if (tb.pair_e[pair] >= 0)
                                            y = fmaf(tb.pair_w[pair],
                                                     __ldcg(p.pair_out + static_cast<long long>(pair) * p.h + row), y);
                                    }
                                    store_dense(p.out, p.type, tok * p.ldo + row, y);
                                }
                            }
                        }
                        cons_bar();  // last_flag is free again
                    }
                }
                if (phase == 1 && ok) {
                    asm volatile("fence.proxy.async.global;" ::: "memory");
                    cons_bar();
                    if (threadIdx.x == 0) grid_arrive(p.ctrl + kBarrier);
                }
            }
        }
    }
    __syncthreads();
    // the last CTA out returns the barrier words to zero
    if (threadIdx.x == 0) {
        __threadfence();
        if (atomicAdd(p.ctrl + kExit, 1u) == grid - 1) {
            p.ctrl[kBarrier] = 0u;
            p.ctrl[kExit] = 0u;
        }
    }
}

// (k, rows, experts) map of an expert stack: box 128 bytes x 128 rows x 1.
bool make_expert_map(CUtensorMap* map, const MoeWeight& w, int k, int rows, int experts) {
    static PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
        cudaDriverEntryPointQueryResult q;
        void* fn = nullptr;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    }();
    if (!encode) return false;
    cuuint64_t dims[3] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(experts)};
    cuuint64_t strides[2] = {static_cast<cuuint64_t>(w.ld), static_cast<cuuint64_t>(w.stride)};
    cuuint32_t box[3] = {kF8Block, kBoxRows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(w.w), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int token_groups(int t) { return t <= 8 ? 1 : t <= 16 ? 2 : t <= 32 ? 4 : 8; }

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// Scratch areas in order, after the zeroed header.
struct MoeScratch {
    size_t logits, xq, hq, part, pair_out, total;
    MoeScratch(int t, int h, int f, int e, int top, int type) {
        const size_t blk = type == kTypeF32 ? ActBlock<true>::kBytes : ActBlock<false>::kBytes;
        const size_t kb_h = (h + 127) / 128, kb_f = (f + 127) / 128, pairs = static_cast<size_t>(t) * top;
        logits = 0;
        xq = logits + up256(static_cast<size_t>(t) * e * 4);
        hq = xq + up256(t * kb_h * blk);
        part = hq + up256(pairs * kb_f * blk);
        pair_out = part + up256(static_cast<size_t>(sm_count()) * 2 * 8 * token_groups(t) * kConsThreads * 4);
        total = pair_out + pairs * h * 4;
    }
};

template <int NG, bool LO>
int launch_cfg(const MoeParams& p, cudaStream_t s) {
    using C = MoeCfg<NG, LO>;
    auto kern = moe_f8_kernel<NG, LO>;
    static bool attr_done[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !attr_done[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kBytes);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) attr_done[dev] = true;
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(sm_count()), 1, 1);
    cfg.blockDim = dim3(kThreads, 1, 1);
    cfg.dynamicSmemBytes = C::kBytes;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

}  // namespace

size_t moe_f8_scratch_bytes(int t, int h, int f, int e, int top, int type) {
    return MoeScratch(t, h, f, e, top, type).total;
}

int launch_moe_f8(const MoeF8& m, int* err, cudaStream_t s) {
    MoeParams p{};
    const MoeScratch sc(m.t, m.h, m.f, m.e, m.top, m.type);
    if (m.scratch_bytes < sc.total) return cudaErrorInvalidValue;
    if (!make_expert_map(&p.tm_gate, m.gate, m.h, m.f, m.e) || !make_expert_map(&p.tm_up, m.up, m.h, m.f, m.e) ||
        !make_expert_map(&p.tm_down, m.down, m.f, m.h, m.e))
        return cudaErrorInvalidValue;
    p.gate_s = m.gate.scales;
    p.up_s = m.up.scales;
    p.down_s = m.down.scales;
    p.gate_ss = m.gate.scale_stride;
    p.up_ss = m.up.scale_stride;
    p.down_ss = m.down.scale_stride;
    p.x = m.x;
    p.out = m.out;
    p.router = m.router;
    p.ldx = m.ldx;
    p.ldo = m.ldo;
    p.ld_router = m.ld_router;
    p.type = m.type;
    p.router_type = m.router_type;
    p.ids = m.ids;
    p.weights = m.weights;
    p.t = m.t;
    p.h = m.h;
    p.f = m.f;
    p.e = m.e;
    p.top = m.top;
    p.renorm = m.renorm;
    p.kb_h = (m.h + kF8Block - 1) / kF8Block;
    p.kb_f = (m.f + kF8Block - 1) / kF8Block;
    p.tiles_f = p.kb_f;
    p.tiles_h = (m.h + 2 * kBoxRows - 1) / (2 * kBoxRows);
    // the line's length is an int and the header has a counter per column tile
    const long long longest = std::max(static_cast<long long>(p.tiles_f) * p.kb_h, static_cast<long long>(p.tiles_h) * p.kb_f);
    if (longest * std::min(m.t * m.top, kMaxPairs) > 0x7fffffffll ||
        p.tiles_h > static_cast<int>(kF8Counters) - kCombine || sm_count() > kCut2 - kCut1)
        return cudaErrorInvalidValue;
    uint8_t* base = static_cast<uint8_t*>(m.scratch);
    p.ctrl = m.counters;
    p.logits = reinterpret_cast<float*>(base + sc.logits);
    p.xq = base + sc.xq;
    p.hq = base + sc.hq;
    p.part = reinterpret_cast<float*>(base + sc.part);
    p.pair_out = reinterpret_cast<float*>(base + sc.pair_out);
    p.err = err;
    const bool lo = m.type == kTypeF32;
    switch (token_groups(m.t)) {
        case 1: return lo ? launch_cfg<1, true>(p, s) : launch_cfg<1, false>(p, s);
        case 2: return lo ? launch_cfg<2, true>(p, s) : launch_cfg<2, false>(p, s);
        case 4: return lo ? launch_cfg<4, true>(p, s) : launch_cfg<4, false>(p, s);
        default: return lo ? launch_cfg<8, true>(p, s) : launch_cfg<8, false>(p, s);
    }
}

}  // namespace rk
