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
// Activations are not quantised: a block of them is scaled by a power of two
// so that its largest magnitude is in [2^14, 2^15) and held in f16.  A second
// f16 holds the remainder, 22 bits in all, of f32 inputs and of the hidden
// values of every type: rounded to 11 bits they alone moved a f16 result by
// as much as its own rounding.  f16 / bf16 inputs fit one f16 (but for what is
// below 2^-39 of their block's largest).  Sums are f32: 128 products per
// block in the MMA's accumulator, times the weight scale and the activation's
// power of two, added to f32 totals.
//
// k order.  The sum over k may run in any order, so thread (g, t) of a warp
// takes 32 consecutive bytes 32 t .. of weight row g (two 16-byte reads that
// the swizzle spreads over all banks) and the activations are laid out in
// memory in the order in which the threads then need them.
//
// Work.  A group is 16 gate and 16 up rows (32 down rows) of one chosen
// expert over the whole of k; the groups of all chosen experts form one line
// that is cut evenly into as many parts as there are SMs, at most one group
// apart.  Groups and not larger tiles, because then nothing of gate / up is
// summed across CTAs (cutting 128-row tiles along k evenly instead left each
// CTA one or two partial tiles to exchange: 6 us between the two products of
// a 10 us layer).  A part runs in passes of up to 8 groups, one per warp;
// with fewer, warps share a group's blocks and add through shared memory.
// Hidden values are scaled per group of 16; the down product brings the
// eight groups of a block to the block's largest scale as it reads them.  A
// group whose scale is less than 2^-14 of that would lose its last bits in
// f16, or all of them; the block's products are then run again for such
// groups alone, brought to the largest scale among them.
//
// The down product may also cut k (a part's groups then divide more evenly);
// its sums go to memory per slot and cut, and are added in a fixed order at
// the end, so results do not depend on who finishes when.
//
// Phases: (0) router products and the activations' layout; (1) every CTA
// picks the experts for itself, gate / up products, SiLU; (2) down products;
// (3) weighted sums of the slots.  A CTA takes a part by ticket and does that part of every
// phase.  One that waits long for the others in phase 0 takes further parts,
// until all are held by CTAs that run, so the launch needs no co-residency (a
// cooperative launch cost 16 us more per call).  The weight copies of phase 2
// start before its wait.  Every wait is bounded.
//
// Measured: one token, 2 of 8 experts, 2048 / 5632, f32: 37.5 us, 69 MB of
// weights (10.6 us at HBM's rate; half is the latency of the phases); 13
// tokens, 4 of 16, 1536 / 2240, f16: 56.5 us, 2.9 TB/s; 64 tokens, 2 of 8, 4096 /
// 8192, bf16: 329 us, 2.5 TB/s, bound by the consumers, two warps per scheduler
// (the hidden values' second term about 20 us, the look for far groups 10).
#include <cuda.h>
#include <cudaTypedefs.h>

#include <algorithm>

#include "f8.cuh"
#include "kernels.h"
#include "ptx.cuh"
#include "quant_math.cuh"

namespace rk {
namespace {

constexpr int kProducers = 4;    // warps that issue copies
constexpr int kPassGroups = 8;   // groups of a pass, at most
constexpr int kRouterWarps = 8;  // warps that share a router task
constexpr int kBoxRows = 16;                 // rows of one TMA box, one MMA tile
constexpr int kBoxBytes = kBoxRows * kF8Block;
constexpr int kGroupBytes = 2 * kBoxBytes;   // gate and up, or two boxes of down rows
constexpr int kMaxPairs = kMoeMaxTokens * kMoeMaxTop;
constexpr int kRouterTokens = 4;             // tokens per router task
constexpr int kMaxParts = 256;               // CTAs of a launch
constexpr int kMaxEntries = kMoeMaxExperts + kMaxPairs / 8;  // an expert's last entry may be short, the others hold 8 or more
constexpr float kNear = 1.0f / 16384.0f;     // hidden groups of a pass: from the largest scale down to this part of it
constexpr uint64_t kHelpNs = 20000;          // wait for the others before taking a further part

// Words of the zeroed header.
constexpr int kTicket = 0, kExit = 32, kDone = 64;  // kDone + 32 i: parts of phase i done

struct MoeParams {
    CUtensorMap tm_gate, tm_up, tm_down;  // (k, rows, expert), boxes of 128 B x 16, 16 and 32 rows
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
    int kb_h, kb_f, max_split;
    int wide;  // x and router rows can be read 16 bytes at a time
    unsigned* ctrl;
    float* logits;    // [t][e]
    uint8_t* xq;      // [kb_h][t] activation blocks
    uint8_t* hq;      // [kb_f][pair] activation blocks, pairs in sorted order
    float* pair_out;  // [pair][max_split][h]
    int* err;
};

// An activation block of 128 values: f16 values (and remainders) in the
// order of the MMA operands, then eight f32 powers of two, one per 16 values
// (x: all the first one's).  Its size is an odd multiple of 64 bytes, so that
// two rows' 64-byte reads fall into different banks of shared memory.
template <bool LO>
struct ActBlock {
    static constexpr int kScaleAt = LO ? 512 : 256;
    static constexpr int kBytes = LO ? 576 : 320;
};

template <int NG, bool LO>
struct MoeCfg {
    using Act = ActBlock<LO>;    // of x
    using Hid = ActBlock<true>;  // of hidden values
    static constexpr int kConsumers = 8;  // a group of a pass each; 16 with fewer registers were slower
    static constexpr int kConsThreads = kConsumers * 32;
    static constexpr int kWarps = kConsumers + kProducers;
    static constexpr int kThreads = kWarps * 32;
    // registers after the split: 256 x 224 + 128 x 56 of 384 x 168
    static constexpr int kConsRegs = 224, kProdRegs = 56;
    static constexpr int kAct = (NG * 8 * Hid::kBytes + 1023) / 1024 * 1024;  // the larger of the two
    static constexpr int kStage = kPassGroups * kGroupBytes + kAct;
    static constexpr int kRedBytes = kConsThreads * 8 * 4;  // sums that warps exchange
    static constexpr int kTableBytes =
        kRedBytes + kMaxPairs * (4 + 2 + 2) + (kMaxEntries + kMoeMaxExperts) * 4 + 16 + kMaxParts * 2;
    static constexpr int kStages = (232448 - 1024 - 256 - kTableBytes) / kStage;  // 256: barriers
    static constexpr int kBarOffset = kStages * kStage;
    static constexpr int kTables = kBarOffset + (2 * kStages * 8 + 32 + 15) / 16 * 16;
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
    float* red;          // MoeCfg::kRedBytes
};

__device__ __forceinline__ void fail(int* err, volatile uint32_t* abort, int code) {
    report(err, code);
    *abort = 1u;
}

__device__ __forceinline__ unsigned ld_relaxed(const unsigned* p) {
    unsigned v;
    asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

// All threads' earlier writes (ordered before by a CTA barrier) are visible
// to whoever sees the count: the release is cumulative.
__device__ __forceinline__ void grid_arrive(unsigned* bar) {
    asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(bar) : "memory");
}

// Waits, for at most ns, until *bar >= need.
__device__ __forceinline__ bool grid_wait_some(const unsigned* bar, unsigned need, uint64_t ns) {
    const uint64_t t0 = globaltimer_ns();
    while (ld_relaxed(bar) < need)
        if (globaltimer_ns() - t0 > ns) return false;
    asm volatile("fence.acq_rel.gpu;" ::: "memory");
    return true;
}

__device__ __forceinline__ bool grid_wait(const unsigned* bar, unsigned need, volatile uint32_t* abort) {
    const uint64_t t0 = globaltimer_ns();
    while (ld_relaxed(bar) < need) {
        if (*abort) return false;
        if (globaltimer_ns() - t0 > kWaitLimitNs) return false;
    }
    asm volatile("fence.acq_rel.gpu;" ::: "memory");
    return true;
}

// Barrier of the N consumer threads; cons_any: whether any passed true.
template <int N>
__device__ __forceinline__ void cons_bar() {
    asm volatile("bar.sync 2, %0;" ::"n"(N) : "memory");
}

template <int N>
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
        : "r"(v ? 1u : 0u), "n"(N)
        : "memory");
    return r != 0;
}

__device__ __forceinline__ float load_dense(const void* p, int type, long long i) {
    if (type == kTypeF32) return __ldg(static_cast<const float*>(p) + i);
    if (type == kTypeF16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// Eight consecutive values at a 16-byte boundary.
__device__ __forceinline__ void load_dense8(const void* p, int type, long long i, float (&v)[8]) {
    if (type == kTypeF32) {
        Raw8<float> r;
        r.load(static_cast<const float*>(p) + i);
        r.values(v);
    } else if (type == kTypeF16) {
        Raw8<__half> r;
        r.load(static_cast<const __half*>(p) + i);
        r.values(v);
    } else {
        Raw8<__nv_bfloat16> r;
        r.load(static_cast<const __nv_bfloat16*>(p) + i);
        r.values(v);
    }
}

__device__ __forceinline__ void store_dense(void* p, int type, long long i, float v) {
    if (type == kTypeF32)
        static_cast<float*>(p)[i] = v;
    else if (type == kTypeF16)
        static_cast<__half*>(p)[i] = __float2half_rn(v);
    else
        static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// Power of two s with amax / s in [2^14, 2^15), at least 2^-126 (zeros too),
// and its exact reciprocal.
__device__ __forceinline__ float act_scale(float amax, float& inv) {
    const uint32_t ex = (__float_as_uint(amax) >> 23) & 0xFFu;
    const uint32_t se = ex > 15u ? ex - 14u : 1u;
    inv = __uint_as_float((254u - se) << 23);
    return __uint_as_float(se << 23);
}

// Byte of value k (0..127) in an activation block: thread t = k / 32 reads
// 16-byte chunk j = (k % 32) / 8 at (4 j + t) * 16.
__device__ __forceinline__ int act_at(int k) { return (((k >> 3) & 3) * 4 + (k >> 5)) * 16 + (k & 7) * 2; }

// Two values as f16 and, with LO, what that leaves as f16.
template <bool LO>
__device__ __forceinline__ void split_half2(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    memcpy(&hi, &h, 4);
    if constexpr (LO) {
        const float2 f = __half22float2(h);
        const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
        memcpy(&lo, &l, 4);
    }
}

// ---- phase 0: activation blocks of x, router products ----------------------

// A half-warp per block, 8 values per lane.
template <bool LO>
__device__ __forceinline__ void layout_x(const MoeParams& p, int half, int halves, int lane) {
    uint32_t most = 0;
    const int l = lane & 15;
    // the two halves of a warp take the same steps
    for (int task = half; task - (lane >> 4) < p.t * p.kb_h; task += halves) {
        const bool live = task < p.t * p.kb_h;
        const int tok = task / p.kb_h, kb = task - tok * p.kb_h, k = kb * kF8Block + l * 8;
        // a token without a slot (a padded row) may hold anything: it counts as
        // zeros; a lane per slot
        static_assert(kMoeMaxTop <= 16, "a slot per lane");
        bool used = p.router != nullptr;
        if (!used) {
            const bool slot = live && l < p.top &&
                              static_cast<unsigned>(__ldg(p.ids + tok * p.top + l)) < static_cast<unsigned>(p.e);
            used = (__ballot_sync(0xffffffffu, slot) >> (lane & 16) & 0xFFFFu) != 0u;
        }
        float v[8];
        if (live && p.wide && k < p.h) {  // h is a multiple of 16
            load_dense8(p.x, p.type, tok * p.ldx + k, v);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = live && k + i < p.h ? load_dense(p.x, p.type, tok * p.ldx + k + i) : 0.0f;
        }
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            v[i] = used ? v[i] : 0.0f;
            m = max(m, mag_bits(v[i]));
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        most = max(most, m);
        float inv;
        const float s = act_scale(__uint_as_float(m), inv);
        if (live) {
            uint8_t* blk = p.xq + (static_cast<long long>(kb) * p.t + tok) * ActBlock<LO>::kBytes;
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) split_half2<LO>(v[2 * i] * inv, v[2 * i + 1] * inv, hi[i], lo[i]);
            *reinterpret_cast<uint4*>(blk + act_at(l * 8)) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (LO) *reinterpret_cast<uint4*>(blk + 256 + act_at(l * 8)) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
            if (l == 0) *reinterpret_cast<float*>(blk + ActBlock<LO>::kScaleAt) = s;
        }
    }
    if (!mag_finite(most)) report(p.err, kErrNonFinite);
}

// This lane's sums of one expert's row with kRouterTokens tokens, over every
// kRouterWarps-th stretch of k from stretch `from`.
__device__ __forceinline__ void router_dot(const MoeParams& p, int ex, int tok0, int from, int lane,
                                           float (&s)[kRouterTokens]) {
#pragma unroll
    for (int i = 0; i < kRouterTokens; ++i) s[i] = 0.0f;
    if (p.wide) {  // h is a multiple of 8
#pragma unroll 2
        for (int k = from * 256 + lane * 8; k < p.h; k += kRouterWarps * 256) {
            float r[8];
            load_dense8(p.router, p.router_type, ex * p.ld_router + k, r);
#pragma unroll
            for (int i = 0; i < kRouterTokens; ++i) {
                if (tok0 + i >= p.t) break;
                float x[8];
                load_dense8(p.x, p.type, (tok0 + i) * p.ldx + k, x);
#pragma unroll
                for (int j = 0; j < 8; ++j) s[i] = fmaf(r[j], x[j], s[i]);
            }
        }
    } else {
#pragma unroll 4
        for (int k = from * 32 + lane; k < p.h; k += kRouterWarps * 32) {
            const float r = load_dense(p.router, p.router_type, ex * p.ld_router + k);
#pragma unroll
            for (int i = 0; i < kRouterTokens; ++i)
                if (tok0 + i < p.t) s[i] = fmaf(r, load_dense(p.x, p.type, (tok0 + i) * p.ldx + k), s[i]);
        }
    }
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Part `part` of the router products.  Few tasks: warps of a CTA share a
// task's stretches of k; many: a warp takes a task's one after the other.  The
// sums are added in one order, lane by lane over the stretches and then over
// the lanes, so a token's logits do not depend on the tokens beside it.
__device__ __forceinline__ void router_products(const MoeParams& p, const Tables& tb, int part, int warp, int warps, int lane) {
    const int groups = (p.t + kRouterTokens - 1) / kRouterTokens, tasks = p.e * groups;
    float s[kRouterTokens];
    if (tasks <= 2 * static_cast<int>(gridDim.x)) {
        static_assert(kRouterWarps * kRouterTokens * 32 * 4 <= 8192, "sums in tb.red");
        for (int task = part; task < tasks; task += gridDim.x) {
            const int ex = task / groups, tok0 = (task - ex * groups) * kRouterTokens;
            if (warp < kRouterWarps) {
                router_dot(p, ex, tok0, warp, lane, s);
#pragma unroll
                for (int i = 0; i < kRouterTokens; ++i) tb.red[(warp * kRouterTokens + i) * 32 + lane] = s[i];
            }
            __syncthreads();
            if (warp < kRouterTokens && tok0 + warp < p.t) {
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kRouterWarps; ++w) sum += tb.red[(w * kRouterTokens + warp) * 32 + lane];
                sum = warp_sum(sum);
                if (lane == 0) __stcg(p.logits + (tok0 + warp) * p.e + ex, sum);
            }
            __syncthreads();
        }
    } else {
        for (int task = part * warps + warp; task < tasks; task += gridDim.x * warps) {
            const int ex = task / groups, tok0 = (task - ex * groups) * kRouterTokens;
            float sum[kRouterTokens] = {};
            for (int from = 0; from < kRouterWarps; ++from) {
                router_dot(p, ex, tok0, from, lane, s);
#pragma unroll
                for (int i = 0; i < kRouterTokens; ++i) sum[i] += s[i];
            }
#pragma unroll
            for (int i = 0; i < kRouterTokens; ++i) {
                sum[i] = warp_sum(sum[i]);
                if (lane == 0 && tok0 + i < p.t) __stcg(p.logits + (tok0 + i) * p.e + ex, sum[i]);
            }
        }
    }
}

// ---- routing ---------------------------------------------------------------

// Order-preserving integer of a logit, above 0; -0 is 0, NaN sorts last.
__device__ __forceinline__ uint32_t sort_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return 1u;
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

// One token: its `top` largest logits, ties to the lower expert.  PER: experts
// per lane.
template <int PER>
__device__ __forceinline__ void load_logits(const MoeParams& p, int tok, int lane, float (&v)[PER]) {
#pragma unroll
    for (int j = 0; j < PER; ++j)
        v[j] = tok < p.t && lane + 32 * j < p.e ? __ldcg(p.logits + tok * p.e + lane + 32 * j) : -INFINITY;
}

template <int PER>
__device__ __forceinline__ void choose(const MoeParams& p, const Tables& tb, int tok, int lane, const float (&v)[PER]) {
    uint32_t key[PER];
    float vmax = -INFINITY;
    bool finite = true;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int ex = lane + 32 * j;
        finite &= ex >= p.e || isfinite(v[j]);
        key[j] = ex < p.e ? sort_key(v[j]) : 0u;
        vmax = fmaxf(vmax, v[j]);
    }
    if (!finite) report(p.err, kErrNonFinite);
    vmax = warp_max(vmax);
    float ev[PER], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        ev[j] = lane + 32 * j < p.e ? expf(v[j] - vmax) : 0.0f;
        sum += ev[j];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    float chosen = 0.0f, mine = 0.0f;  // lane k keeps slot k
    int mine_e = 0;
    for (int k = 0; k < p.top; ++k) {
        uint32_t best = 0;
#pragma unroll
        for (int j = 0; j < PER; ++j) best = max(best, key[j]);
        best = __reduce_max_sync(0xffffffffu, best);
        uint32_t at = 0xffffffffu;
#pragma unroll
        for (int j = PER - 1; j >= 0; --j)
            if (key[j] == best) at = lane + 32 * j;
        at = __reduce_min_sync(0xffffffffu, at);
        float w = 0.0f;
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (static_cast<uint32_t>(lane + 32 * j) == at) {
                w = ev[j];
                key[j] = 0u;
            }
        w = __shfl_sync(0xffffffffu, w, at & 31);
        chosen += w;
        if (lane == k) {
            mine = w;
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

// A warp's tokens, the next one's logits on their way meanwhile.
template <int PER>
__device__ __forceinline__ void choose_all(const MoeParams& p, const Tables& tb, int warp, int warps, int lane) {
    float v[PER], next[PER];
    load_logits<PER>(p, warp, lane, v);
    for (int tok = warp; tok < p.t; tok += warps) {
        load_logits<PER>(p, tok + warps, lane, next);
        choose<PER>(p, tb, tok, lane, v);
#pragma unroll
        for (int j = 0; j < PER; ++j) v[j] = next[j];
    }
}

// Pairs sorted by expert (then token); experts with pairs become entries of
// at most `cap` pairs each.
__device__ __forceinline__ void build_tables(const MoeParams& p, const Tables& tb, int cap, int warp, int warps, int lane) {
    // a warp per expert, 32 pairs at a time
    const int pairs = p.t * p.top;
    for (int ex = warp; ex < p.e; ex += warps) {
        int n = 0;
        for (int i = lane; i - lane < pairs; i += 32)
            n += __popc(__ballot_sync(0xffffffffu, i < pairs && tb.pair_e[i] == ex));
        if (lane == 0) tb.count[ex] = n;
    }
    __syncthreads();
    if (warp == 0) {
        int pos = 0, ents = 0;
        for (int e0 = 0; e0 < p.e; e0 += 32) {
            const int ex = e0 + lane, n = ex < p.e ? tb.count[ex] : 0, ne = (n + cap - 1) / cap;
            int both = n | (ne << 16);  // pairs and entries before and with this expert
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, both, o);
                if (lane >= o) both += up;
            }
            const int first = pos + (both & 0xFFFF) - n, entry0 = ents + (both >> 16) - ne;
            for (int i = 0; i < ne; ++i) tb.entry[entry0 + i] = (ex << 16) | (first + i * cap);
            if (ex < p.e) tb.count[ex] = n ? first : -1;  // now the expert's first position
            const int all = __shfl_sync(0xffffffffu, both, 31);
            pos += all & 0xFFFF;
            ents += all >> 16;
        }
        if (lane == 0) tb.info[0] = ents, tb.info[1] = pos;
    }
    __syncthreads();
    for (int ex = warp; ex < p.e; ex += warps) {
        int at = tb.count[ex];
        if (at < 0) continue;
        for (int i = lane; i - lane < pairs; i += 32) {
            const bool hit = i < pairs && tb.pair_e[i] == ex;
            const uint32_t hits = __ballot_sync(0xffffffffu, hit);
            if (hit) tb.order[at + __popc(hits & ((1u << lane) - 1u))] = static_cast<short>(i);
            at += __popc(hits);
        }
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

// ---- the line of groups ----------------------------------------------------

struct Line {
    int groups, log_splits, nkb, total;  // groups per (entry, split), splits of k, blocks of k, groups in all
    int each, more;                      // groups per part, and those left over, spread over the parts
    __device__ __forceinline__ Line(int entries, int groups_, int log_splits_, int nkb_)
        : groups(groups_), log_splits(log_splits_), nkb(nkb_), total((entries * groups_) << log_splits_) {
        each = static_cast<int>(static_cast<unsigned>(total) / gridDim.x);
        more = total - each * static_cast<int>(gridDim.x);
    }
    __device__ __forceinline__ int start(int part) const { return part * each + static_cast<int>(static_cast<unsigned>(part * more) / gridDim.x); }
};

// Splits of k for the down product: a part takes q = ceil(groups / parts)
// groups of ceil(kb / splits) blocks.  A stage of q groups takes q blocks'
// time, but at least about three: it holds one block of k of each group, and
// five stages in flight have to cover the latency of memory.  A power of two:
// its logarithm is returned.
__device__ __forceinline__ int choose_splits(const MoeParams& p, int entries, int groups) {
    int best = 0;
    unsigned least = 0xffffffffu;
    for (int log = 0, s = 1; s <= p.max_split && s <= p.kb_f; ++log, s *= 2) {
        const unsigned q = (static_cast<unsigned>(entries * groups * s) + gridDim.x - 1) / gridDim.x;
        const unsigned cost = max(q, 3u) * (static_cast<unsigned>(p.kb_f + s - 1) >> log);
        if (cost < least) {
            least = cost;
            best = log;
        }
    }
    return best;
}

// Up to 8 consecutive groups of the line.  They share the blocks of k, and the
// activation rows of all their entries (consecutive positions) fit a stage:
// groups of several entries go together where k is not cut.
struct Pass {
    int u0, n, split, k0, k1;  // first group in the line
    int pos0, npos;            // positions of its entries
};

struct Walk {
    int cur, end;
    __device__ __forceinline__ Walk(const Line& l, int part) : cur(l.start(part)), end(l.start(part + 1)) {}
    __device__ __forceinline__ bool next(const Line& l, const Tables& tb, int cap, Pass& s) {
        if (cur >= end) return false;
        const int es = cur / l.groups, entry = es >> l.log_splits;
        s.u0 = cur;
        s.split = es - (entry << l.log_splits);
        s.k0 = (s.split * l.nkb) >> l.log_splits;
        s.k1 = ((s.split + 1) * l.nkb) >> l.log_splits;
        int n;
        entry_pairs(tb, entry, cap, s.pos0, n);
        s.npos = n;
        int avail = min((es + 1) * l.groups, end) - cur;
        if (l.log_splits == 0) {
            // on into the next entries, up to 8 groups
            for (int e = entry + 1; avail < kPassGroups && cur + avail < end; ++e) {
                int first;
                entry_pairs(tb, e, cap, first, n);
                if (s.npos + n > cap) break;
                s.npos += n;
                avail = min((e + 1) * l.groups, end) - cur;
            }
        }
        // full passes first: the rest then shares its blocks among more warps
        s.n = min(avail, kPassGroups);
        cur += s.n;
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
    asm(
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

__device__ __forceinline__ uint32_t mul_half2(uint32_t v, __half2 s) {
    __half2 x;
    memcpy(&x, &v, 4);
    x = __hmul2(x, s);
    memcpy(&v, &x, 4);
    return v;
}

template <int NG, bool LO>
struct Consumer {
    using C = MoeCfg<NG, LO>;
    using Hid = typename C::Hid;
    // gate / up (or the two halves of 32 down rows) x token groups x fragment
    float acc[2][NG][4];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int n = 0; n < NG; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[b][n][i] = 0.0f;
    }

    // One block of 128, 64 values (thread t's chunk c of 16) at a time: a
    // group's 16 rows of both boxes times ng token groups.  at: byte of this
    // lane's token's row behind act, per token group.
    // GROUPED: hidden values, a scale per 16 (thread t's two chunks have their
    // own) and remainders.
    // PACKED (remainders, at most 4 tokens): column 2c is token c's f16 values
    // and column 2c + 1 their remainders, in one MMA; unpack() adds them.
    // A pass takes the groups of at least 2^-14 of the largest scale among those
    // whose bit of `left` is set (two per token group), and clears their bits;
    // returns whether any lane has groups left.
    template <bool GROUPED, bool PACKED>
    __device__ __forceinline__ bool block(const uint8_t* rows, const uint8_t* act, const int (&at)[NG], int lane, int ng,
                                          float s0, float s1, uint32_t& left) {
        using Act = ActBlock<LO || GROUPED>;
        constexpr int kTerms = (LO || GROUPED) && !PACKED ? 2 : 1;
        const int g = lane >> 2, t = lane & 3;
        // per token group: the power of two of columns 2t and 2t + 1 (times the
        // weights' scales below), and what brings this lane's chunks to it
        float x0[NG], x1[NG];
        __half2 f[NG][2];
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            if (n >= (PACKED ? 1 : ng)) break;
            const uint8_t* row = act + at[n];
            float xs;
            if constexpr (GROUPED) {
                const float2 s = *reinterpret_cast<const float2*>(row + Act::kScaleAt + t * 8);
                const float u = left >> (2 * n) & 1 ? s.x : 0.0f, v = left >> (2 * n) & 2 ? s.y : 0.0f;
                xs = fmaxf(u, v);
                xs = fmaxf(xs, __shfl_xor_sync(0xffffffffu, xs, 1));
                xs = fmaxf(xs, __shfl_xor_sync(0xffffffffu, xs, 2));
                const float least = xs * kNear;
                const float inv = __uint_as_float((254u << 23) - __float_as_uint(xs));  // powers of two, scales at most 2^114
                // a group of zeros, of scale 0, counts as taken
                const bool far0 = u > 0.0f && u < least, far1 = v > 0.0f && v < least;
                f[n][0] = __float2half2_rn(far0 ? 0.0f : u * inv);
                f[n][1] = __float2half2_rn(far1 ? 0.0f : v * inv);
                if (!far0) left &= ~(1u << (2 * n));
                if (!far1) left &= ~(2u << (2 * n));
            } else {
                xs = *reinterpret_cast<const float*>(row + Act::kScaleAt);
            }
            x0[n] = __shfl_sync(0xffffffffu, xs, 8 * t);
            x1[n] = __shfl_sync(0xffffffffu, xs, 8 * t + 4);
        }
        const bool more = GROUPED && __any_sync(0xffffffffu, left != 0u);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            uint32_t a[2][4][4];  // box, k step, fragment
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const uint8_t* row = rows + b * kBoxBytes + g * kF8Block + ((2 * t + c) ^ g) * 16;
                const uint4 lo = *reinterpret_cast<const uint4*>(row);
                const uint4 hi = *reinterpret_cast<const uint4*>(row + 8 * kF8Block);
                const uint32_t wl[4] = {lo.x, lo.y, lo.z, lo.w}, wh[4] = {hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    a[b][i][0] = e4m3_to_half2(wl[i] & 0xFFFFu);
                    a[b][i][1] = e4m3_to_half2(wh[i] & 0xFFFFu);
                    a[b][i][2] = e4m3_to_half2(wl[i] >> 16);
                    a[b][i][3] = e4m3_to_half2(wh[i] >> 16);
                }
            }
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                if (n >= (PACKED ? 1 : ng)) break;
                const uint8_t* row = act + at[n];
                // two accumulators each: eight MMAs one behind the other would
                // take longer than the block's copy
                float d[2][2][4] = {};
#pragma unroll
                for (int part = 0; part < kTerms; ++part)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        uint4 v = *reinterpret_cast<const uint4*>(row + (PACKED ? g & 1 : part) * 256 + (2 * c + j) * 64 + t * 16);
                        if constexpr (GROUPED) {
                            v.x = mul_half2(v.x, f[n][c]);
                            v.y = mul_half2(v.y, f[n][c]);
                            v.z = mul_half2(v.z, f[n][c]);
                            v.w = mul_half2(v.w, f[n][c]);
                        }
                        mma_f16(d[0][0], a[0][2 * j], v.x, v.y);
                        mma_f16(d[1][0], a[1][2 * j], v.x, v.y);
                        mma_f16(d[0][1], a[0][2 * j + 1], v.z, v.w);
                        mma_f16(d[1][1], a[1][2 * j + 1], v.z, v.w);
                    }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float x = (i & 1) ? x1[n] : x0[n];
                    acc[0][n][i] = fmaf(d[0][0][i] + d[0][1][i], s0 * x, acc[0][n][i]);
                    acc[1][n][i] = fmaf(d[1][0][i] + d[1][1][i], s1 * x, acc[1][n][i]);
                }
            }
        }
        return more;
    }

    // PACKED sums to the plain layout: token c = 2t + j in thread t's column j.
    __device__ __forceinline__ void unpack(int lane) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const float sum = acc[b][0][2 * r] + acc[b][0][2 * r + 1];  // token t
                const int from = (lane & ~3) | ((2 * lane) & 3);
                acc[b][0][2 * r] = __shfl_sync(0xffffffffu, sum, from);
                acc[b][0][2 * r + 1] = __shfl_sync(0xffffffffu, sum, from | 1);
            }
    }

    // Adds the sums of the warps that share this one's group (ways of them,
    // n2 warps apart) to the first one's, in order.
    __device__ __forceinline__ void reduce(float* red, int warp, int lane, int ng, int n2, int ways) {
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            if (n >= ng) break;
            float4* mine = reinterpret_cast<float4*>(red) + (warp * 2) * 32 + lane;
            if (warp >= n2) {
                mine[0] = make_float4(acc[0][n][0], acc[0][n][1], acc[0][n][2], acc[0][n][3]);
                mine[32] = make_float4(acc[1][n][0], acc[1][n][1], acc[1][n][2], acc[1][n][3]);
            }
            cons_bar<C::kConsThreads>();
            if (warp < n2)
                for (int w = 1; w < ways; ++w) {
                    const float4 u = mine[w * n2 * 64], v = mine[w * n2 * 64 + 32];
                    acc[0][n][0] += u.x, acc[0][n][1] += u.y, acc[0][n][2] += u.z, acc[0][n][3] += u.w;
                    acc[1][n][0] += v.x, acc[1][n][1] += v.y, acc[1][n][2] += v.z, acc[1][n][3] += v.w;
                }
            cons_bar<C::kConsThreads>();
        }
    }

    // This group's 16 hidden values per token, from gate and up.
    __device__ __forceinline__ void hidden(const MoeParams& p, int group, int first, int n, int ng, int lane) const {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            if (i >= ng) break;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float h[2];
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float gate = acc[0][i][j + 2 * r];
                    h[r] = gate / (1.0f + expf(-gate)) * acc[1][i][j + 2 * r];
                }
                float m = fmaxf(fabsf(h[0]), fabsf(h[1])), inv;
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
                float sc = act_scale(m, inv);
                if (m == 0.0f) sc = 0.0f;  // zeros ask for no further pass
                const int col = i * 8 + 2 * t + j;
                if (col < n) {
                    uint8_t* blk = p.hq + (static_cast<long long>(group >> 3) * p.t * p.top + first + col) * Hid::kBytes;
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float v = h[r] * inv;
                        const __half hi = __float2half_rn(v);
                        const int at = act_at((group & 7) * 16 + g + 8 * r);
                        *reinterpret_cast<__half*>(blk + at) = hi;
                        *reinterpret_cast<__half*>(blk + 256 + at) = __float2half_rn(v - __half2float(hi));
                    }
                    if (g == 0) reinterpret_cast<float*>(blk + Hid::kScaleAt)[group & 7] = sc;
                    // the rest of the last block: zeros
                    if ((group + 1) * kBoxRows == p.f)
                        for (int rest = (group & 7) + 1; rest < 8; ++rest) {
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const int at = act_at(rest * 16 + g + 8 * r);
                                *reinterpret_cast<__half*>(blk + at) = __half(0.0f);
                                *reinterpret_cast<__half*>(blk + 256 + at) = __half(0.0f);
                            }
                            if (g == 0) reinterpret_cast<float*>(blk + Hid::kScaleAt)[rest] = 0.0f;
                        }
                }
            }
        }
    }

    // This group's 32 down rows of its slots.
    __device__ __forceinline__ void slot_rows(const MoeParams& p, const Tables& tb, int group, int split, int splits,
                                              int first, int n, int ng, int lane) const {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            if (i >= ng) break;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int col = i * 8 + 2 * t + j;
                if (col < n) {
                    float* o = p.pair_out + (static_cast<long long>(tb.order[first + col]) * splits + split) * p.h;
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const int row = group * 32 + b * kBoxRows + g + 8 * r;
                            if (row < p.h) __stcg(o + row, acc[b][i][j + 2 * r]);
                        }
                }
            }
        }
    }
};

// The weighted sums of the slots, a warp per token and 128 columns; slots and
// cuts of k in order, up to eight reads at a time.
__device__ __forceinline__ void combine(const MoeParams& p, const Tables& tb, int log_splits, int warp, int warps, int lane) {
    const int chunks = (p.h + 127) / 128, items = chunks * p.t;
    for (int item = warp; item < items; item += warps) {
        const int tok = item / chunks, col = (item - tok * chunks) * 128 + lane * 4;
        if (col >= p.h) continue;  // h is a multiple of 16
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        const int terms = p.top << log_splits;
        const float* from = p.pair_out + static_cast<long long>(tok) * terms * p.h + col;
        for (int i0 = 0; i0 < terms; i0 += 8) {
            float4 d[8];
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // an empty slot's rows are whatever they were
                const int pair = tok * p.top + (min(i0 + i, terms - 1) >> log_splits);
                const bool live = i0 + i < terms && tb.pair_e[pair] >= 0;
                w[i] = live ? tb.pair_w[pair] : 0.0f;
                d[i] = live ? __ldcg(reinterpret_cast<const float4*>(from + static_cast<long long>(i0 + i) * p.h))
                            : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y.x = fmaf(w[i], d[i].x, y.x);
                y.y = fmaf(w[i], d[i].y, y.y);
                y.z = fmaf(w[i], d[i].z, y.z);
                y.w = fmaf(w[i], d[i].w, y.w);
            }
        }
        const long long o = tok * p.ldo + col;
        store_dense(p.out, p.type, o, y.x);
        store_dense(p.out, p.type, o + 1, y.y);
        store_dense(p.out, p.type, o + 2, y.z);
        store_dense(p.out, p.type, o + 3, y.w);
    }
}

template <int NG, bool LO>
__global__ void __launch_bounds__(MoeCfg<NG, LO>::kThreads, 1) moe_f8_kernel(const __grid_constant__ MoeParams p) {
    using C = MoeCfg<NG, LO>;
    using Act = typename C::Act;
    using Hid = typename C::Hid;
    constexpr int S = C::kStages, kCap = NG * 8;
    constexpr int kConsumers = C::kConsumers, kConsThreads = C::kConsThreads, kThreads = C::kThreads, kWarps = C::kWarps;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::kBarOffset);
    uint64_t* empty = full + S;
    volatile uint32_t* abort = reinterpret_cast<uint32_t*>(empty + S);
    volatile int* ticket = reinterpret_cast<int*>(empty + S) + 2;
    Tables tb;
    tb.red = reinterpret_cast<float*>(smem + C::kTables);
    tb.pair_w = tb.red + C::kRedBytes / 4;
    tb.entry = reinterpret_cast<int*>(tb.pair_w + kMaxPairs);
    tb.count = tb.entry + kMaxEntries;
    tb.info = tb.count + kMoeMaxExperts;
    tb.pair_e = reinterpret_cast<short*>(tb.info + 4);
    tb.order = tb.pair_e + kMaxPairs;
    short* held = tb.order + kMaxPairs;  // this CTA's parts

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int parts = static_cast<int>(gridDim.x);
    if (threadIdx.x == 0) {
        *ticket = static_cast<int>(atomicAdd(p.ctrl + kTicket, 1u));
        for (int s = 0; s < S; ++s) {
            mbar_init(&full[s], kProducers);  // three for weights, one for activations
            mbar_init(&empty[s], kConsumers);
        }
        *abort = 0u;
        fence_mbar_init();
        prefetch_tmap(&p.tm_gate);
        prefetch_tmap(&p.tm_up);
        prefetch_tmap(&p.tm_down);
    }
    __syncthreads();

    // ---- phase 0 ----
    int nheld = 0;
    bool ready = false;
    while (!ready) {
        const int part = *ticket;
        if (part < parts) {
            layout_x<LO>(p, (part * kWarps + warp) * 2 + (lane >> 4), parts * kWarps * 2, lane);
            if (p.router) router_products(p, tb, part, warp, kWarps, lane);
            asm volatile("fence.proxy.async.global;" ::: "memory");
            if (threadIdx.x == 0) held[nheld] = static_cast<short>(part);
            ++nheld;
        }
        __syncthreads();
        bool here = false;
        if (threadIdx.x == 0) {
            if (part < parts) {
                grid_arrive(p.ctrl + kDone);
                here = grid_wait_some(p.ctrl + kDone, parts, kHelpNs);
                if (!here) *ticket = static_cast<int>(atomicAdd(p.ctrl + kTicket, 1u));
            } else {
                // every part is held by a CTA that runs
                here = true;
                if (!grid_wait(p.ctrl + kDone, parts, abort)) fail(p.err, abort, kErrTimeoutGrid);
            }
        }
        ready = __syncthreads_or(here);
    }
    if (!__syncthreads_or(threadIdx.x == 0 && *abort != 0u)) {
        // ---- routing, by every CTA for itself ----
        if (p.router) {
            if (p.e <= 64)
                choose_all<2>(p, tb, warp, kWarps, lane);
            else
                choose_all<kMoeMaxExperts / 32>(p, tb, warp, kWarps, lane);
        } else {
            for (int i = threadIdx.x; i < p.t * p.top; i += kThreads) {
                int ex = p.ids[i];
                const float w = p.weights[i];
                if (ex >= p.e) {
                    if (blockIdx.x == 0) report(p.err, kErrBadIndex);
                    ex = -1;
                }
                if (ex >= 0 && !isfinite(w) && blockIdx.x == 0) report(p.err, kErrNonFinite);
                tb.pair_e[i] = static_cast<short>(ex < 0 ? -1 : ex);
                tb.pair_w[i] = w;
            }
        }
        __syncthreads();
        build_tables(p, tb, kCap, warp, kWarps, lane);
        const int entries = tb.info[0];
        const int groups1 = p.f / kBoxRows, groups2 = (p.h + 31) / 32;
        const Line line1(entries, groups1, 0, p.kb_h);

        if (warp >= kConsumers) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kProdRegs));
            // ---- producers.  Phase 1: each of four warps issues every fourth box (one
            // thread) and every fourth token row (a lane each) of a stage; an issued
            // copy costs its thread 100 to 150 cycles, and one thread for all took
            // longer over a stage than the copies.  Phase 2: three issue the weights,
            // up to S stages ahead of the wait for phase 1, the fourth the hidden
            // values, one copy per stage. ----
            const int pw = warp - kConsumers;
            asm volatile("fence.proxy.async.global;" ::: "memory");
            int g = 0;  // stages issued
            bool ok = true;
            // lane 0 waits for the next stage; all learn
            auto stage_free = [&] {
                if (lane == 0 && g >= S && !wait_or_abort(&empty[g % S], ((g / S) & 1) ^ 1, abort)) {
                    if (!*abort) fail(p.err, abort, kErrTimeoutEmpty);
                    ok = false;
                }
                ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
                return ok;
            };
            Pass s;
            for (int i = 0; ok && i < nheld; ++i) {
                Walk walk(line1, held[i]);
                while (ok && walk.next(line1, tb, kCap, s)) {
                    // few tokens: all of them, in one copy
                    const bool all = p.t <= 8;
                    const int rows = all ? (pw == 0 ? p.t : 0) : max(0, s.npos - pw + kProducers - 1) / kProducers;
                    const uint32_t bytes = (2 * s.n - pw + kProducers - 1) / kProducers * kBoxBytes + rows * Act::kBytes;
                    const CUtensorMap* map = pw & 1 ? &p.tm_up : &p.tm_gate;  // box i: group i / 2, gate or up
                    int ex[2 * kPassGroups / kProducers], row[2 * kPassGroups / kProducers];
#pragma unroll
                    for (int j = 0; j < 2 * kPassGroups / kProducers; ++j) {
                        const int u = min(s.u0 + (pw + j * kProducers) / 2, line1.total - 1), entry = u / line1.groups;
                        ex[j] = tb.entry[entry] >> 16;
                        row[j] = (u - entry * line1.groups) * kBoxRows;
                    }
                    // this lane's token rows
                    constexpr int kRows = (kCap + 127) / 128;
                    int from[kRows];
#pragma unroll
                    for (int r = 0; r < kRows; ++r)
                        from[r] = tb.order[s.pos0 + min(pw + kProducers * (lane + 32 * r), s.npos - 1)] / p.top * Act::kBytes;
                    for (int kb = s.k0; kb < s.k1 && stage_free(); ++kb, ++g) {
                        uint64_t* bar = &full[g % S];
                        uint8_t* dst = smem + g % S * C::kStage;
                        uint8_t* act = dst + kPassGroups * kGroupBytes;
                        const uint8_t* src = p.xq + static_cast<long long>(kb) * p.t * Act::kBytes;
                        if (lane == 0) {
                            mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
                            for (int j = 0; j < 2 * kPassGroups / kProducers; ++j)
                                if (pw + j * kProducers < 2 * s.n)
                                    tma_load_3d(dst + (pw + j * kProducers) * kBoxBytes, map, bar, kb * kF8Block, row[j], ex[j]);
                            if (all && pw == 0) bulk_load(act, src, p.t * Act::kBytes, bar);
                        }
                        __syncwarp();
                        if (!all) {
#pragma unroll
                            for (int r = 0; r < kRows; ++r) {
                                const int i = pw + kProducers * (lane + 32 * r);
                                if (i < s.npos) bulk_load(act + i * Act::kBytes, src + from[r], Act::kBytes, bar);
                            }
                        }
                    }
                }
            }
            const Line line2(entries, groups2, choose_splits(p, entries, groups2), p.kb_f);
            if (ok && pw == kProducers - 1) {
                if (lane == 0 && !grid_wait(p.ctrl + kDone + 32, parts, abort)) {
                    if (!*abort) fail(p.err, abort, kErrTimeoutGrid);
                    ok = false;
                }
                asm volatile("fence.proxy.async.global;" ::: "memory");
                ok = __all_sync(0xffffffffu, ok);
            }
            for (int i = 0; ok && i < nheld; ++i) {
                Walk walk(line2, held[i]);
                while (ok && walk.next(line2, tb, kCap, s)) {
                    constexpr int kEach = (kPassGroups + kProducers - 2) / (kProducers - 1);
                    const uint32_t bytes = max(0, s.n - pw + kProducers - 2) / (kProducers - 1) * kGroupBytes;
                    int ex[kEach], row[kEach];
#pragma unroll
                    for (int j = 0; j < kEach; ++j) {
                        const int u = min(s.u0 + pw + j * (kProducers - 1), line2.total - 1), es = u / line2.groups;
                        ex[j] = tb.entry[es >> line2.log_splits] >> 16;
                        row[j] = (u - es * line2.groups) * 32;
                    }
                    for (int kb = s.k0; kb < s.k1 && stage_free(); ++kb, ++g) {
                        uint64_t* bar = &full[g % S];
                        uint8_t* dst = smem + g % S * C::kStage;
                        if (lane != 0) continue;
                        if (pw == kProducers - 1) {
                            mbar_arrive_expect_tx(bar, s.npos * Hid::kBytes);
                            bulk_load(dst + kPassGroups * kGroupBytes,
                                      p.hq + (static_cast<long long>(kb) * p.t * p.top + s.pos0) * Hid::kBytes,
                                      s.npos * Hid::kBytes, bar);
                        } else {
                            mbar_arrive_expect_tx(bar, bytes);
#pragma unroll
                            for (int j = 0; j < kEach; ++j)
                                if (pw + j * (kProducers - 1) < s.n)
                                    tma_load_3d(dst + (pw + j * (kProducers - 1)) * kGroupBytes, &p.tm_down, bar,
                                                kb * kF8Block, row[j], ex[j]);
                        }
                    }
                }
            }
            __syncwarp();
            // copies in flight must land before the CTA exits
            if (lane == 0)
                for (int i = max(0, g - S); i < g; ++i)
                    if (!mbar_wait(&full[i % S], (i / S) & 1)) {
                        report(p.err, kErrTimeoutDrain);
                        break;
                    }
            __syncwarp();
        } else {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kConsRegs));
            // ---- consumer warps ----
            Consumer<NG, LO> c;
            int stage = 0;
            bool ok = true;
            Line line = line1;
            for (int step = 0; ok && step < 2 * nheld; ++step) {
                const int phase = step < nheld ? 1 : 2, part = held[step < nheld ? step : step - nheld];
                if (step == nheld) line = Line(entries, groups2, choose_splits(p, entries, groups2), p.kb_f);
                Walk walk(line, part);
                Pass s;
                while (ok && walk.next(line, tb, kCap, s)) {
                    // n2 warps with a group each, `ways` of them sharing its blocks
                    const int n2 = s.n > 4 ? 8 : s.n > 2 ? 4 : s.n, ways = kConsumers / n2;
                    const int gi = warp & (n2 - 1), way = warp / n2;
                    const bool mine = gi < s.n;
                    const int es = (s.u0 + (mine ? gi : 0)) / line.groups, entry = es >> line.log_splits;
                    const int group = s.u0 + (mine ? gi : 0) - es * line.groups;
                    int first, n;
                    entry_pairs(tb, entry, kCap, first, n);
                    const int ng = (n + 7) / 8, ex = tb.entry[entry] >> 16;
                    const bool packed = NG == 1 && n <= 4 && (LO || phase == 2);
                    const float *s0, *s1;
                    if (phase == 1) {
                        s0 = p.gate_s + ex * p.gate_ss + static_cast<long long>(group >> 3) * p.kb_h;
                        s1 = p.up_s + ex * p.up_ss + static_cast<long long>(group >> 3) * p.kb_h;
                    } else {
                        s0 = s1 = p.down_s + ex * p.down_ss + static_cast<long long>(group >> 2) * p.kb_f;
                    }
                    // this lane's token's row: its own place, or the token's among all
                    int row_at[NG];
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        // columns behind the last token repeat it; nothing of them is kept
                        const int col = min(packed ? lane >> 3 : i * 8 + (lane >> 2), n - 1);
                        row_at[i] = (phase == 1 && p.t <= 8 ? tb.order[first + col] / p.top : first - s.pos0 + col) *
                                    (phase == 1 ? Act::kBytes : Hid::kBytes);
                    }
                    c.clear();
                    float w0 = __ldg(s0 + min(s.k0 + way, s.k1 - 1)), w1 = __ldg(s1 + min(s.k0 + way, s.k1 - 1));
                    for (int kb = s.k0; kb < s.k1; ++kb, ++stage) {
                        const int st = stage % S;
                        if (!wait_or_abort(&full[st], (stage / S) & 1, abort)) {
                            if (!*abort) fail(p.err, abort, kErrTimeoutFull);  // any lane's wait
                            ok = false;
                        }
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (mine && ((kb - s.k0) & (ways - 1)) == way) {
                            const int nk = min(kb + ways, s.k1 - 1);
                            const float n0 = __ldg(s0 + nk), n1 = __ldg(s1 + nk);
                            const uint8_t* at = smem + st * C::kStage;
                            const uint8_t *rows = at + gi * kGroupBytes, *act = at + kPassGroups * kGroupBytes;
                            uint32_t left = (1u << 2 * ng) - 1u;  // hidden groups still to be added
                            if (phase == 1) {
                                if (LO && NG == 1 && packed)
                                    c.template block<false, LO && NG == 1>(rows, act, row_at, lane, ng, w0, w1, left);
                                else
                                    c.template block<false, false>(rows, act, row_at, lane, ng, w0, w1, left);
                            } else if (NG == 1 && packed) {
                                while (c.template block<true, NG == 1>(rows, act, row_at, lane, ng, w0, w1, left)) {}
                            } else {
                                while (c.template block<true, false>(rows, act, row_at, lane, ng, w0, w1, left)) {}
                            }
                            w0 = n0;
                            w1 = n1;
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&empty[st]);
                    }
                    // one decision for all consumer warps
                    if (cons_any<kConsThreads>(!ok)) {
                        ok = false;
                        break;
                    }
                    if (packed) c.unpack(lane);
                    if (ways > 1) c.reduce(tb.red, warp, lane, (min(s.npos, kCap) + 7) / 8, n2, ways);
                    const bool owner = mine && way == 0;
                    if (phase == 1) {
                        if (owner) c.hidden(p, group, first, n, ng, lane);
                    } else {
                        if (owner) c.slot_rows(p, tb, group, s.split, 1 << line.log_splits, first, n, ng, lane);
                    }
                }
                if (ok) {
                    asm volatile("fence.proxy.async.global;" ::: "memory");
                    cons_bar<kConsThreads>();
                    if (threadIdx.x == 0) grid_arrive(p.ctrl + kDone + 32 * phase);
                }
            }
            // ---- phase 3 ----
            if (threadIdx.x == 0 && ok && !grid_wait(p.ctrl + kDone + 64, parts, abort)) {
                if (!*abort) fail(p.err, abort, kErrTimeoutGrid);
                ok = false;
            }
            if (!cons_any<kConsThreads>(!ok))
                for (int i = 0; i < nheld; ++i) combine(p, tb, line.log_splits, held[i] * kConsumers + warp, parts * kConsumers, lane);
        }
    }
    __syncthreads();
    // the last CTA out returns the words to zero
    if (threadIdx.x == 0) {
        __threadfence();
        if (atomicAdd(p.ctrl + kExit, 1u) == static_cast<unsigned>(parts) - 1) {
            p.ctrl[kTicket] = 0u;
            p.ctrl[kExit] = 0u;
            for (int i = 0; i < 3; ++i) p.ctrl[kDone + 32 * i] = 0u;
        }
    }
}

// (k, rows, experts) map of an expert stack: box 128 bytes x box_rows x 1.
bool make_expert_map(CUtensorMap* map, const MoeWeight& w, int k, int rows, int experts, unsigned box_rows) {
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
    cuuint32_t box[3] = {kF8Block, box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<uint8_t*>(w.w), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Token groups of 8 per expert and entry: twice the mean number of tokens per
// expert, at most all.  An expert with n pairs is n / (8 groups) entries,
// rounded up, and its weights are copied for each: with even routing once, for
// all of 64 tokens on one of 64 experts eight times (2048 / 1024, bf16, 1 of
// 64, launch included: even 123 us, 40 of the tokens on one expert 80, all 49).
int token_groups(int t, int e, int top) {
    const int cap = std::min(t, 2 * ((t * top + e - 1) / e));
    return cap <= 8 ? 1 : cap <= 16 ? 2 : cap <= 32 ? 4 : 8;
}

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// Splits of k (at most 8) that the slots' partial rows have room for: 256 rows.
int split_limit(int pairs) { return std::max(1, std::min(8, 256 / pairs)); }

// Scratch areas in order, after the zeroed header.
struct MoeScratch {
    size_t logits, xq, hq, pair_out, total;
    MoeScratch(int t, int h, int f, int e, int top, int type) {
        const size_t blk = type == kTypeF32 ? ActBlock<true>::kBytes : ActBlock<false>::kBytes, hid = ActBlock<true>::kBytes;
        const size_t kb_h = (h + 127) / 128, kb_f = (f + 127) / 128, pairs = static_cast<size_t>(t) * top;
        logits = 0;
        xq = logits + up256(static_cast<size_t>(t) * e * 4);
        hq = xq + up256(t * kb_h * blk);
        pair_out = hq + up256(pairs * kb_f * hid);
        total = pair_out + pairs * split_limit(static_cast<int>(pairs)) * h * 4;
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
    kern<<<sm_count(), C::kThreads, C::kBytes, s>>>(p);
    return cudaGetLastError();
}

}  // namespace

size_t moe_f8_scratch_bytes(int t, int h, int f, int e, int top, int type) {
    return MoeScratch(t, h, f, e, top, type).total;
}

int launch_moe_f8(const MoeF8& m, int* err, cudaStream_t s) {
    MoeParams p{};
    const MoeScratch sc(m.t, m.h, m.f, m.e, m.top, m.type);
    if (m.scratch_bytes < sc.total) return cudaErrorInvalidValue;
    if (!make_expert_map(&p.tm_gate, m.gate, m.h, m.f, m.e, kBoxRows) ||
        !make_expert_map(&p.tm_up, m.up, m.h, m.f, m.e, kBoxRows) ||
        !make_expert_map(&p.tm_down, m.down, m.f, m.h, m.e, 2 * kBoxRows))
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
    p.max_split = split_limit(m.t * m.top);
    const size_t es = m.type == kTypeF32 ? 4 : 2, rs = m.router_type == kTypeF32 ? 4 : 2;
    p.wide = reinterpret_cast<uintptr_t>(m.x) % 16 == 0 && m.ldx * es % 16 == 0 &&
             (!m.router || (reinterpret_cast<uintptr_t>(m.router) % 16 == 0 && m.ld_router * rs % 16 == 0));
    // lines are ints
    if (sm_count() > kMaxParts || static_cast<long long>(m.f / kBoxRows + 1) * kMaxPairs > 0x7fffffffll ||
        static_cast<long long>(m.h / 32 + 1) * kMaxPairs * 8 > 0x7fffffffll)
        return cudaErrorInvalidValue;
    uint8_t* base = static_cast<uint8_t*>(m.scratch);
    p.ctrl = m.counters;
    p.logits = reinterpret_cast<float*>(base + sc.logits);
    p.xq = base + sc.xq;
    p.hq = base + sc.hq;
    p.pair_out = reinterpret_cast<float*>(base + sc.pair_out);
    p.err = err;
    const bool lo = m.type == kTypeF32;
    switch (token_groups(m.t, m.e, m.top)) {
        case 1: return lo ? launch_cfg<1, true>(p, s) : launch_cfg<1, false>(p, s);
        case 2: return lo ? launch_cfg<2, true>(p, s) : launch_cfg<2, false>(p, s);
        case 4: return lo ? launch_cfg<4, true>(p, s) : launch_cfg<4, false>(p, s);
        default: return lo ? launch_cfg<8, true>(p, s) : launch_cfg<8, false>(p, s);
    }
}

}  // namespace rk
