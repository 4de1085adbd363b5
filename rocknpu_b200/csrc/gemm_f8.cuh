// What the one-SM (gemm_f8.cu) and two-SM (gemm_f8_pair.cu) kernels of the
// block-scaled e4m3 product share.
#pragma once

#include <cuda.h>

#include "f8.cuh"
#include "kernels.h"
#include "ptx.cuh"

namespace rk {
namespace f8_detail {

struct F8Params {
    CUtensorMap tmap_w, tmap_a;
    const float* w_scale;
    const float* a_scale;
    long long ld_as;
    void* out;
    long long ldo;
    int out_type;
    int m, n, num_kb;
    int tiles_n, tiles_m, group_m;
    int stream;   // blocks of all tiles in one line, cut evenly
    int total;    // stream: blocks; else tiles
    int early_weights;
    float* part;  // [CTA][2][BT / 2][kEpiThreads] partial tiles
    unsigned* counters;
    int* err;
};

// Two-SM 256 x 256 tiles resident at once; one launch over whole tiles.
int pair_slots();
int launch_pair(const F8Params& p, int npairs, cudaStream_t s);

__device__ __forceinline__ void fail(int* err, volatile uint32_t* abort, int code) {
    report(err, code);
    *abort = 1u;
}

}  // namespace f8_detail
}  // namespace rk
