// maya_scan.cuh - ranks within one thread block of kPlan threads: the sum of a number over the threads in front of each.
#pragma once

#include "maya_common.cuh"

namespace maya {

constexpr int kPlan = 1024;                    // threads that count and rank

struct PlanShared {
    int part[kPlan / 32];
    int total;
};
// The sum of v over the threads in front of this one; total: over all.
__device__ __forceinline__ int rank_of(int v, PlanShared& sh, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += u;
    }
    if (lane == 31) sh.part[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        const int mine = sh.part[lane];
        int in = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, in, o);
            if (lane >= o) in += u;
        }
        sh.part[lane] = in - mine;
        if (lane == 31) sh.total = in;
    }
    __syncthreads();
    const int r = sh.part[warp] + incl - v;
    total = sh.total;
    __syncthreads();                                      // (the next call writes part)
    return r;
}

}  // namespace maya
