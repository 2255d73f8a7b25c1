// router_groups.cu - the router over groups of experts (maya_route_groups.cuh): a warp a token.
//
// What bounds it is instructions, some 1650 a token of 256 experts, k = 8 (scores, groups, the lanes' sorting, nine rounds of choice, the k weights in 64 bits), not
// the 1 KB of logits: 8192 tokens 23 us, 0.4 TB/s; issue slots are 60 % busy.  A single token is a chain of latencies, 5.7 us.
#include "maya_route_groups.cuh"

namespace maya {
namespace {

template<int PER>
__global__ void __launch_bounds__(128) router_groups_kernel(const RouteGroups A, int n_tokens, int key_words, int* __restrict__ ids,
                                                            float* __restrict__ weights) {
    extern __shared__ __align__(16) unsigned long long keys[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int64_t t = (int64_t) blockIdx.x * (blockDim.x >> 5) + warp;
    grid_launch_dependents();
    grid_dependency_wait();
    if (t >= n_tokens) return;
    int id[2];
    float w[2];
    route_groups_warp<PER>(A, t, keys + (size_t) warp * key_words, lane, id, w);
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (j * 32 + lane < A.k) {
            ids[t * A.k + j * 32 + lane] = id[j];
            weights[t * A.k + j * 32 + lane] = w[j];
        }
}

}  // namespace
}  // namespace maya

using namespace maya;

extern "C" int maya_router_groups(const maya_route_args* a, void* stream) {
    if (!a) return refuse(MAYA_ERR_ARG);
    if (a->n_tokens <= 0) return MAYA_OK;
    if (!a->logits || !a->ids || !a->weights || a->n_expert <= 0 || a->k <= 0) return refuse(MAYA_ERR_ARG);
    if (a->n_group < 1 || a->n_keep < 1 || a->n_keep > a->n_group || a->n_expert % a->n_group) return refuse(MAYA_ERR_ARG);
    if (a->n_expert > kRouteExpertsMost || a->k > kRouteKMost || a->n_group > kGroupsMost) return refuse(MAYA_ERR_LIMIT);
    const int size = a->n_expert / a->n_group;
    if (a->k > a->n_keep * size) return refuse(MAYA_ERR_LIMIT);
    const RouteGroups A{a->logits, a->bias, a->n_expert, a->k, a->n_group, a->n_keep, a->sigmoid, a->top2, a->norm_w, a->w_scale,
                        size > 1 ? (unsigned) (((1ull << 32) + size - 1) / size) : 0u};
    const int words = a->n_keep < a->n_group ? a->n_group * route_stride(size, route_lanes(a->n_group)) : 0;
    // tokens a block: one while every block can have an SM for itself, else four, as far as their keys fit without a raised limit
    int warps = a->n_tokens <= sm_count() ? 1 : 4;
    while (warps > 1 && (size_t) warps * words * 8 > kSmemNoLimit) warps /= 2;
    const dim3 grid((unsigned) ((a->n_tokens + warps - 1) / warps)), block(32 * warps);
    const size_t smem = (size_t) warps * words * 8;
    cudaStream_t s = as_stream(stream);
    const int per = (a->n_expert + 31) / 32;
#define ROUTE_CASE(P) launch_dependent(router_groups_kernel<P>, grid, block, smem, s, A, a->n_tokens, words, a->ids, a->weights)
    if (per <= 2) ROUTE_CASE(2);
    else if (per <= 4) ROUTE_CASE(4);
    else if (per <= 8) ROUTE_CASE(8);
    else if (per <= 16) ROUTE_CASE(16);
    else if (per <= 32) ROUTE_CASE(32);
    else ROUTE_CASE(64);
#undef ROUTE_CASE
    return note_launch("router_groups");
}
