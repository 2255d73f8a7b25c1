// lora_prompt.cu - low-rank adapters for prompts (see lora.cu for the operator), on tcgen05.
//
// Three launches:
//   lora_tiles_kernel  one thread block sorts the tokens by adapter into tiles of 128 rows of one adapter (tokens without one last: copied)
//   lora_down_kernel   z = A x of a tile: a cluster of up to eight thread blocks takes a tile, each a part of n_in; their partial sums meet over
//                      distributed shared memory, in the order of the parts, so that no partial sum leaves the chip and none depends on who is first
//   lora_up_kernel     out = y + B z: a thread block takes a run of groups of 64 outputs of a tile.  The first one's y is asked for before z is there.
// What bounds it is memory: x once, y and out once; the adapters' matrices come out of L2.
//
// Numbers.  The products run on bf16 matrix instructions.  An f32 is three bf16 terms cut off its mantissa, 8 bits each, exactly; an f16 weight
// two (8 + 3 bits), a bf16 value one.  Terms that are 2^-8 and less of a product are added up apart from the leading ones, and those over two accumulators
// in turn where tensor memory has room: the tensor cores cut every sum towards zero, and fewer and smaller sums are cut by less.  z is again three terms; scale
// multiplies the sum behind it.
// Infinities.  One of x leaves inf - inf behind its first term and meets the second term of a weight that is 0 (inf * 0): a z that is no number is done over in plain f32, from x
// and A.  An infinite z stands in the third term, which meets weights' first terms alone: these are 0 where the weight is.
#include "maya_lora.cuh"
#include "maya_scan.cuh"
#include "maya_tcgen05.cuh"

namespace maya {
namespace {

constexpr int kDownThreads = 512;
constexpr int kChunk = 64;                     // values of a contraction in a stage: 128 bytes of bf16 a row
constexpr int kTileBytes = kLoraTile * kChunk * 2;
constexpr uint32_t kBf16 = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t) (128 >> 4) << 24);       // instruction: f32 sums of bf16, 128 rows; + columns / 8 << 17

struct Tiles {
    int* words;                  // [0] error, [1] tiles
    int* adapter;                // [most] of a tile; -1: tokens without one
    int* token;                  // [most][128] of a row; -1: none
    uint16_t* z;                 // [most][128][3][rank] bf16 terms of z
    int most;
};

int tiles_most(int n_tokens, int n_adapters) {
    const int groups = n_adapters + 1 < n_tokens ? n_adapters + 1 : n_tokens;
    return n_tokens / kLoraTile + groups;      // every group rounds up
}
size_t up256(size_t v) { return (v + 255) & ~(size_t) 255; }
size_t carve_tiles(int n_tokens, int n_adapters, int rank, uint8_t* base, Tiles* t) {
    const int most = tiles_most(n_tokens, n_adapters);
    const size_t at_adapter = 256, at_token = at_adapter + up256((size_t) most * 4), at_z = at_token + up256((size_t) most * kLoraTile * 4);
    if (t) *t = Tiles{(int*) base, (int*) (base + at_adapter), (int*) (base + at_token), (uint16_t*) (base + at_z), most};
    return at_z + (size_t) most * kLoraTile * 3 * rank * 2;
}

// ---------------------------------------------------------------- tokens by adapter
__global__ void __launch_bounds__(kPlan) lora_tiles_kernel(const Lora A, const Tiles G) {
    __shared__ PlanShared sh;
    __shared__ int count[kLoraAdaptersMost + 1];
    const int tid = threadIdx.x, n = A.n_adapters;
    grid_launch_dependents();
    grid_dependency_wait();
    for (int a = tid; a <= n; a += kPlan) count[a] = 0;
    __syncthreads();
    // A place among a group's tokens for each token: one addition a group and warp (prompts are runs of one adapter), four tokens of a thread on their
    // way at a time.  Places wait for the second pass where z will be.
    const int lane = tid & 31;
    int* places = (int*) G.z;
    auto group_of = [&](int i) { return i >= 0 && i < n ? i : n; };
    for (int t0 = 0; t0 < A.n_tokens; t0 += 4 * kPlan) {
        int i[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) i[q] = t0 + q * kPlan + tid < A.n_tokens ? A.idx[t0 + q * kPlan + tid] : 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int t = t0 + q * kPlan + tid, g = t < A.n_tokens ? group_of(i[q]) : n + 1;
            const unsigned same = __match_any_sync(0xffffffffu, g);
            const int first = __ffs(same) - 1;
            int at = 0;
            if (lane == first && g <= n) at = atomicAdd(&count[g], __popc(same));
            at = __shfl_sync(0xffffffffu, at, first) + __popc(same & ((1u << lane) - 1u));
            if (t < A.n_tokens) places[t] = at;
        }
    }
    __syncthreads();
    int tiles = 0;
    for (int a0 = 0; a0 <= n; a0 += kPlan) {
        const int a = a0 + tid, c = a <= n ? count[a] : 0, mine = (c + kLoraTile - 1) / kLoraTile;
        int total;
        const int first = tiles + rank_of(mine, sh, total);
        for (int j = 0; j < mine; ++j) G.adapter[first + j] = a < n ? a : -1;
        for (int r = c; r < mine * kLoraTile; ++r) G.token[(size_t) first * kLoraTile + r] = -1;
        if (a <= n) count[a] = first * kLoraTile;          // where its next token goes
        tiles += total;
    }
    __syncthreads();
    // (which row of its tiles a token gets changes nothing that is computed for it)
    for (int t0 = 0; t0 < A.n_tokens; t0 += 4 * kPlan) {
        int i[4], at[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int t = t0 + q * kPlan + tid;
            i[q] = t < A.n_tokens ? A.idx[t] : 0;
            at[q] = t < A.n_tokens ? places[t] : 0;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int t = t0 + q * kPlan + tid;
            if (t < A.n_tokens) G.token[count[group_of(i[q])] + at[q]] = t;
        }
    }
    if (tid == 0) G.words[1] = tiles;
}

// ---------------------------------------------------------------- operands
// Offset of 16 bytes of a row in an operand tile (rows of 128 bytes under the 128-byte swizzle).
__device__ __forceinline__ uint32_t sw128(int row, int c) { return (uint32_t) (row * 128 + ((c ^ (row & 7)) << 4)); }
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&r)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
// The leading 8 bits of each of 8 values as bf16; v becomes what is left, exactly.
__device__ __forceinline__ void cut8(float (&v)[8], uint32_t (&o)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t a = __float_as_uint(v[2 * i]), b = __float_as_uint(v[2 * i + 1]);
        o[i] = __byte_perm(a, b, 0x7632);
        v[2 * i] -= __uint_as_float(a & 0xFFFF0000u);
        v[2 * i + 1] -= __uint_as_float(b & 0xFFFF0000u);
    }
}
__device__ __forceinline__ void weights_to(uint32_t tile, uint32_t at, uint4 u, bool f16, uint32_t next) {
    if (f16) {
        float v[8];
        uint32_t o[4];
        weights8<true>(u, v);
        cut8(v, o);
        st16(tile + at, o);
        cut8(v, o);
        st16(tile + next + at, o);
    } else {
        const uint32_t o[4] = {u.x, u.y, u.z, u.w};
        st16(tile + at, o);
    }
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ float4 ld_peer(uint32_t addr, uint32_t rank) {
    float4 v;
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %4, %5;\n\tld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [a];\n\t}"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr), "r"(rank) : "memory");
    return v;
}

// Shared memory of lora_down_kernel: a stage of x's terms and the weights' for each set of warps, over which the partial sums lie at the end.
__host__ __device__ constexpr int x_terms(bool x_bf16) { return x_bf16 ? 1 : 3; }
__host__ __device__ constexpr int w_terms(bool f16) { return f16 ? 2 : 1; }
__host__ __device__ inline int stage_bytes(bool x_bf16, bool f16, int rank) { return x_terms(x_bf16) * kTileBytes + w_terms(f16) * rank * 128; }
__host__ __device__ inline int z_stride(int rank) { return rank + 4; }           // floats: rows of a quarter warp in different banks
__host__ __device__ inline int down_body(bool x_bf16, bool f16, int rank) {
    const int stages = 2 * stage_bytes(x_bf16, f16, rank), sums = kLoraTile * z_stride(rank) * 4;
    return stages > sums ? stages : sums;
}
// Tensor memory: each set's leading sums and, where there is room, the rest apart.
__host__ __device__ inline bool rest_apart(int rank) { return rank <= 128; }
__host__ __device__ inline int set_cols(int rank) { return rest_apart(rank) ? 2 * rank : rank; }
__host__ __device__ inline int pow2_cols(int c) { int p = 32; while (p < c) p *= 2; return p; }

// Four z of one token by the calling warp, in plain f32.  x: its row, a: the first of four rows of A.
template<bool XB, bool F16> __device__ __noinline__ float4 plain_z(const uint8_t* x, const uint16_t* a, int n_in, int lane) {
    float z[4] = {};
    for (int k = lane * 8; k < n_in; k += 256) {
        float v[8];
        if constexpr (XB) {
            weights8<false>(*(const uint4*) (x + 2 * k), v);
        } else {
            const float4 p = *(const float4*) (x + 4 * k), q = *(const float4*) (x + 4 * k + 16);
            v[0] = p.x; v[1] = p.y; v[2] = p.z; v[3] = p.w; v[4] = q.x; v[5] = q.y; v[6] = q.z; v[7] = q.w;
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float w[8];
            weights8<F16>(*(const uint4*) (a + (size_t) r * n_in + k), w);
#pragma unroll
            for (int j = 0; j < 8; ++j) z[r] = __fmaf_rn(w[j], v[j], z[r]);
        }
    }
    return make_float4(warp_sum(z[0]), warp_sum(z[1]), warp_sum(z[2]), warp_sum(z[3]));
}

// ---------------------------------------------------------------- z of a tile
// XB: x is bf16.  F16: weights are.  WI: 16-byte pieces of a weight stage a thread brings (rank * 8 / 256, rounded up).
// Two sets of eight warps take chunks of 64 values in turn, so that one's fence, barrier and products run under the other's cutting of x into terms:
// with one set a chunk took 1.3 us, most of it waiting (4096 tokens, 4096 -> rank 64: kernel 31 us, two sets 24; x is 8 of them at the memory's rate).  Taken
// back: two chunks of a set on their way instead of one (24), x as two 32-bit (tf32) terms, two operations a value instead of six (26).
template<bool XB, bool F16, int WI>
__global__ void __launch_bounds__(kDownThreads, 1) lora_down_kernel(const Lora A, const Tiles G, int parts) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t done[2];                 // of a set: its stage has been read
    __shared__ uint32_t tmem_base;
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0), set = warp >> 3, st = tid & 255;
    const int part = blockIdx.x % parts, tile = blockIdx.x / parts;
    grid_dependency_wait();
    if (tile >= G.words[1]) return;            // (the whole cluster)
    const int adapter = G.adapter[tile];
    if (adapter < 0) return;
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int rank = A.rank, chunks = (A.n_in + kChunk - 1) / kChunk;
    const int c_first = (int) ((int64_t) chunks * part / parts), c_end = (int) ((int64_t) chunks * (part + 1) / parts);
    const uint32_t stage = (uint32_t) stage_bytes(XB, F16, rank), at = smem + set * stage, w_at = at + x_terms(XB) * kTileBytes, w_next = (uint32_t) rank * 128;
    const int cols = pow2_cols(2 * set_cols(rank));
    if (tid == 0) {
        mbar_init(&done[0], 1);
        mbar_init(&done[1], 1);
        mbar_fence_init();
    }
    if (warp == 0) tmem_alloc(&tmem_base, (uint32_t) cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    grid_launch_dependents();                  // (behind the wait: what the next launch reads ahead of its own is finished)
    const bool apart = rest_apart(rank);
    const uint32_t tmem = tmem_base, lead = tmem + (uint32_t) (set * set_cols(rank)), rest = lead + (apart ? (uint32_t) rank : 0u);
    const uint32_t idesc = kBf16 | ((uint32_t) (rank >> 3) << 17);

    // this thread's pieces: 8 values of a row, four rows of x (32 apart) and WI rows of A
    const int c8 = tid & 7, r0 = st >> 3;
    const uint16_t* wrow = (const uint16_t*) A.a + ((size_t) adapter * rank + r0) * A.n_in + c8 * 8;
    int tok[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) tok[i] = G.token[(size_t) tile * kLoraTile + r0 + 32 * i];
    uint4 xr[4][XB ? 1 : 2], wr[WI];
    auto load = [&](int c) {
        const int k = c * kChunk + c8 * 8;
        const bool in = k < A.n_in;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool live = in && tok[i] >= 0;
            xr[i][0] = make_uint4(0u, 0u, 0u, 0u);
            if constexpr (XB) {
                if (live) xr[i][0] = *(const uint4*) ((const uint16_t*) A.x + (int64_t) tok[i] * A.ld_x + k);
            } else {
                xr[i][1] = make_uint4(0u, 0u, 0u, 0u);
                if (live) {
                    const uint4* p = (const uint4*) ((const float*) A.x + (int64_t) tok[i] * A.ld_x + k);
                    xr[i][0] = p[0];
                    xr[i][1] = p[1];
                }
            }
        }
#pragma unroll
        for (int j = 0; j < WI; ++j) {
            wr[j] = make_uint4(0u, 0u, 0u, 0u);
            if (in && r0 + 32 * j < rank) wr[j] = __ldg((const uint4*) (wrow + (size_t) (32 * j) * A.n_in + c * kChunk));
        }
    };
    bool lost = false;
    int issued = 0;
    if (c_first + set < c_end) load(c_first + set);
    for (int c = c_first + set; c < c_end; c += 2) {
        if (issued > 0) lost |= !mbar_wait(&done[set], (issued - 1) & 1);
        if (!lost) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t off = sw128(r0 + 32 * i, c8);
                if constexpr (XB) {
                    const uint32_t o[4] = {xr[i][0].x, xr[i][0].y, xr[i][0].z, xr[i][0].w};
                    st16(at + off, o);
                } else {
                    float v[8] = {__uint_as_float(xr[i][0].x), __uint_as_float(xr[i][0].y), __uint_as_float(xr[i][0].z), __uint_as_float(xr[i][0].w),
                                  __uint_as_float(xr[i][1].x), __uint_as_float(xr[i][1].y), __uint_as_float(xr[i][1].z), __uint_as_float(xr[i][1].w)};
                    uint32_t o[4];
#pragma unroll
                    for (int q = 0; q < 3; ++q) {
                        cut8(v, o);
                        st16(at + q * kTileBytes + off, o);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < WI; ++j)
                if (r0 + 32 * j < rank) weights_to(w_at, sw128(r0 + 32 * j, c8), wr[j], F16, w_next);
        }
        if (c + 2 < c_end) load(c + 2);
        fence_proxy_async();
        lost = named_bar_or(1 + set, 256, lost);
        if (lost) break;
        if ((warp & 7) == 0) {
            tc_fence_after();
            const uint64_t w0 = smem_desc_sw128(w_at), w1 = smem_desc_sw128(w_at + w_next);
            uint32_t more = issued > 0;
            mma4_ss(lead, smem_desc_sw128(at), w0, idesc, more);
            if (!apart) more = 1u;             // the terms that are less
            if constexpr (!XB) {
                mma4_ss(rest, smem_desc_sw128(at + 2 * kTileBytes), w0, idesc, more);
                mma4_ss(rest, smem_desc_sw128(at + kTileBytes), w0, idesc, 1u);
                more = 1u;
            }
            if constexpr (F16) {
                mma4_ss(rest, smem_desc_sw128(at), w1, idesc, more);
                if constexpr (!XB) mma4_ss(rest, smem_desc_sw128(at + kTileBytes), w1, idesc, 1u);
            }
            mma_commit_elect(smem_u32(&done[set]));
        }
        ++issued;
    }
    // the last commit of a set stands for every product of its in front
    if (issued > 0) lost |= !mbar_wait(&done[set], (issued - 1) & 1);
    lost = __syncthreads_or(lost);
    if (lost && tid == 0) G.words[0] = 1;
    tc_fence_after();
    const int stride = z_stride(rank);
    {
        const int row = 32 * (warp & 3) + lane;
        const uint32_t from = tmem + ((uint32_t) (32 * (warp & 3)) << 16), dst = smem + (uint32_t) (row * stride) * 4u, next = (uint32_t) set_cols(rank);
        const bool both = c_end - c_first > 1, small = apart && (!XB || F16);
        for (int c = (warp >> 2) * 8; c < rank; c += 32) {
            float v[8], u[8];
            auto add = [&](uint32_t addr) {
                tmem_ld8(addr, u);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += u[i];
            };
            tmem_ld8(from + (uint32_t) c, v);
            if (both) add(from + next + (uint32_t) c);
            if (small) add(from + (uint32_t) (rank + c));
            if (small && both) add(from + next + (uint32_t) (rank + c));
#pragma unroll
            for (int i = 0; i < 8; i += 4)
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (uint32_t) (c + i) * 4u), "f"(v[i]), "f"(v[i + 1]), "f"(v[i + 2]), "f"(v[i + 3]) : "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, (uint32_t) cols);      // (given back before the cluster is waited for: who waits for tensor memory waits for no cluster)
    cluster_arrive();
    cluster_wait();
    const int quads = rank >> 2, rows = kLoraTile / parts;
    for (int i = tid; i < rows * quads; i += kDownThreads) {        // (whole warps: at least 16 rows of 4 quads)
        const int row = part * rows + i / quads, c = (i % quads) * 4;
        const uint32_t from = smem + (uint32_t) (row * stride + c) * 4u;
        float4 u[8], v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int p = 0; p < 8; ++p)
            if (p < parts) u[p] = ld_peer(from, (uint32_t) p);
#pragma unroll
        for (int p = 0; p < 8; ++p)
            if (p < parts) { v.x += u[p].x; v.y += u[p].y; v.z += u[p].z; v.w += u[p].w; }
        if constexpr (!XB || F16) {
            const float sum = (v.x + v.y) + (v.z + v.w);
            for (unsigned odd = __ballot_sync(0xffffffffu, sum != sum); odd != 0u; odd &= odd - 1u) {
                const int who = __ffs(odd) - 1, r = __shfl_sync(0xffffffffu, row, who), q = __shfl_sync(0xffffffffu, c, who);
                const int t = G.token[(size_t) tile * kLoraTile + r];
                if (t < 0) continue;
                const float4 u = plain_z<XB, F16>((const uint8_t*) A.x + (int64_t) t * A.ld_x * (XB ? 2 : 4), (const uint16_t*) A.a + ((size_t) adapter * rank + q) * A.n_in, A.n_in, lane);
                if (lane == who) v = u;
            }
        }
        float f[4] = {v.x, v.y, v.z, v.w};
        uint16_t* z = G.z + ((size_t) tile * kLoraTile + row) * 3 * rank + c;
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            uint32_t o[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t a = q < 2 && fabsf(f[2 * j]) == INFINITY ? 0u : __float_as_uint(f[2 * j]);
                const uint32_t b = q < 2 && fabsf(f[2 * j + 1]) == INFINITY ? 0u : __float_as_uint(f[2 * j + 1]);
                o[j] = __byte_perm(a, b, 0x7632);
                f[2 * j] -= __uint_as_float(a & 0xFFFF0000u);
                f[2 * j + 1] -= __uint_as_float(b & 0xFFFF0000u);
            }
            *(uint2*) (z + (size_t) q * rank) = make_uint2(o[0], o[1]);
        }
    }
    cluster_arrive();                          // (nobody leaves while others read from it)
    cluster_wait();
}

// ---------------------------------------------------------------- out of a tile
// The pairs of a tile and a group of 64 outputs are shared out evenly, one run of them a thread block.  z's three terms lie in tensor memory; a group's products run
// under the write-back of the one in front.  A warp turns its 32 x 32 sums around in shared memory, so that a lane has four neighbours of a row: 16
// bytes a load of y and a store of out.  y is on its way in registers from the last group's write-back on.
// Ways to this (the kernel alone, 4096 tokens, rank 64 -> 6144, us): a thread block a tile and 128 outputs, 4 bytes a lane 53; several groups a thread block with the
// loads of y between the uses of the last ones, each of which then waits for the loads in front of it, 145; outputs as the product's rows, so
// that nothing has to be turned, 124 and, with fewer instructions, 83; z in shared memory, y by asynchronous copies two groups ahead, two sets of warps a thread block 51: four
// ways through shared memory for every value beside the products' operands; as it is 44, of them 31 at the memory's rate.
constexpr int kUpThreads = 256;
constexpr int kOutCols = 64;
constexpr int kOutBytes = kOutCols * kChunk * 2;              // a group's weights, one term
constexpr int kTurnBytes = 32 * 32 * 4;                       // a warp's part of a group
constexpr int kUpCols = 256;                                  // tensor memory: two groups' sums, then z: 3 * 32 columns
__host__ __device__ constexpr int up_bytes(bool f16) { return 2 * w_terms(f16) * kOutBytes + 8 * kTurnBytes + 1024; }

// (each time anew: kept in registers over the groups, 32 rows' tokens leave too few for y)
__device__ __forceinline__ int look_up(const int* p) {
    int v;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(smem_u32(p)) : "memory");
    return v;
}

// VEC: y and out in whole 16 bytes.  k0: the first of the up to 64 ranks that this launch adds; y is then what the launch in front left.
template<bool F16, bool VEC>
__global__ void __launch_bounds__(kUpThreads, 2) lora_up_kernel(const Lora A, const Tiles G, int k0) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t ready[2];                // a group's sums are there
    __shared__ uint32_t tmem_base;
    __shared__ int tok[kLoraTile];                            // -1: none
    const int tid = threadIdx.x, lane = tid & 31, ld_y = (int) A.ld_y, ld_out = (int) A.ld_out;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    // What is read ahead of the wait was written at least two launches ago, and is read out of L2: L1 may hold what an earlier call left there.
    if (k0 > 0) grid_dependency_wait();                       // (y is the launch in front's out)
    const int groups = (A.n_out + kOutCols - 1) / kOutCols;
    const int tiles = __ldcg(G.words + 1), split = gridDim.x / (tiles > 0 ? tiles : 1);
    int64_t u, u_end;
    if (split >= 4) {                                         // so many thread blocks a tile: none has to begin with another (8 us)
        const int t = blockIdx.x / split, i = blockIdx.x - t * split;
        if (t >= tiles) return;
        u = (int64_t) t * groups + groups * i / split;
        u_end = (int64_t) t * groups + groups * (i + 1) / split;
    } else {
        const int64_t units = (int64_t) tiles * groups;
        u = units * blockIdx.x / gridDim.x;
        u_end = units * (blockIdx.x + 1) / gridDim.x;
    }
    if (u >= u_end) return;
    if (tid == 0) {
        mbar_init(&ready[0], 1);
        mbar_init(&ready[1], 1);
        mbar_fence_init();
    }
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    float4* turn = (float4*) (smem_raw + (smem - smem_u32(smem_raw)) + 2 * w_terms(F16) * kOutBytes + warp * kTurnBytes);
    // a lane's outputs of a group: four neighbours of rows row0, row0 + 4, ..., or (without VEC) one of each of the 32 rows, so that a warp has a line of a row
    constexpr int kRows = VEC ? 8 : 32;
    const int tile_row = 32 * (warp & 3), row0 = VEC ? lane >> 3 : 0, col0 = (warp >> 2) * 32 + (VEC ? (lane & 7) * 4 : lane), rank = A.rank, c8 = tid & 7;
    float y[32];
    int mine[VEC ? 8 : 1];                                    // VEC: the rows' tokens
    auto token = [&](int r) {
        if constexpr (VEC) return mine[r];
        else return look_up(tok + tile_row + r);
    };
    uint4 wr[2];
    int adapter = -1;
    float scale = 1.0f;
    auto fetch = [&](int g) {
        const int n = g * kOutCols + col0;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int t = token(r);
            const int64_t at = (int64_t) t * ld_y;
            const bool has = A.y != nullptr && t >= 0 && n < A.n_out;
            if constexpr (VEC) {
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (has) v = __ldcg((const float4*) (A.y + at + n));
                y[4 * r] = v.x; y[4 * r + 1] = v.y; y[4 * r + 2] = v.z; y[4 * r + 3] = v.w;
            } else {
                y[r] = 0.0f;
                if (has) y[r] = __ldcg(A.y + at + n);
            }
        }
    };
    auto store = [&](int g) {
        const int n = g * kOutCols + col0;
        if (n >= A.n_out) return;
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
            const int t = token(r);
            const int64_t at = (int64_t) t * ld_out;
            if (t < 0) continue;
            if constexpr (VEC) __stcs((float4*) (A.out + at + n), make_float4(y[4 * r], y[4 * r + 1], y[4 * r + 2], y[4 * r + 3]));
            else __stcs(A.out + at + n, y[r]);
        }
    };
    auto weights = [&](int g) {                               // 64 rows of B, 8 pieces each
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int o = g * kOutCols + (tid >> 3) + 32 * q, k = k0 + c8 * 8;
            wr[q] = make_uint4(0u, 0u, 0u, 0u);
            if (k < rank && o < A.n_out) wr[q] = __ldcg((const uint4*) ((const uint16_t*) A.b + ((size_t) adapter * A.n_out + o) * rank + k));
        }
    };
    const uint32_t idesc = kBf16 | ((uint32_t) (kOutCols >> 3) << 17);
    uint32_t tmem = 0u;
    int made = 0;                                             // groups whose products were issued, over all tiles
    bool lost = false, waited = k0 > 0;
    while (u < u_end && !lost) {
        const int tile = (int) (u / groups), g_first = (int) (u - (int64_t) tile * groups);
        const int g_end = (int) min((int64_t) groups, (int64_t) g_first + (u_end - u));
        u += g_end - g_first;
        adapter = __ldcg(G.adapter + tile);
        if (adapter < 0 && (A.y == A.out || k0 > 0)) continue;
        if (adapter >= 0 && A.scale != nullptr) scale = __ldcg(A.scale + adapter);
        __syncthreads();                                      // (the last tile's rows have been looked up)
        if (tid < kLoraTile) tok[tid] = __ldcg(G.token + (size_t) tile * kLoraTile + tid);
        __syncthreads();
        if constexpr (VEC) {
#pragma unroll
            for (int r = 0; r < 8; ++r) mine[r] = look_up(tok + tile_row + row0 + 4 * r);
        }
        fetch(g_first);
        if (adapter >= 0) weights(g_first);
        if (!waited) { grid_dependency_wait(); waited = true; }
        if (adapter < 0) {
            for (int g = g_first; g < g_end; ++g) {
                store(g);
                if (g + 1 < g_end) fetch(g + 1);
            }
            continue;
        }
        if (tmem == 0u) {                                     // (behind the wait: the launch in front needs tensor memory to get there)
            if (warp == 0) tmem_alloc(&tmem_base, kUpCols);
            tc_fence_before();
            __syncthreads();
            tc_fence_after();
            tmem = tmem_base | 0x80000000u;
            grid_launch_dependents();                         // (a block that never gets here: when it ends)
        }
        const uint32_t tm = tmem & 0x7FFFFFFFu, z_tm = tm + 2 * kOutCols;
        // half of a row's terms: 32 values in 16 columns of its lane
        const int half = warp >> 2, k_half = k0 + 32 * half;
        const uint4* zp = (const uint4*) (G.z + ((size_t) tile * kLoraTile + tile_row + lane) * 3 * rank + k_half);
        uint32_t zr[3][16];
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint4 z = make_uint4(0u, 0u, 0u, 0u);
                if (k_half + c * 8 < rank) z = __ldcg((const uint4*) ((const uint16_t*) zp + q * rank) + c);
                zr[q][4 * c] = z.x; zr[q][4 * c + 1] = z.y; zr[q][4 * c + 2] = z.z; zr[q][4 * c + 3] = z.w;
            }
#pragma unroll
        for (int q = 0; q < 3; ++q) tmem_st16(z_tm + ((uint32_t) tile_row << 16) + (uint32_t) (32 * q + 16 * half), zr[q]);
        tmem_wait_st();
        tc_fence_before();                                    // (ahead of the barrier in front of the first products)
        auto stage = [&](int m) {                             // what `weights` brought, for the m-th products
#pragma unroll
            for (int q = 0; q < 2; ++q) weights_to(smem + (uint32_t) ((m & 1) * w_terms(F16) * kOutBytes), sw128((tid >> 3) + 32 * q, c8), wr[q], F16, kOutBytes);
        };
        auto issue = [&]() {                                  // by one warp; the smallest terms first: a sum is cut by less while it is small
            if (warp == 0) {
                const uint32_t wt = smem + (uint32_t) ((made & 1) * w_terms(F16) * kOutBytes), d = tm + (uint32_t) ((made & 1) * kOutCols);
                const uint64_t w0 = smem_desc_sw128(wt), w1 = smem_desc_sw128(wt + kOutBytes);
                mma4_ts(d, z_tm + 64u, w0, idesc, 0u);
                if constexpr (F16) mma4_ts(d, z_tm + 32u, w1, idesc, 1u);
                mma4_ts(d, z_tm + 32u, w0, idesc, 1u);
                if constexpr (F16) mma4_ts(d, z_tm, w1, idesc, 1u);
                mma4_ts(d, z_tm, w0, idesc, 1u);
                mma_commit_elect(smem_u32(&ready[made & 1]));
            }
            ++made;
        };
        int writes = made;
        stage(made);
        if (g_first + 1 < g_end) {
            weights(g_first + 1);
            stage(made + 1);
        }
        fence_proxy_async();
        __syncthreads();
        tc_fence_after();
        issue();
        if (g_first + 1 < g_end) issue();
        for (int g = g_first; g < g_end; ++g, ++writes) {
            lost = __any_sync(0xffffffffu, !mbar_wait(&ready[writes & 1], (writes >> 1) & 1));      // (a warp reads tensor memory as one)
            tc_fence_after();
            if (g + 2 < g_end) weights(g + 2);                // (used below, ahead of the next loads of y: a use waits for what was asked for since, too)
            if (!lost) {
                const uint32_t sums = tm + ((uint32_t) tile_row << 16) + (uint32_t) ((writes & 1) * kOutCols + (warp >> 2) * 32);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float v[16];
                    tmem_ld16(sums + 16u * h, v);
#pragma unroll
                    for (int c = 0; c < 4; ++c)               // (16 bytes of a row at a place that the row's number turns)
                        turn[lane * 8 + ((4 * h + c) ^ (lane & 7))] = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
                }
                __syncwarp();
#pragma unroll
                for (int r = 0; r < kRows; ++r) {
                    if constexpr (VEC) {
                        const int row = row0 + 4 * r;
                        const float4 d = turn[row * 8 + ((lane & 7) ^ (row & 7))];
                        y[4 * r] = __fmaf_rn(scale, d.x, y[4 * r]); y[4 * r + 1] = __fmaf_rn(scale, d.y, y[4 * r + 1]);
                        y[4 * r + 2] = __fmaf_rn(scale, d.z, y[4 * r + 2]); y[4 * r + 3] = __fmaf_rn(scale, d.w, y[4 * r + 3]);
                    } else {
                        y[r] = __fmaf_rn(scale, ((const float*) (turn + r * 8 + ((lane >> 2) ^ (r & 7))))[lane & 3], y[r]);
                    }
                }
                __syncwarp();
                store(g);
                if (g + 2 < g_end) stage(writes);             // (these products are done: their weights' room is free)
            }
            if (g + 1 < g_end) fetch(g + 1);
            fence_proxy_async();
            tc_fence_before();                                // (the sums are read, ahead of the barrier that the next products into them come behind)
            lost = __syncthreads_or(lost);
            tc_fence_after();
            if (lost) break;                                  // nothing more is asked for
            if (g + 2 < g_end) issue();
        }
    }
    // A block whose tiles have nothing to do waits too: were there no others, this launch would end ahead of the one in front, and who waits for this one alone
    // would begin while tiles are still being looked up.
    if (!waited) grid_dependency_wait();
    if (lost) {
        if (tid == 0) G.words[0] = 1;
        for (int m = made; m > 0 && m > made - 2; --m) mbar_wait(&ready[(m - 1) & 1], ((m - 1) >> 1) & 1);        // what is in flight gets its time
    }
    if (tmem != 0u) {
        tc_fence_before();
        __syncthreads();
        if (warp == 0) tmem_dealloc(tmem & 0x7FFFFFFFu, kUpCols);
    }
}

constexpr int kDownMost = 226 * 1024;          // (1 KB is static)

template<class K> bool raise(SmemLimit& limit, K kernel, size_t bytes) { return limit.raise((const void*) kernel, bytes); }

template<bool XB, bool F16, int WI> int launch_down(const Lora& A, const Tiles& G, int parts, cudaStream_t s) {
    static SmemLimit limit;
    const int bytes = down_body(XB, F16, A.rank) + 1024;
    if (!raise(limit, lora_down_kernel<XB, F16, WI>, kDownMost)) return note_launch("lora smem attribute");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned) (G.most * parts));
    cfg.blockDim = dim3(kDownThreads);
    cfg.dynamicSmemBytes = (size_t) bytes;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned) parts;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, lora_down_kernel<XB, F16, WI>, A, G, parts);
    return note_launch("lora down");
}
template<bool F16, bool VEC> int launch_up(const Lora& A, const Tiles& G, int k0, cudaStream_t s) {
    static SmemLimit limit;
    if (!raise(limit, lora_up_kernel<F16, VEC>, up_bytes(F16))) return note_launch("lora smem attribute");
    const int64_t most = (int64_t) ((A.n_out + kOutCols - 1) / kOutCols) * G.most, blocks = 2 * sm_count();
    launch_dependent(lora_up_kernel<F16, VEC>, dim3((unsigned) (most < blocks ? most : blocks)), dim3(kUpThreads), (size_t) up_bytes(F16), s, A, G, k0);
    return note_launch("lora up");
}
template<bool XB, bool F16> int launch_prompt(const Lora& A, const Tiles& G, cudaStream_t s) {
    launch_dependent(lora_tiles_kernel, dim3(1), dim3(kPlan), 0, s, A, G);
    int st = note_launch("lora tiles");
    if (st != MAYA_OK) return st;
    // as many parts of n_in as the SMs have thread blocks for, a quarter more at most, a chunk for each at least
    const int chunks = (A.n_in + kChunk - 1) / kChunk, tiles = (A.n_tokens + kLoraTile - 1) / kLoraTile;
    int parts = 1;
    while (parts < 8 && 2 * parts <= chunks && tiles * parts * 2 <= sm_count() + sm_count() / 4) parts *= 2;
    st = A.rank <= 32 ? launch_down<XB, F16, 1>(A, G, parts, s) : A.rank <= 64 ? launch_down<XB, F16, 2>(A, G, parts, s)
       : A.rank <= 128 ? launch_down<XB, F16, 4>(A, G, parts, s) : launch_down<XB, F16, 8>(A, G, parts, s);
    if (st != MAYA_OK) return st;
    const bool vec = A.n_out % 4 == 0 && aligned16(A.out) && A.ld_out % 4 == 0 && (A.y == nullptr || (aligned16(A.y) && A.ld_y % 4 == 0));
    Lora U = A;
    for (int k0 = 0; k0 < A.rank; k0 += kChunk) {             // ranks beyond 64: a launch for every 64 adds to what the one in front left
        st = vec ? launch_up<F16, true>(U, G, k0, s) : launch_up<F16, false>(U, G, k0, s);
        if (st != MAYA_OK) return st;
        U.y = A.out;
        U.ld_y = A.ld_out;
    }
    return MAYA_OK;
}

}  // namespace

// Few tokens read their adapter's matrices one by one; these kernels begin with 17 us, and a tile that few tokens share costs 1 to 1.4 us.  Measured (4096 -> 6144, few /
// many, us): rank 16, one adapter, 128 tokens 17 / 17, 192 25 / 20, 1024 120 / 29; 8 adapters 192 25 / 24, 256 32 / 24; 64 adapters 512 62 / 96, 1024
// 121 / 102; rank 64, one adapter, 32 tokens 13 / 20, 64 24 / 20, 1024 332 / 34; 8 adapters 64 24 / 28, 96 33 / 28; 64 adapters 256 90 / 114, 384 132 / 115.
static int64_t token_ranks(int n_tokens, int n_adapters, int rank) {
    return (int64_t) n_tokens * rank - (190ll + (rank < 64 ? rank : 64)) * (n_adapters < n_tokens ? n_adapters : n_tokens);
}
bool lora_many_fits(int n_tokens, int n_adapters, int rank) { return n_adapters <= kLoraAdaptersMost && token_ranks(n_tokens, n_adapters, rank) > 0; }
bool lora_many_better(int n_tokens, int n_adapters, int rank, int width) {
    const int launches = (rank + kChunk - 1) / kChunk;        // (each adds 64 ranks and reads and writes out)
    return lora_many_fits(n_tokens, n_adapters, rank) && token_ranks(n_tokens, n_adapters, rank) * width > 11250000ll * (launches + 1);
}
size_t lora_prompt_bytes(int n_tokens, int n_adapters, int rank) { return carve_tiles(n_tokens, n_adapters, rank, nullptr, nullptr); }

int lora_prompt(const Lora& A, int x_is_bf16, int w_is_f16, void* scratch, cudaStream_t s) {
    Tiles G;
    carve_tiles(A.n_tokens, A.n_adapters, A.rank, (uint8_t*) scratch, &G);
    if (x_is_bf16) return w_is_f16 ? launch_prompt<true, true>(A, G, s) : launch_prompt<true, false>(A, G, s);
    return w_is_f16 ? launch_prompt<false, true>(A, G, s) : launch_prompt<false, false>(A, G, s);
}

}  // namespace maya
