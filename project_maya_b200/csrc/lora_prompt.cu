// lora_prompt.cu - low-rank adapters for prompts (see lora.cu for the operator), on tcgen05.
//
// Three launches:
//   lora_tiles_kernel  one thread block sorts the tokens by adapter into tiles of 128 rows of one adapter (tokens without one last: copied)
//   lora_down_kernel   z = A x of a tile: a cluster of up to eight thread blocks takes a tile, each a part of n_in; their partial sums meet over
//                      distributed shared memory, in the order of the parts, so that no partial sum leaves the chip and none depends on who is first
//   lora_up_kernel     out = y + B z: a thread block takes a tile and 128 outputs.  Its 64 KB of y are asked for, straight into registers, before z is there.
// What bounds it is memory: x once, y and out once; the adapters' matrices come out of L2.
//
// Numbers.  The products run on bf16 matrix instructions.  An f32 is three bf16 terms cut off its mantissa, 8 bits each, exactly; an f16 weight
// two (8 + 3 bits), a bf16 value one.  Terms that are 2^-8 and less of a product are added up apart from the leading ones, and those over two accumulators
// in turn where tensor memory has room: the tensor cores cut every sum towards zero, and fewer and smaller sums are cut by less.  z is scaled in f32 and
// again three terms.
#include "maya_lora.cuh"
#include "maya_scan.cuh"
#include "maya_tcgen05.cuh"

namespace maya {
namespace {

constexpr int kThreads = 256;
constexpr int kChunk = 64;                     // values of a contraction in a stage: 128 bytes of bf16 a row
constexpr int kTileBytes = kLoraTile * kChunk * 2;
constexpr int kOutCols = 128;                  // outputs of a thread block of lora_up_kernel
constexpr uint32_t kBf16 = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t) (128 >> 4) << 24);       // instruction: f32 sums of bf16, 128 rows; + columns / 8 << 17

struct Tiles {
    int* words;                  // [0] error, [1] tiles
    int* adapter;                // [most] of a tile; -1: tokens without one
    int* token;                  // [most][128] of a row; -1: none
    uint16_t* z;                 // [most][128][3][rank] bf16 terms of scale * z
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
    auto group_of = [&](int t) { const int i = A.idx[t]; return i >= 0 && i < n ? i : n; };
    for (int t = tid; t < A.n_tokens; t += kPlan) atomicAdd(&count[group_of(t)], 1);
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
    for (int t = tid; t < A.n_tokens; t += kPlan) G.token[atomicAdd(&count[group_of(t)], 1)] = t;
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

// Shared memory of lora_down_kernel: two stages of x's terms and the weights', over which the partial sums lie at the end.
__host__ __device__ constexpr int x_terms(bool x_bf16) { return x_bf16 ? 1 : 3; }
__host__ __device__ constexpr int w_terms(bool f16) { return f16 ? 2 : 1; }
__host__ __device__ inline int stage_bytes(bool x_bf16, bool f16, int rank) { return x_terms(x_bf16) * kTileBytes + w_terms(f16) * rank * 128; }
__host__ __device__ inline int z_stride(int rank) { return rank + 4; }           // floats: rows of a quarter warp in different banks
__host__ __device__ inline int down_cols(int rank) { return (3 * rank <= 256 ? 3 : 2) * rank; }       // tensor memory: the leading sums (two of them or one), the rest
__host__ __device__ inline int pow2_cols(int c) { int p = 32; while (p < c) p *= 2; return p; }

// ---------------------------------------------------------------- z of a tile
// XB: x is bf16.  F16: weights are.  WI: 16-byte pieces of a weight stage a thread brings (rank * 8 / 256, rounded up).
template<bool XB, bool F16, int WI>
__global__ void __launch_bounds__(kThreads) lora_down_kernel(const Lora A, const Tiles G, int parts) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t done[2];
    __shared__ uint32_t tmem_base;
    const int tid = threadIdx.x, lane = tid & 31;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    const int part = blockIdx.x % parts, tile = blockIdx.x / parts;
    grid_dependency_wait();
    grid_launch_dependents();                  // (behind the wait: what the next launch reads ahead of its own is finished)
    if (tile >= G.words[1]) return;            // (the whole cluster)
    const int adapter = G.adapter[tile];
    if (adapter < 0) return;
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const int rank = A.rank, chunks = (A.n_in + kChunk - 1) / kChunk;
    const int c_first = (int) ((int64_t) chunks * part / parts), c_end = (int) ((int64_t) chunks * (part + 1) / parts);
    const uint32_t stage = (uint32_t) stage_bytes(XB, F16, rank), w_at = x_terms(XB) * kTileBytes, w_next = (uint32_t) rank * 128;
    const int cols = pow2_cols(down_cols(rank)), mains = down_cols(rank) / rank - 1;
    if (tid == 0) {
        mbar_init(&done[0], 1);
        mbar_init(&done[1], 1);
        mbar_fence_init();
    }
    if (warp == 0) tmem_alloc(&tmem_base, (uint32_t) cols);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base, rest = tmem + (uint32_t) (mains * rank), idesc = kBf16 | ((uint32_t) (rank >> 3) << 17);

    // this thread's pieces: 8 values of a row, four rows of x (32 apart) and WI rows of A
    const int c8 = tid & 7;
    const uint16_t* wrow = (const uint16_t*) A.a + ((size_t) adapter * rank + (tid >> 3)) * A.n_in + c8 * 8;
    int tok[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) tok[i] = G.token[(size_t) tile * kLoraTile + (tid >> 3) + 32 * i];
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
            if (in && (tid >> 3) + 32 * j < rank) wr[j] = __ldg((const uint4*) (wrow + (size_t) (32 * j) * A.n_in + c * kChunk));
        }
    };
    bool lost = false;
    int issued = 0;
    load(c_first);
    for (int c = c_first; c < c_end; ++c, ++issued) {
        const int it = c - c_first, s = it & 1;
        const uint32_t at = smem + s * stage;
        if (it >= 2) lost |= !mbar_wait(&done[s], ((it >> 1) - 1) & 1);
        if (!lost) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t off = sw128((tid >> 3) + 32 * i, c8);
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
            for (int j = 0; j < WI; ++j) {
                const int r = (tid >> 3) + 32 * j;
                if (r < rank) weights_to(at + w_at, sw128(r, c8), wr[j], F16, w_next);
            }
        }
        fence_proxy_async();
        if (c + 1 < c_end) load(c + 1);
        lost = __syncthreads_or(lost);
        if (lost) break;
        if (warp == 0) {
            tc_fence_after();
            const uint64_t w0 = smem_desc_sw128(at + w_at), w1 = smem_desc_sw128(at + w_at + w_next);
            mma4_ss(tmem + (uint32_t) ((it % mains) * rank), smem_desc_sw128(at), w0, idesc, it >= mains);
            uint32_t more = it > 0;            // the terms that are less
            if constexpr (!XB) {
                mma4_ss(rest, smem_desc_sw128(at + 2 * kTileBytes), w0, idesc, more);
                mma4_ss(rest, smem_desc_sw128(at + kTileBytes), w0, idesc, 1u);
                more = 1u;
            }
            if constexpr (F16) {
                mma4_ss(rest, smem_desc_sw128(at), w1, idesc, more);
                if constexpr (!XB) mma4_ss(rest, smem_desc_sw128(at + kTileBytes), w1, idesc, 1u);
            }
            mma_commit_elect(smem_u32(&done[s]));
        }
    }
    // the last commit stands for every product in front of it
    const int n = c_end - c_first;
    if (issued > 0) lost |= !mbar_wait(&done[(issued - 1) & 1], ((issued - 1) >> 1) & 1);
    lost = __syncthreads_or(lost);
    if (lost && tid == 0) G.words[0] = 1;
    tc_fence_after();
    const int stride = z_stride(rank);
    {
        const int row = 32 * (warp & 3) + lane, half = rank >> 1, first = (warp >> 2) * half;
        const uint32_t lanes = (uint32_t) (32 * (warp & 3)) << 16, dst = smem + (uint32_t) (row * stride) * 4u;
        for (int c = first; c < first + half; c += 8) {
            float v[8], u[8];
            tmem_ld8(tmem + lanes + (uint32_t) c, v);
            if (mains == 2 && n > 1) {
                tmem_ld8(tmem + lanes + (uint32_t) (rank + c), u);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += u[i];
            }
            if constexpr (!XB || F16) {
                tmem_ld8(rest + lanes + (uint32_t) c, u);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] += u[i];
            }
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
    const float scale = A.scale != nullptr ? A.scale[adapter] : 1.0f;
    const int quads = rank >> 2, rows = kLoraTile / parts;
    for (int i = tid; i < rows * quads; i += kThreads) {
        const int row = part * rows + i / quads, c = (i % quads) * 4;
        const uint32_t from = smem + (uint32_t) (row * stride + c) * 4u;
        float4 v = ld_peer(from, 0);
        for (int p = 1; p < parts; ++p) {
            const float4 u = ld_peer(from, (uint32_t) p);
            v.x += u.x; v.y += u.y; v.z += u.z; v.w += u.w;
        }
        float f[4] = {v.x * scale, v.y * scale, v.z * scale, v.w * scale};
        uint16_t* z = G.z + ((size_t) tile * kLoraTile + row) * 3 * rank + c;
#pragma unroll
        for (int q = 0; q < 3; ++q) {
            uint32_t o[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t a = __float_as_uint(f[2 * j]), b = __float_as_uint(f[2 * j + 1]);
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
constexpr int kStage = 32 * 33;                // floats a warp turns its rows around in
__host__ __device__ constexpr int up_bytes(bool f16) {
    const int operands = (3 + w_terms(f16)) * kTileBytes, turn = (kThreads / 32) * kStage * 4;
    return (operands > turn ? operands : turn) + 1024;
}

template<bool F16>
__global__ void __launch_bounds__(kThreads, 2) lora_up_kernel(const Lora A, const Tiles G) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t done;
    __shared__ uint32_t tmem_base;
    __shared__ int tok[kLoraTile];
    const int tid = threadIdx.x, lane = tid & 31, tile = blockIdx.y, n0 = blockIdx.x * kOutCols;
    const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
    if (tile >= G.words[1]) return;
    const int adapter = G.adapter[tile];
    if (tid < kLoraTile) tok[tid] = G.token[(size_t) tile * kLoraTile + tid];
    if (tid == 0) {
        mbar_init(&done, 1);
        mbar_fence_init();
    }
    __syncthreads();
    // a warp's part of the tile: 32 rows, 64 outputs; a lane has outputs col and col + 32 of every row
    const int row0 = 32 * (warp & 3), col = n0 + (warp >> 2) * 64 + lane;
    float y[32][2];
#pragma unroll
    for (int r = 0; r < 32; ++r) {
        const int t = tok[row0 + r];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            y[r][j] = 0.0f;
            if (A.y != nullptr && t >= 0 && col + 32 * j < A.n_out) y[r][j] = __ldcs(A.y + (int64_t) t * A.ld_y + col + 32 * j);
        }
    }
    auto store = [&](int r, int j, float v) {
        const int t = tok[row0 + r];
        if (t >= 0 && col + 32 * j < A.n_out) __stcs(A.out + (int64_t) t * A.ld_out + col + 32 * j, v);
    };
    grid_launch_dependents();
    grid_dependency_wait();
    if (adapter < 0) {
#pragma unroll
        for (int r = 0; r < 32; ++r)
#pragma unroll
            for (int j = 0; j < 2; ++j) store(r, j, y[r][j]);
        return;
    }
    const uint32_t smem = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* base = smem_raw + (smem - smem_u32(smem_raw));
    if (warp == 0) tmem_alloc(&tmem_base, kOutCols);         // (behind the wait: the launch in front needs tensor memory to get there)
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base, idesc = kBf16 | ((uint32_t) (kOutCols >> 3) << 17);
    const int rank = A.rank, c8 = tid & 7;
    bool lost = false;
    int n = 0;
    for (int k0 = 0; k0 < rank; k0 += kChunk, ++n) {
        if (n > 0) {                                          // one stage: ranks beyond 64 are rare
            lost |= !mbar_wait(&done, (n - 1) & 1);
            lost = __syncthreads_or(lost);
            if (lost) break;
        }
        const bool in = k0 + c8 * 8 < rank;
        uint4 wr[4], zr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int o = n0 + (tid >> 3) + 32 * i;
            wr[i] = make_uint4(0u, 0u, 0u, 0u);
            if (in && o < A.n_out) wr[i] = __ldg((const uint4*) ((const uint16_t*) A.b + ((size_t) adapter * A.n_out + o) * rank + k0 + c8 * 8));
        }
#pragma unroll
        for (int q = 0; q < 3; ++q) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = (tid >> 3) + 32 * i;
                zr[i] = make_uint4(0u, 0u, 0u, 0u);
                if (in) zr[i] = __ldcg((const uint4*) (G.z + (((size_t) tile * kLoraTile + r) * 3 + q) * rank + k0 + c8 * 8));
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t o[4] = {zr[i].x, zr[i].y, zr[i].z, zr[i].w};
                st16(smem + q * kTileBytes + sw128((tid >> 3) + 32 * i, c8), o);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) weights_to(smem + 3 * kTileBytes, sw128((tid >> 3) + 32 * i, c8), wr[i], F16, kTileBytes);
        fence_proxy_async();
        __syncthreads();
        if (warp == 0) {                                      // the smallest terms first: a sum is cut by less while it is small
            tc_fence_after();
            const uint64_t w0 = smem_desc_sw128(smem + 3 * kTileBytes), w1 = smem_desc_sw128(smem + 4 * kTileBytes);
            const uint64_t z0 = smem_desc_sw128(smem), z1 = smem_desc_sw128(smem + kTileBytes), z2 = smem_desc_sw128(smem + 2 * kTileBytes);
            mma4_ss(tmem, z2, w0, idesc, n > 0);
            if constexpr (F16) mma4_ss(tmem, z1, w1, idesc, 1u);
            mma4_ss(tmem, z1, w0, idesc, 1u);
            if constexpr (F16) mma4_ss(tmem, z0, w1, idesc, 1u);
            mma4_ss(tmem, z0, w0, idesc, 1u);
            mma_commit_elect(smem_u32(&done));
        }
    }
    if (n > 0) lost |= !mbar_wait(&done, (n - 1) & 1);
    lost = __syncthreads_or(lost);
    if (lost && tid == 0) G.words[0] = 1;
    tc_fence_after();
    float* turn = (float*) base + warp * kStage;              // (every product is done: the operands' room is free)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        uint32_t v[32];
        tmem_ld32(tmem + ((uint32_t) row0 << 16) + (uint32_t) ((warp >> 2) * 64 + 32 * j), v);
        tmem_wait_ld();
#pragma unroll
        for (int c = 0; c < 32; ++c) turn[lane * 33 + c] = __uint_as_float(v[c]);
        __syncwarp();
        if (!lost) {
#pragma unroll
            for (int r = 0; r < 32; ++r) store(r, j, y[r][j] + turn[r * 33 + lane]);
        }
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, kOutCols);
}

template<class K> bool raise(SmemLimit& limit, K kernel, size_t bytes) { return limit.raise((const void*) kernel, bytes); }

template<bool XB, bool F16, int WI> int launch_down(const Lora& A, const Tiles& G, int parts, cudaStream_t s) {
    static SmemLimit limit;
    // never so little that more thread blocks fit an SM than its 512 columns of tensor memory serve
    const int cols = pow2_cols(down_cols(A.rank)), least = 227 * 1024 / (512 / cols + 1);
    int bytes = 2 * stage_bytes(XB, F16, A.rank);
    const int sums = kLoraTile * z_stride(A.rank) * 4;
    if (bytes < sums) bytes = sums;
    if (bytes < least) bytes = least;
    bytes += 1024;
    if (bytes > 227 * 1024 - 64) return refuse(MAYA_ERR_LIMIT);
    if (!raise(limit, lora_down_kernel<XB, F16, WI>, 227 * 1024 - 64)) return note_launch("lora smem attribute");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned) (G.most * parts));
    cfg.blockDim = dim3(kThreads);
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
template<bool XB, bool F16> int launch_prompt(const Lora& A, const Tiles& G, cudaStream_t s) {
    launch_dependent(lora_tiles_kernel, dim3(1), dim3(kPlan), 0, s, A, G);
    int st = note_launch("lora tiles");
    if (st != MAYA_OK) return st;
    // the fewest parts of n_in that give every SM two thread blocks, a chunk each at least
    const int chunks = (A.n_in + kChunk - 1) / kChunk, tiles = (A.n_tokens + kLoraTile - 1) / kLoraTile;
    int parts = 1;
    while (parts < 8 && 2 * parts <= chunks && tiles * parts < 2 * sm_count()) parts *= 2;
    st = A.rank <= 32 ? launch_down<XB, F16, 1>(A, G, parts, s) : A.rank <= 64 ? launch_down<XB, F16, 2>(A, G, parts, s)
       : A.rank <= 128 ? launch_down<XB, F16, 4>(A, G, parts, s) : launch_down<XB, F16, 8>(A, G, parts, s);
    if (st != MAYA_OK) return st;
    static SmemLimit limit;
    if (!raise(limit, lora_up_kernel<F16>, up_bytes(F16))) return note_launch("lora smem attribute");
    launch_dependent(lora_up_kernel<F16>, dim3((unsigned) ((A.n_out + kOutCols - 1) / kOutCols), (unsigned) G.most), dim3(kThreads), up_bytes(F16), s, A, G);
    return note_launch("lora up");
}

}  // namespace

bool lora_takes_prompt(int n_tokens, int n_adapters) { return n_tokens >= 192 && n_adapters <= kLoraAdaptersMost && n_tokens >= 8 * n_adapters; }
size_t lora_prompt_bytes(int n_tokens, int n_adapters, int rank) { return carve_tiles(n_tokens, n_adapters, rank, nullptr, nullptr); }

int lora_prompt(const Lora& A, int x_is_bf16, int w_is_f16, void* scratch, cudaStream_t s) {
    Tiles G;
    carve_tiles(A.n_tokens, A.n_adapters, A.rank, (uint8_t*) scratch, &G);
    if (x_is_bf16) return w_is_f16 ? launch_prompt<true, true>(A, G, s) : launch_prompt<true, false>(A, G, s);
    return w_is_f16 ? launch_prompt<false, true>(A, G, s) : launch_prompt<false, false>(A, G, s);
}

}  // namespace maya
