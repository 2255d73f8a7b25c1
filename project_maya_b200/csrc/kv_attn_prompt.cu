// kv_attn_prompt.cu - attention over the paged 8-bit cache for prompts (many query rows a sequence), on tcgen05.  bf16 activations, head sizes
// 64 and 128.
//
// A thread block owns 256 rows - (token, head of the group) pairs of one key/value head, two tiles of 128 - and walks over the cache
// blocks they see, 128 tokens a step:
//   warps 0..3, 4..7   softmax of tile 0, 1: a thread a row.  64 scores at a time (a cache block: one scale) from tensor memory, 2^x, P back
//                      to tensor memory as f16 over the scores it came from.
//   warps 8..14        expand the codes of K and V to f16 into the swizzled shared-memory tiles that the tensor cores read, one step
//                      ahead (codes come straight to registers).
//   warp 15            issues the products: S = Q K^T (both operands in shared memory), O += P V (P from tensor memory), with few
//                      instructions and few barriers: what it takes to issue them shows in the whole call's time.
// The two tiles take turns: while one is in its softmax the tensor cores work on the other.  Both bounds are close: a step is 2048 cycles of
// tensor pipe (D = 128; what the operands' way out of shared memory adds is not counted) and 2048 of the exponential's pipe.  Measured, one B200: chunks of 4096
// and 2923 tokens, 32 heads over 8, 421 us, 797 TFLOP/s (418 to 426 from one B200 to another).
// Sequences with fewer rows in the same call come here too, one thread block a head and uncut: a chunk beside single tokens at long contexts is better as two calls.
// What bounds it is the chain from part to part with the products in it, 5200 cycles a step, and 62 us of starts: without the exponentials, the loads or the
// stores of codes it takes as long, without the softmax 378, without the products 357 (of 428 then).  Dropped: the softmax of a row over two threads (486), codes
// staged by bulk copies (446), thread blocks that stay (460).
//
// Numbers.  A query row is scaled by a power of two into f16 (exact for bf16).  With vs the block's scale of V,
//   P = 2^(s + log2 vs - m + 4),  O = sum P code,  l = sum P / vs:
// V's scale rides in the exponent, so P is in f16's range whatever the scales.  m is raised only when a row's maximum passes it by more than 8 (P
// then stays below 2^12): O in tensor memory is rescaled a few times a row instead of at every step.
#include <cuda_fp16.h>

#include "kv_attn.cuh"
#include "maya_tcgen05.cuh"

namespace maya {
namespace {

constexpr int kPThreads = 16 * 32;
constexpr int kExpandWarps = 7, kIssueWarp = 15;
// Registers a thread of each part, out of the 128 a thread that 512 threads are launched with: 256 * 168 + 256 * 88 = 65536.
constexpr int kRegsSoftmax = 168, kRegsOther = 88;
constexpr float kUp = 4.0f;
constexpr int kMetaRing = 4;                     // (a step's numbers are written while the softmax may be three steps behind)

struct StepMeta {                                // of the two cache blocks of a step
    int lb[2];
    float ks[2], lv[2], ivs[2];
};

template<int D> struct PCfg {
    static constexpr int panels = D / 64;
    static constexpr int tile = 128 * D * 2;     // bytes of a 128-row f16 tile (Q, K; V transposed the same)
    static constexpr int q = 0, k = 2 * tile, v = 4 * tile, end = 6 * tile;
    static constexpr size_t smem = (size_t) end + 1024;      // + the start's rounding to 1024
    static constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t) (64 >> 3) << 17) | ((uint32_t) (128 >> 4) << 24);
    static constexpr uint32_t idesc_o = (1u << 4) | ((uint32_t) (D >> 3) << 17) | ((uint32_t) (128 >> 4) << 24);
    static constexpr int col_s = 0, col_o = 256; // tensor memory: S of tile x's even blocks at 128 x, of odd ones at 128 x + 64, O at 256 + D x
};

__device__ __forceinline__ float ex2p(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// two f32 operations at once; the largest of three
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(*(unsigned long long*) &d) : "l"(*(unsigned long long*) &a), "l"(*(unsigned long long*) &b), "l"(*(unsigned long long*) &c));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(*(unsigned long long*) &d) : "l"(*(unsigned long long*) &a), "l"(*(unsigned long long*) &b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint32_t half2_of(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*) &h;
}
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// Four K = 16 products one behind the other (32 bytes of a 128-byte row on each), operands in shared memory (SS) or A in tensor memory (TS); `acc` = 0: the first
// overwrites.  By one elected lane of a converged warp.  (In one piece, so that the issuing warp keeps ahead of the tensor cores.)
__device__ __forceinline__ void mma4_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred e, p, q;\n\t.reg .b64 b1, b2, b3;\n\t.reg .b64 a1, a2, a3;\n\tadd.s64 a1, %1, 2;\n\tadd.s64 a2, %1, 4;\n\tadd.s64 a3, %1, 6;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 q, 0, 0;\n\tadd.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, q;\n\t"
        "}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void mma4_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred e, p, q;\n\t.reg .b64 b1, b2, b3;\n\t.reg .b32 a1, a2, a3;\n\tadd.s32 a1, %1, 8;\n\tadd.s32 a2, %1, 16;\n\tadd.s32 a3, %1, 24;\n\t"
        "setp.ne.b32 p, %4, 0;\n\tsetp.eq.b32 q, 0, 0;\n\tadd.s64 b1, %2, 2;\n\tadd.s64 b2, %2, 4;\n\tadd.s64 b3, %2, 6;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, q;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, q;\n\t"
        "}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}

template<int D>
__global__ void __launch_bounds__(kPThreads, 1) prompt_kernel(const KvView C, const BatchView B, const AttnView A) {
    using K = PCfg<D>;
    constexpr int P = K::panels;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t k_full[2], k_free[2], v_full[2], v_free[2], s_full[2], p_ready[2][2], pv_done, o_done[2], q_ready[2];
    __shared__ StepMeta meta[kMetaRing];
    __shared__ uint32_t tmem_base;
    __shared__ int lost;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    uint8_t* smem = (uint8_t*) (((uintptr_t) smem_raw + 1023) & ~(uintptr_t) 1023);

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], kExpandWarps); mbar_init(&k_free[i], 1); mbar_init(&v_full[i], kExpandWarps); mbar_init(&v_free[i], 1);
            mbar_init(&s_full[i], 1); mbar_init(&p_ready[i][0], 4); mbar_init(&p_ready[i][1], 4);
            mbar_init(&o_done[i], 1); mbar_init(&q_ready[i], 4);
        }
        mbar_init(&pv_done, 1);
        lost = 0;
        mbar_fence_init();
    }
    if (warp == kIssueWarp) tmem_alloc(&tmem_base, 512);
    grid_launch_dependents();
    grid_dependency_wait();

    // ---- the rows, and the cache blocks they see
    const int h = blockIdx.x % C.n_kv, tile = blockIdx.x / C.n_kv, si = tile % B.n_seq, r0 = (A.row_tiles - 1 - tile / B.n_seq) * 256;   // every sequence's last rows first
    const Seq s = seq_of(B, si);
    const int n_rows = s.n_new * A.group, first = s.len - s.n_new;
    const bool here = r0 < n_rows;
    const int last_row = min(r0 + 256, n_rows) - 1;
    const int pos_lo = first + r0 / A.group, pos_hi = here ? first + last_row / A.group : -1;
    const int b_first = A.window > 0 ? max(0, pos_lo - A.window + 1) / kKvBlock : 0;
    // (few tiles over a long context: a tile's blocks in A.fixed pieces, whose parts the join puts together)
    const int all_blocks = pos_hi < 0 ? 0 : max(0, pos_hi / kKvBlock + 1 - b_first), cuts = max(1u, A.fixed), each = (all_blocks + cuts - 1) / cuts;
    const int b_lo = b_first + (int) blockIdx.z * each, n_blocks = max(0, min(each, all_blocks - (int) blockIdx.z * each));
    const int steps = (n_blocks + 1) / 2;
    const int tiles = here && n_rows - r0 > 128 ? 2 : 1;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
        if (mbar_wait(bar, parity)) return true;
        lost = 1;
        return false;
    };

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base;

    // (each part sets its registers in a branch of its own: where paths meet the smallest number holds)
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
        if (warp != kIssueWarp) {
            // ================================================================ codes -> f16 operands
            // A warp takes every seventh group of eight rows of a tile, a lane 16 codes of it: group u lies 1024 u bytes into the f16 tile, for keys
            // (panel, block, tokens) and for values (block, values) alike.
            constexpr int groups = 128 * D / 512, pieces = (groups + kExpandWarps - 1) / kExpandWarps;
            const int cw = warp - 8, r8 = lane >> 2, c4 = lane & 3;
            const uint32_t to0 = r8 * 128 + (((2 * c4) ^ r8) << 4), to1 = r8 * 128 + (((2 * c4 + 1) ^ r8) << 4);
            int batch = -1;
            int my_bh = -1, my_lb = -1;
            float my_ks = 0.0f, my_vs = 0.0f;
            auto look_up = [&](int b) {                                     // cache block b_lo + b of this range: 32 at a time, a lane each
                if ((b >> 5) != batch) {
                    batch = b >> 5;
                    const int x = (batch << 5) + lane;
                    my_lb = x < n_blocks ? b_lo + x : -1;
                    const int phys = my_lb >= 0 ? block_of(C, si, my_lb) : -1;
                    my_bh = phys >= 0 ? phys * C.n_kv + h : -1;
                    my_ks = my_bh >= 0 ? C.k_scale[my_bh] : 0.0f;
                    my_vs = my_bh >= 0 ? C.v_scale[my_bh] : 0.0f;
                }
            };
            uint4 cur[pieces], nxt[pieces];
            int bh[2];                                                      // the step's blocks and head in the cache, -1: none
            auto load = [&](uint4 (&w)[pieces], const uint8_t* cache, bool val) {
                const uint8_t* src[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) src[x] = cache + (size_t) max(bh[x], 0) * (kKvBlock * D) + lane * 16;
#pragma unroll
                for (int i = 0; i < pieces; ++i) {
                    const int u = cw + i * kExpandWarps, x = val ? u / (D / 8) : (u >> 3) & 1;
                    const int at = val ? u % (D / 8) : (u >> 4) * 8 + (u & 7);                             // group of the block's 512-byte groups
                    w[i] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
                    if (u < groups && (x == 0 ? bh[0] : bh[1]) >= 0) w[i] = *(const uint4*) ((x == 0 ? src[0] : src[1]) + at * 512);
                }
            };
            auto store = [&](const uint4 (&w)[pieces], uint8_t* dst) {
#pragma unroll
                for (int i = 0; i < pieces; ++i) {
                    const int u = cw + i * kExpandWarps;
                    if (u >= groups) break;
                    uint32_t o[8];
                    codes_to_half(w[i].x, o[0], o[1]); codes_to_half(w[i].y, o[2], o[3]);
                    codes_to_half(w[i].z, o[4], o[5]); codes_to_half(w[i].w, o[6], o[7]);
                    *(uint4*) (dst + u * 1024 + to0) = make_uint4(o[0], o[1], o[2], o[3]);
                    *(uint4*) (dst + u * 1024 + to1) = make_uint4(o[4], o[5], o[6], o[7]);
                }
                fence_proxy_async();
                __syncwarp();
            };
            auto find = [&](int j) {                                        // the step's two blocks
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    look_up(2 * j + x);
                    bh[x] = __shfl_sync(0xffffffffu, my_bh, (2 * j + x) & 31);
                }
                if (warp == 8 && ((2 * j) & 31) == (lane & 30)) {           // their numbers, from the two lanes that have them
                    StepMeta& m = meta[j % kMetaRing];
                    const float vs = fmaxf(my_vs, kVsLeast);
                    m.lb[lane & 1] = my_bh >= 0 ? my_lb : -1;
                    m.ks[lane & 1] = my_ks;
                    m.lv[lane & 1] = __log2f(vs);
                    m.ivs[lane & 1] = __fdividef(1.0f, vs);
                }
            };
            if (here && steps > 0) {
                find(0);
                load(cur, C.k, false);
                for (int j = 0; j < steps; ++j) {
                    load(nxt, C.v, true);                                         // this step's values, under the conversion of its keys
                    if (j >= 2 && !wait(&k_free[j & 1], ((j >> 1) - 1) & 1)) break;
                    store(cur, smem + K::k + (j & 1) * K::tile);
                    if (lane == 0) mbar_arrive_one(&k_full[j & 1]);
                    if (j + 1 < steps) {
                        find(j + 1);
                        load(cur, C.k, false);
                    }
                    if (j >= 2 && !wait(&v_free[j & 1], ((j >> 1) - 1) & 1)) break;
                    store(nxt, smem + K::v + (j & 1) * K::tile);
                    if (lane == 0) mbar_arrive_one(&v_full[j & 1]);
                }
            }
        } else if (here) {
            // ================================================================ products
            const uint32_t base = smem_u32(smem);
            // k counts cache blocks of 64 tokens; even and odd ones have their own scores, so that the next block's are there when the softmax of
            // this one ends.  (Products run in the order they are issued in: P of block k - 1 has been read before S of k + 1 takes its place.)
            const int blocks = 2 * steps;
            auto scores = [&](int x, int k) {
                const uint32_t qa = base + K::q + x * K::tile, ka = base + K::k + ((k >> 1) & 1) * K::tile + (k & 1) * (64 * 128);
#pragma unroll
                for (int p = 0; p < P; ++p)
                    mma4_ss(tmem + K::col_s + 128 * x + 64 * (k & 1), smem_desc_sw128(qa + p * (128 * 128)), smem_desc_sw128(ka + p * (128 * 128)), K::idesc_s, p);
            };
            bool ok = steps == 0 || (wait(&k_full[0], 0) && wait(&q_ready[0], 0) && (tiles == 1 || wait(&q_ready[1], 0)));
            tc_fence_after();
            if (ok && steps > 0) {
                for (int x = 0; x < tiles; ++x) scores(x, 0);
                mma_commit_elect(smem_u32(&s_full[0]));
            }
            for (int k = 0; k < blocks && ok; ++k) {
                const int j = k >> 1;
                if (k + 1 < blocks) {
                    const int j1 = (k + 1) >> 1;
                    if (j1 != j) ok = wait(&k_full[j1 & 1], (j1 >> 1) & 1);
                    if (!ok) break;
                    tc_fence_after();
                    scores(0, k + 1);
                    if (tiles > 1) scores(1, k + 1);
                    mma_commit_elect(smem_u32(&s_full[(k + 1) & 1]));
                    if (j1 == j) mma_commit_elect(smem_u32(&k_free[j & 1]));
                }
                if ((k & 1) == 0) ok = wait(&v_full[j & 1], (j >> 1) & 1);
                const uint32_t va = base + K::v + (j & 1) * K::tile + (k & 1) * (D * 128);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    if (x >= tiles || !ok) break;
                    ok = wait(&p_ready[x][k & 1], j & 1);
                    if (!ok) break;
                    tc_fence_after();
                    mma4_ts(tmem + K::col_o + D * x, tmem + K::col_s + 128 * x + 64 * (k & 1), smem_desc_sw128(va), K::idesc_o, k);
                    if (k + 1 == blocks) mma_commit_elect(smem_u32(&o_done[x]));
                }
                if (ok && (k & 1)) mma_commit_elect(smem_u32(&v_free[j & 1]));
                if (ok && k + 2 == blocks) mma_commit_elect(smem_u32(&pv_done));
            }
            if (!ok && steps > 0) {                                         // what has been issued ends before the memory is given back
                mma_commit_elect(smem_u32(&o_done[1]));
                mbar_wait(&o_done[1], 0);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        if (here && warp < 4 * tiles) {
            // ================================================================ softmax, a row a thread
            const int x = warp >> 2, row = r0 + tid;
            // ---- queries into shared memory: row r of tile x is thread 128 x + r
            float qinv;
            {
                uint8_t* dst = smem + K::q + (warp >> 2) * K::tile;
                const int r = tid & 127;
                uint32_t w[D / 2];
                if (row < n_rows) {
                    const uint16_t* src = (const uint16_t*) A.q + (size_t) (s.row + row / A.group) * A.ld_q + (size_t) (h * A.group + row % A.group) * D;
                    if (A.wide_q) {
#pragma unroll
                        for (int i = 0; i < D / 8; ++i) *(uint4*) &w[4 * i] = ((const uint4*) src)[i];
                    } else {
#pragma unroll
                        for (int i = 0; i < D / 2; ++i) w[i] = src[2 * i] | (uint32_t) src[2 * i + 1] << 16;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < D / 2; ++i) w[i] = 0u;
                }
                float amax = 0.0f;
#pragma unroll
                for (int i = 0; i < D / 2; ++i) amax = fmaxf(amax, fmaxf(fabsf(__uint_as_float(w[i] << 16)), fabsf(__uint_as_float(w[i] & 0xFFFF0000u))));
                const int e2 = up_of_row(amax);    // amax * 2^e2 in [2^11, 2^12)
                const float up = __uint_as_float((uint32_t) (127 + e2) << 23);
                qinv = scale_of_row(amax, __uint_as_float((uint32_t) (127 - e2) << 23) * A.scale_log2);
#pragma unroll
                for (int c = 0; c < D / 8; ++c) {
                    uint4 o;
                    uint32_t* ow = (uint32_t*) &o;
#pragma unroll
                    for (int i = 0; i < 4; ++i) ow[i] = half2_of(__uint_as_float(w[4 * c + i] << 16) * up, __uint_as_float(w[4 * c + i] & 0xFFFF0000u) * up);
                    *(uint4*) (dst + (c >> 3) * (128 * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = o;
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive_one(&q_ready[warp >> 2]);
            }
            const uint32_t lane_base = tmem + ((uint32_t) (32 * (warp & 3)) << 16);
            const uint32_t at_s = lane_base + K::col_s + 128 * x, at_o = lane_base + K::col_o + D * x;
            const int pos = row < n_rows ? first + row / A.group : 0x3fffffff;
            const int wlo = __reduce_min_sync(0xffffffffu, pos), whi = first + min(last_row, r0 + warp * 32 + 31) / A.group;
            float m = kNone, l = 0.0f;
            bool ok = true;
#pragma unroll 1
            for (int k = 0; k < 2 * steps; ++k) {                       // (not unrolled: the parts' code side by side is more than the instruction cache holds)
                    if (!wait(&s_full[k & 1], (k >> 1) & 1)) { ok = false; break; }
                    tc_fence_after();
                    const uint32_t at_k = at_s + 64 * (k & 1);
                    const StepMeta& sm = meta[(k >> 1) % kMetaRing];
                    const int lb = sm.lb[k & 1];
                    const float lv = sm.lv[k & 1], ivs = sm.ivs[k & 1];
                    float f = qinv * sm.ks[k & 1];
                    uint32_t v[64];
                    tmem_ld32(at_k, *(uint32_t(*)[32]) &v[0]);
                    tmem_ld32(at_k + 32, *(uint32_t(*)[32]) &v[32]);
                    tmem_wait_ld();
                    const int tb = lb >= 0 ? lb * kKvBlock : 0x3ffffffe;    // (no block: behind every row)
                    if (tb + kKvBlock - 1 > wlo || (A.window > 0 && tb <= whi - A.window)) {      // not visible to every row in whole
                        const int from = A.window > 0 && pos != 0x3fffffff ? pos - A.window - tb : -1, to = lb >= 0 ? pos - tb : -1;
#pragma unroll
                        for (int i = 0; i < 64; ++i) v[i] = __float_as_uint(i <= to && i > from ? __uint_as_float(v[i]) * f : kNone);
                        f = 1.0f;
                    }
                    float mx[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = fmaxf(__uint_as_float(v[e]), __uint_as_float(v[e + 4]));
#pragma unroll
                    for (int i = 8; i < 64; i += 8)
#pragma unroll
                        for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(v[i + e]), __uint_as_float(v[i + e + 4]));
                    const float top = fmaf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), f, lv);
                    if (__any_sync(0xffffffffu, top > m + kRise || (m == kNone && top > kNone))) {      // the warp's rows are rescaled together
                        const bool mine = top > m + kRise || m == kNone;
                        const float up = mine ? top : m;
                        const float alpha = !mine ? 1.0f : m == kNone ? 0.0f : ex2p(m - up);
                        m = up;
                        l *= alpha;
                        if (k > 0) {
                            // O up to the block before is there when the next scores are, which are issued behind it; at the last block it has a barrier of its own.
                            if (!(k + 1 < 2 * steps ? wait(&s_full[(k + 1) & 1], ((k + 1) >> 1) & 1) : wait(&pv_done, 0))) { ok = false; break; }
                            tc_fence_after();
#pragma unroll 1
                            for (int d = 0; d < D; d += 16) {
                                float o[16];
                                tmem_ld16(at_o + d, o);
                                uint32_t ow[16];
#pragma unroll
                                for (int i = 0; i < 16; ++i) ow[i] = __float_as_uint(o[i] * alpha);
                                tmem_st16(at_o + d, ow);
                            }
                            tmem_wait_st();
                        }
                    }
                    const float off = m == kNone ? kNone : lv - m + kUp;
                    float2 sum[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
                    const float2 f2 = make_float2(f, f), off2 = make_float2(off, off);
#pragma unroll
                    for (int i = 0; i < 64; i += 32) {
                        uint32_t p[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float2 y = fma2(make_float2(__uint_as_float(v[i + e]), __uint_as_float(v[i + e + 1])), f2, off2);
                            y.x = ex2p(y.x);
                            y.y = ex2p(y.y);
                            sum[(e >> 1) & 1] = add2(sum[(e >> 1) & 1], y);
                            p[e / 2] = half2_of(y.x, y.y);
                        }
                        tmem_st16(at_k + i / 2, p);
                    }
                    sum[0] = add2(sum[0], sum[1]);
                    l = fmaf(sum[0].x + sum[0].y, ivs, l);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_one(&p_ready[x][k & 1]);
            }
            // ---- O / l
            if (ok && steps > 0) ok = wait(&o_done[x], 0);
            tc_fence_after();
            if (ok) {                                                       // (warp-uniform: a wait runs out for a whole warp)
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;                  // (a row that saw nothing; a NaN stays one)
                const int n = s.row + row / A.group, hq = h * A.group + row % A.group;
                const size_t part = (((size_t) (si * A.row_tiles + A.row_tiles - 1 - r0 / 256) * C.n_kv + h) * A.fixed + blockIdx.z) * 256 + tid;
                const bool cut = A.fixed > 1;
                uint16_t* dst = (uint16_t*) A.out + ((size_t) n * A.n_q + hq) * D;
#pragma unroll
                for (int d = 0; d < D; d += 16) {
                    float o[16];
                    if (steps > 0) tmem_ld16(at_o + d, o);
                    else
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] = 0.0f;
                    if (cut) {
                        if (row < n_rows)
#pragma unroll
                            for (int i = 0; i < 16; i += 4) *(float4*) (A.part_o + part * D + d + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                    } else if (row < n_rows) {
                        uint32_t w[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const __nv_bfloat162 b = __floats2bfloat162_rn(l == 0.0f ? 0.0f : o[2 * i] * inv, l == 0.0f ? 0.0f : o[2 * i + 1] * inv);
                            w[i] = *(const uint32_t*) &b;
                        }
                        ((uint4*) (dst + d))[0] = make_uint4(w[0], w[1], w[2], w[3]);
                        ((uint4*) (dst + d))[1] = make_uint4(w[4], w[5], w[6], w[7]);
                    }
                }
                if (cut && row < n_rows) A.part_ml[part] = make_float2(m, l);
                else if (A.lse != nullptr && row < n_rows)
                    A.lse[(size_t) n * A.n_q + hq] = lse_of(m, l, kUp);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kIssueWarp) tmem_dealloc(tmem, 512);
    if (tid == 0 && lost) atomicExch(A.error, 1u);
}

template<int D> int launch_prompt(const maya_kv_cache& c, const maya_attn_batch& b, AttnView A, cudaStream_t s) {
    const long long rows = (long long) b.max_new * A.group;
    A.row_tiles = (int) ((rows + 255) / 256);
    const long long tiles = (long long) A.row_tiles * b.n_seq;
    // Pieces: as many as fill the SMs, of 16 blocks at least, as far as there is room for parts (61 tokens of four sequences at up to 34k, 12 heads over 4: in
    // one piece each 643 us, so 90).
    const long long pairs = tiles * c.n_kv;
    if (pairs > 0x7fffffffll) return refuse(MAYA_ERR_LIMIT);
    long long most = (b.max_len + kKvBlock - 1) / kKvBlock;
    if (A.window > 0 && most > (A.window + 255ll / A.group) / kKvBlock + 2) most = (A.window + 255ll / A.group) / kKvBlock + 2;
    long long cuts = sm_count() / pairs;
    if (cuts > most / 16) cuts = most / 16;
    if (cuts > kPartRows / (256 * pairs)) cuts = kPartRows / (256 * pairs);
    if (cuts < 1) cuts = 1;
    A.tiles = (int) tiles;
    A.fixed = cuts > 1 ? (unsigned) cuts : 0u;
    static SmemLimit limit;
    if (!limit.raise((const void*) prompt_kernel<D>, PCfg<D>::smem)) return note_launch("kv prompt attention smem attribute");
    launch_dependent(prompt_kernel<D>, dim3((unsigned) pairs, 1, (unsigned) cuts), dim3(kPThreads), PCfg<D>::smem, s, kv_view(c), batch_view(b), A);
    const int st = note_launch("attn_q8 prompt");
    if (st != MAYA_OK || cuts == 1) return st;
    return attn_join(c, b, A, 256, s);
}

}  // namespace

// Attention of a prompt's rows on tcgen05; kNotTaken: not this kernel's call, nothing launched.
int attn_prompt(const maya_kv_cache& c, const maya_attn_batch& b, const AttnView& A, bool bf16, cudaStream_t s) {
    if (!bf16 || A.sel != nullptr || (c.head_dim != 64 && c.head_dim != 128)) return kNotTaken;
    if ((long long) b.max_new * A.group < 128) return kNotTaken;
    return c.head_dim == 64 ? launch_prompt<64>(c, b, A, s) : launch_prompt<128>(c, b, A, s);
}

}  // namespace maya
