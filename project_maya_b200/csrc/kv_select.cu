// kv_select.cu - the blocks each query reads: a cheap score for every block of its sequence, and the n_sel highest.
//
// score(block) = max over the group's heads g of f32(q8_g . k_sum) * s_g * k_scale: the query's dot with the block's mean key (times 64), from 8-bit
// queries and the exact sums of the keys' codes.  Whole-number dots do not depend on the order of their sums, so the lists are
// the same bits whatever the split.  k_sum's 16 bits enter the int8 tensor cores (mma.sync m16n8k32) as two digits, its upper byte signed
// and its lower byte not: dot = 256 hi + lo.  A block's sums are 2 * head_dim bytes beside its 128 * head_dim bytes of codes, so
// a decode step's selection reads a 64th of the cache; what bounds it there is latency (scores, then the search, one behind the other).
//
// A thread block scores a few tokens of one sequence for one key/value head (their heads fill 16-row tiles; the sums' fragments are loaded
// once for all) and keeps the scores in shared memory as ordered 32-bit keys; the n_sel-th largest key is found bit by bit, the list
// is written in ascending order.  With few tokens the blocks of a sequence are shared out over a cluster, whose first member gathers the keys.
#include <cooperative_groups.h>

#include "maya_kv.cuh"

namespace maya {
namespace {

namespace cg = cooperative_groups;

constexpr int kSelThreads = 256, kSelWarps = kSelThreads / 32;
constexpr uint32_t kForced = 0xffffffffu;

struct SelView {
    const void* q;
    int64_t ld_q;
    int n_q, group, rows_per_token;              // rows_per_token: the group padded to 1, 2, 4, 8 or a multiple of 16
    int tokens, tiles;                           // of a thread block; 16-row tiles they fill
    int token_tiles;                             // thread blocks (clusters) of a sequence
    int n_first, n_last, n_sel, ld_keys, wide_q;
    int* sel;
};

__device__ __forceinline__ void mma_s8(int (&d)[4], const uint4 a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_s8u8(int (&d)[4], const uint4 a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// Floats as unsigned numbers of the same order, above 0 (0: no block) and below kForced; NaN below all, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float s) {
    if (!(s == s)) return 1u;
    const uint32_t u = __float_as_uint(s + 0.0f);
    const uint32_t k = u & 0x80000000u ? ~u : u | 0x80000000u;
    return max(1u, min(k, kForced - 1));
}

template<int D, bool BF16>
__global__ void __launch_bounds__(kSelThreads) select_kernel(const KvView C, const BatchView B, const SelView S) {
    constexpr int V = D / 32, ST = D / 32;
    extern __shared__ __align__(16) uint8_t smem[];
    uint32_t* keys = (uint32_t*) smem;                                    // [tokens][ld_keys]
    uint8_t* frag = smem + (size_t) S.tokens * S.ld_keys * 4;             // [tiles][ST][32 lanes][16]
    float* qs = (float*) (frag + (size_t) S.tiles * ST * 512);            // [tiles * 16]; < 0: no row
    __shared__ int counts[kSelWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int) cluster.block_rank(), parts = (int) cluster.num_blocks();
    grid_launch_dependents();
    grid_dependency_wait();

    const int item = blockIdx.x / parts, h = blockIdx.y;
    const int si = item / S.token_tiles, i0 = (item % S.token_tiles) * S.tokens;
    const Seq s = seq_of(B, si);
    const int n_tok = min(S.tokens, s.n_new - i0);                        // the same in the whole cluster
    if (n_tok <= 0) return;
    const int first = s.len - s.n_new + i0;                               // position of the first of them
    const int nb = first + n_tok - 1 < 0 ? 0 : min((first + n_tok - 1) / kKvBlock + 1, S.ld_keys);

    // ---- queries as whole numbers, one row a warp, laid out as fragments
    for (int r = warp; r < S.tiles * 16; r += kSelWarps) {
        const int i = r / S.rows_per_token, hg = r % S.rows_per_token;
        const bool real = i < n_tok && hg < S.group;
        float x[V];
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = 0.0f;
        if (real) ld_acts<BF16, V>(S.q, (size_t) (s.row + i0 + i) * S.ld_q + (size_t) (h * S.group + hg) * D + lane * V, S.wide_q, x);
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) amax = fmaxf(amax, fabsf(x[e]));
        amax = warp_max(amax);
        const float scale = __fmul_rn(amax, kInv127);
        if (lane == 0) qs[r] = real ? scale : -1.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int d = lane * V + e;
            const float y = scale > 0.0f ? rintf(__fdiv_rn(x[e], scale)) : 0.0f;
            const int c = y == y ? (int) fmaxf(-127.0f, fminf(127.0f, y)) : 0;
            frag[(((r >> 4) * ST + (d >> 5)) * 32 + (r & 7) * 4 + ((d & 31) >> 3)) * 16 + (((d >> 2) & 1) * 2 + ((r >> 3) & 1)) * 4 + (d & 3)] = (uint8_t) (int8_t) c;
        }
    }
    if (parts > 1) cluster.sync();                                        // every member runs before one writes to another's memory
    else __syncthreads();

    // ---- scores: eight blocks a warp, their sums straight from memory as fragments
    uint32_t* into = parts > 1 ? cluster.map_shared_rank(keys, 0) : keys;
    for (int b8 = (rank * kSelWarps + warp) * 8; b8 < nb; b8 += parts * kSelWarps * 8) {
        const int b = b8 + g, phys = b < nb ? block_of(C, si, b) : -1;
        uint32_t hi[ST][2], lo[ST][2];
        const uint4* src = (const uint4*) (C.k_sum + ((size_t) max(phys, 0) * C.n_kv + h) * D) + t;
#pragma unroll
        for (int st = 0; st < ST; ++st) {
            const uint4 w = phys >= 0 ? src[st * 4] : make_uint4(0u, 0u, 0u, 0u);
            lo[st][0] = __byte_perm(w.x, w.y, 0x6420); hi[st][0] = __byte_perm(w.x, w.y, 0x7531);
            lo[st][1] = __byte_perm(w.z, w.w, 0x6420); hi[st][1] = __byte_perm(w.z, w.w, 0x7531);
        }
        const float ks = phys >= 0 ? C.k_scale[(size_t) phys * C.n_kv + h] : 0.0f;
        float kc[2];                                                      // of columns 2 t, 2 t + 1
        kc[0] = __shfl_sync(0xffffffffu, ks, 8 * t);
        kc[1] = __shfl_sync(0xffffffffu, ks, 8 * t + 4);
        for (int tile = 0; tile < S.tiles; ++tile) {
            int ch[4] = {0, 0, 0, 0}, cl[4] = {0, 0, 0, 0};
#pragma unroll
            for (int st = 0; st < ST; ++st) {
                const uint4 a = *(const uint4*) (frag + ((tile * ST + st) * 32 + lane) * 16);
                mma_s8(ch, a, hi[st][0], hi[st][1]);
                mma_s8u8(cl, a, lo[st][0], lo[st][1]);
            }
            float sc[4];
            const float q0 = qs[tile * 16 + g], q1 = qs[tile * 16 + g + 8];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float qr = e < 2 ? q0 : q1;
                sc[e] = qr < 0.0f ? -INFINITY : __fmul_rn(__fmul_rn((float) (ch[e] * 256 + cl[e]), qr), kc[e & 1]);
            }
            const int span = min(S.rows_per_token, 16);                   // rows of the tile that are one token's
            if (span == 16) { sc[0] = fmaxf(sc[0], sc[2]); sc[1] = fmaxf(sc[1], sc[3]); }
            for (int x = 1; x < min(span, 8); x *= 2)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[e] = fmaxf(sc[e], __shfl_xor_sync(0xffffffffu, sc[e], 4 * x));
            if (g % min(span, 8) == 0)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (span == 16 && e >= 2) break;
                    const int row = tile * 16 + g + (e >= 2 ? 8 : 0), i = row / S.rows_per_token, bb = b8 + 2 * t + (e & 1);
                    if (i >= n_tok || bb >= nb) continue;
                    const int own = first + i < 0 ? -1 : (first + i) / kKvBlock;
                    uint32_t k = bb > own ? 0u : bb < S.n_first || bb > own - S.n_last ? kForced : key_of(sc[e]);
                    uint32_t* p = into + (size_t) i * S.ld_keys + bb;
                    if (row % S.rows_per_token >= 16) k = max(k, *p);     // a token of more than 16 heads: the same lane's earlier tile
                    *p = k;
                }
        }
    }
    if (parts > 1) {
        cluster.sync();
        if (rank != 0) return;
    } else {
        __syncthreads();
    }

    // ---- the lists: a warp a token, or the whole block for one
    const bool together = n_tok == 1;
    for (int i = together ? 0 : warp; i < n_tok; i += together ? 1 : kSelWarps) {
        const uint32_t* k = keys + (size_t) i * S.ld_keys;
        const int step = together ? kSelThreads : 32, at = together ? tid : lane;
        auto count = [&](uint32_t least) {                                // keys of the token that are at least `least`
            int n = 0;
            for (int b = at; b < nb; b += step) n += k[b] >= least;
            n = __reduce_add_sync(0xffffffffu, n);
            if (together) {
                __syncthreads();
                if (lane == 0) counts[warp] = n;
                __syncthreads();
                n = 0;
#pragma unroll
                for (int w = 0; w < kSelWarps; ++w) n += counts[w];
            }
            return n;
        };
        uint32_t least = 1;
        int above = 0;                                                    // keys above `least`
        if (count(1) > S.n_sel) {
            least = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const uint32_t c = least | (1u << bit);
                const int n = count(c);
                if (n >= S.n_sel) least = c;
                else above = n;
            }
        } else {
            above = S.n_sel;                                              // all of them; nothing is cut among equals
        }
        if (together && warp != 0) return;
        int* out = S.sel + ((size_t) (s.row + i0 + i) * C.n_kv + h) * S.n_sel;
        int equal = above == S.n_sel ? S.n_sel : S.n_sel - above, done = 0;   // how many of the keys equal to `least` are taken: the lowest blocks
        for (int b0 = 0; b0 < nb; b0 += 32) {
            const uint32_t key = b0 + lane < nb ? k[b0 + lane] : 0u;
            const unsigned same = __ballot_sync(0xffffffffu, key == least), below = (1u << lane) - 1;
            const bool take = key > least || (key == least && __popc(same & below) < equal);
            const unsigned taken = __ballot_sync(0xffffffffu, take);
            if (take) out[done + __popc(taken & below)] = b0 + lane;
            done += __popc(taken);
            equal -= min(equal, __popc(same));
        }
        for (int e = done + lane; e < S.n_sel; e += 32) out[e] = -1;
    }
}

template<int D, bool BF16>
int launch_select(const maya_kv_cache& c, const maya_attn_batch& b, const maya_select_args& a, cudaStream_t s) {
    SelView S{};
    S.q = a.q; S.ld_q = a.ld_q; S.n_q = a.n_q; S.group = a.n_q / c.n_kv; S.sel = a.sel;
    S.n_first = a.n_first; S.n_last = a.n_last; S.n_sel = a.n_sel;
    S.wide_q = rows_wide(a.q, a.ld_q, BF16 ? 2 : 4);
    S.rows_per_token = 1;
    while (S.rows_per_token < S.group && S.rows_per_token < 16) S.rows_per_token *= 2;
    if (S.group > 16) S.rows_per_token = (S.group + 15) / 16 * 16;
    S.ld_keys = (b.max_len + kKvBlock - 1) / kKvBlock;
    if (S.ld_keys < 1) S.ld_keys = 1;
    // Tokens a thread block: four tiles of rows, as far as the tokens reach and their keys fit shared memory.
    const size_t row_bytes_ = (size_t) (D / 32) * 512 / 16 + 4;
    int tokens = S.rows_per_token >= 64 ? 1 : 64 / S.rows_per_token;
    if (tokens > b.max_new) tokens = b.max_new;
    auto need = [&](int n) {
        const int tiles = (n * S.rows_per_token + 15) / 16;
        return (size_t) n * S.ld_keys * 4 + (size_t) tiles * 16 * row_bytes_;
    };
    while (tokens > 1 && need(tokens) > kSmemMost) --tokens;
    if (need(tokens) > kSmemMost) return refuse(MAYA_ERR_LIMIT);
    S.ld_keys = (S.ld_keys + 3) / 4 * 4;                 // the fragments behind the keys start on 16 bytes
    while (tokens > 1 && need(tokens) > kSmemMost) --tokens;
    S.tokens = tokens;
    S.tiles = (tokens * S.rows_per_token + 15) / 16;
    S.token_tiles = (b.max_new + tokens - 1) / tokens;
    const size_t smem = need(tokens);
    // A cluster a (sequence, head) where they are fewer than half the SMs, of as many thread blocks as have 64 cache blocks each.
    const long long items = (long long) b.n_seq * S.token_tiles;
    int parts = 1;
    while (parts < 8 && items * c.n_kv * parts * 2 <= sm_count() && S.ld_keys >= parts * 128) parts *= 2;
    if (items * parts > 0x7fffffffll) return refuse(MAYA_ERR_LIMIT);
    static SmemLimit limit;
    if (smem > kSmemNoLimit && !limit.raise((const void*) select_kernel<D, BF16>, kSmemMost + 4096)) return note_launch("block_select smem attribute");
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned) (items * parts), (unsigned) c.n_kv);
    cfg.blockDim = dim3(kSelThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim = {(unsigned) parts, 1, 1};
    cfg.attrs = at;
    cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, select_kernel<D, BF16>, kv_view(c), batch_view(b), S);
    return note_launch("block_select");
}

}  // namespace
}  // namespace maya

using namespace maya;

extern "C" int maya_block_select(const maya_kv_cache* c, const maya_attn_batch* b, const maya_select_args* a, void* stream) {
    int st = kv_check(c);
    if (st == MAYA_OK) st = batch_check(c, b);
    if (st == MAYA_OK && !a) st = MAYA_ERR_ARG;
    if (st != MAYA_OK) return refuse(st);
    if (b->n_tokens == 0) return MAYA_OK;
    if (!a->q || !a->sel || !c->k_sum || a->n_q <= 0 || a->n_q % c->n_kv != 0) return refuse(MAYA_ERR_ARG);
    if (a->ld_q < (int64_t) a->n_q * c->head_dim || a->n_first < 0 || a->n_last < 1) return refuse(MAYA_ERR_ARG);
    if (a->n_sel < 1 || a->n_first > a->n_sel || a->n_last > a->n_sel - a->n_first) return refuse(MAYA_ERR_ARG);
    if (a->n_sel > MAYA_MAX_SELECTED || b->max_len > MAYA_MAX_KV_BLOCKS * kKvBlock || c->n_kv > 65535) return refuse(MAYA_ERR_LIMIT);
    cudaStream_t s = as_stream(stream);
#define SELECT(D) a->is_bf16 ? launch_select<D, true>(*c, *b, *a, s) : launch_select<D, false>(*c, *b, *a, s)
    switch (c->head_dim) {
        case 64: return SELECT(64);
        case 128: return SELECT(128);
        case 192: return SELECT(192);
        default: return SELECT(256);
    }
#undef SELECT
}
