// kv_select.cu - the blocks each query reads: a cheap score for every block of its sequence, and the n_sel highest.
//
// score(block) = max over the group's heads g of f32(q8_g . k_sum) * s_g * k_scale: the query's dot with the block's mean key (times 64), from 8-bit
// queries and the exact sums of the keys' codes.  Whole-number dots do not depend on the order of their sums, so the lists are
// the same bits whatever the split.  k_sum's 16 bits enter the tensor cores (mma.sync m16n8k16, f16 into f32)
// as two digits, its upper byte signed and its lower byte not: dot = 256 hi + lo, whose sums stay below 2^24 and so are exact in f32.  (With
// m16n8k32 in 8 bits, which sm_100a has no direct form of: 1024 thread blocks of a prompt's selection ran 143 million warp instructions, 174 us.)  A block's sums are 2 * head_dim bytes beside its 128 * head_dim bytes of codes, so
// a decode step's selection reads a 64th of the cache; what bounds it there is latency (scores, then the search, one behind the other).
//
// A thread block scores a few tokens of one sequence for one key/value head (their heads fill 16-row tiles; the sums' fragments are loaded
// once for all) and keeps the scores in shared memory as ordered 32-bit keys; the n_sel-th largest key is found bit by bit, the list
// is written in ascending order.  With few tokens the blocks of a sequence are shared out over a cluster, whose first member gathers the keys.
#include <cooperative_groups.h>

#include <type_traits>

#include "maya_kv.cuh"

namespace maya {
namespace {

namespace cg = cooperative_groups;

constexpr int kSelThreads = 256, kSelWarps = kSelThreads / 32;
constexpr int kFrag = 32 * 16 + 16;                     // bytes of a 16 x 16 fragment, and what moves the next one's banks on

struct SelView {
    const void* q;
    int64_t ld_q;
    int n_q, group;
    int span_log2, tiles_per_token;              // rows of a tile that are one token's: 1 .. 16; tiles of a token of more than 16 heads, else 1
    int tokens, tiles, room;                     // of a thread block; 16-row tiles they fill; tokens those have room for
    int token_tiles;                             // thread blocks (clusters) of a sequence
    int n_first, n_last, n_sel, ld_keys, wide_q;
    int* sel;
};

__device__ __forceinline__ void mma_half(float (&d)[4], const uint4 a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// The two digits of two 16-bit sums as f16, exactly: sum = 256 hi + lo, hi the upper byte (signed), lo the lower one (0 .. 255).
__device__ __forceinline__ void digits(uint32_t w, uint32_t& hi, uint32_t& lo) {
    const uint32_t l = (w & 0x00ff00ffu) | 0x64006400u, h = ((w >> 8 & 0x00ff00ffu) ^ 0x00800080u) | 0x64006400u;     // 1024 + byte
    const __half2 lb = __halves2half2(__ushort_as_half(0x6400), __ushort_as_half(0x6400)), hb = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const __half2 x = __hsub2(*(const __half2*) &l, lb), y = __hsub2(*(const __half2*) &h, hb);
    lo = *(const uint32_t*) &x;
    hi = *(const uint32_t*) &y;
}
// Floats as unsigned numbers of the same order, above 0 (no block); NaN as -infinity, -0 as 0.
__device__ __forceinline__ uint32_t key_of(float s) {
    const uint32_t u = __float_as_uint(fmaxf(s, -INFINITY) + 0.0f);
    return u ^ ((uint32_t) ((int) u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k ^ (k & 0x80000000u ? 0x80000000u : 0xffffffffu)); }

// The list of one token, whose own block is `own`, from its keys, by WARPS warps (1: any warp; else the whole thread block; `at`: the thread's place
// among them).  Between the forced blocks the largest number that `need` keys reach is sought between the smallest and the largest score, by turns
// where a straight line through the two counts puts it and in the middle; a number that exactly `need` keys reach ends the search.  A member holds its first keys in registers.  Then the keys above the number and the lowest blocks of those
// equal to it are written in ascending order, every warp its share of the blocks.
constexpr int kHeld = 8;
template<int WARPS>
__device__ __forceinline__ void list_of(int n_sel, int n_first, int n_last, const uint32_t* keys, int nb, int own, int* out, int at) {
    __shared__ uint2 counts[2][WARPS];
    constexpr int step = 32 * WARPS;
    const int lane = at & 31, warp = at >> 5;
    nb = min(nb, own + 1);
    const bool all = nb <= n_sel;                                       // (then every block is forced)
    const int lo_b = all ? 0 : n_first, hi_b = all ? 0 : nb - n_last; // the blocks in between
    auto key = [&](int b) { return b >= lo_b && b < hi_b ? keys[b] : 0u; };
    uint32_t held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = key(at + i * step);
    int round = 0;
    uint32_t lo = 0;                                                      // `need` keys reach it; the result: keys above lo are taken
    int equal = 0;                                                        // and so many of those equal to it, the lowest blocks first
    const int need = n_sel - n_first - n_last;
    if (!all) {
        uint32_t hi = 0;                                                  // fewer than `need` reach it
        uint32_t small = 0xffffffffu;
#pragma unroll
        for (int i = 0; i < kHeld; ++i) { hi = max(hi, held[i]); small = min(small, held[i] - 1u); }      // (0 - 1 is the largest)
        for (int b = at + kHeld * step; b < nb; b += step) { const uint32_t k = key(b); hi = max(hi, k); small = min(small, k - 1u); }
        hi = __reduce_max_sync(0xffffffffu, hi);
        small = __reduce_min_sync(0xffffffffu, small);
        if constexpr (WARPS > 1) {
            uint2* c = counts[round++ & 1];
            if (lane == 0) c[warp] = make_uint2(hi, small);
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WARPS; ++w) { hi = max(hi, c[w].x); small = min(small, c[w].y); }
        }
        lo = need > 0 ? small + 1u : hi;
        hi += 1u;
        int n_lo = hi_b - lo_b, n_hi = 0;                                 // keys that reach lo, hi
        for (int turn = 0; n_lo != need && hi - lo > 1u && need > 0; ++turn) {
            uint32_t c = lo + ((hi - lo) >> 1);
            if (turn < 12 && (turn & 3) != 3) {                           // by the scores themselves; every fourth turn, and from some point on, halves the keys
                const float f = value_of(lo), w = value_of(hi) - f;
                const float part = turn & 1 ? 0.5f : __fdividef((float) (n_lo - need) + 0.5f, (float) (n_lo - n_hi));
                c = max(lo + 1u, min(key_of(fmaf(w, part, f)), hi - 1u));
            }
            uint32_t n = 0;
#pragma unroll
            for (int i = 0; i < kHeld; ++i) n += held[i] >= c ? 1u : 0u;
            for (int b = at + kHeld * step; b < nb; b += step) n += key(b) >= c ? 1u : 0u;
            n = __reduce_add_sync(0xffffffffu, n);
            if constexpr (WARPS > 1) {
                uint2* k = counts[round++ & 1];
                if (lane == 0) k[warp].x = n;
                __syncthreads();
                n = 0;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) n += k[w].x;
            }
            if ((int) n >= need) { lo = c; n_lo = (int) n; }
            else { hi = c; n_hi = (int) n; }
        }
        if (need == 0) lo = 0xffffffffu;                                  // none in between
        else if (n_lo == need) lo -= 1u;                                  // exactly these
        else equal = need - n_hi;
    }
    const int share = (nb + step - 1) / step * 32, from = warp * share, to = min(nb, from + share);
    auto forced = [&](int b) { return all || b < lo_b || b >= hi_b; };
    int done = 0;
    if constexpr (WARPS > 1) {                                            // what the warps in front of this one write
        uint32_t more = 0, same = 0;
        for (int b = from + lane; b < to; b += 32) {
            const uint32_t k = key(b);
            more += forced(b) || k > lo;
            same += !forced(b) && k == lo;
        }
        more = __reduce_add_sync(0xffffffffu, more);
        same = __reduce_add_sync(0xffffffffu, same);
        uint2* c = counts[round & 1];
        if (lane == 0) c[warp] = make_uint2(more, same);
        __syncthreads();
        for (int w = 0; w < warp; ++w) {
            const int e = min((int) c[w].y, equal);
            done += (int) c[w].x + e;
            equal -= e;
        }
    }
    for (int b0 = from; b0 < to; b0 += 32) {
        const int b = b0 + lane;
        const uint32_t k = b < to ? key(b) : 0u;
        const bool must = b < to && (forced(b) || k > lo);
        const unsigned same = __ballot_sync(0xffffffffu, b < to && !must && k == lo), below = (1u << lane) - 1;
        const bool take = must || ((same >> lane & 1u) && __popc(same & below) < equal);
        const unsigned taken = __ballot_sync(0xffffffffu, take);
        if (take) out[done + __popc(taken & below)] = b;
        done += __popc(taken);
        equal -= min(equal, __popc(same));
    }
    if (warp == WARPS - 1)
        for (int e = done + lane; e < n_sel; e += 32) out[e] = -1;
}

template<int D, bool BF16>
__global__ void __launch_bounds__(kSelThreads) select_kernel(const KvView C, const BatchView B, const SelView S) {
    constexpr int V = D / 32, ST = D / 16;
    extern __shared__ __align__(16) uint8_t smem[];
    uint32_t* keys = (uint32_t*) smem;                                    // [tokens the tiles have room for][ld_keys]
    uint8_t* frag = smem + (size_t) S.room * S.ld_keys * 4;             // [tiles][ST][kFrag]: f16
    float* qs = (float*) (frag + (size_t) S.tiles * ST * kFrag);            // [tiles * 16]; NaN: no row
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
    const int nb = min(((first + n_tok - 1) >> 6) + 1, S.ld_keys);        // (none or less: all of them stand before the sequence)

    // row r of the tiles: which of the block's tokens, and which head of its group
    auto token_of = [&](int r) { return S.tiles_per_token > 1 ? (r >> 4) / S.tiles_per_token : r >> S.span_log2; };
    auto head_of = [&](int r) { return S.tiles_per_token > 1 ? r - token_of(r) * S.tiles_per_token * 16 : r & ((1 << S.span_log2) - 1); };

    // the first cache blocks' sums are asked for before anything else
    const int stride = parts * kSelWarps * 8;
    int b8 = (rank * kSelWarps + warp) * 8;
    uint4 raw[D / 32];
    float raw_ks;
    auto ask = [&](int at, uint4 (&w)[D / 32], float& ks) {
        const int phys = at + g < nb ? block_of(C, si, at + g) : -1;
        const size_t bh = (size_t) max(phys, 0) * C.n_kv + h;
        const uint4* src = (const uint4*) (C.k_sum + bh * D) + t;
#pragma unroll
        for (int i = 0; i < D / 32; ++i) w[i] = phys >= 0 ? src[i * 4] : make_uint4(0u, 0u, 0u, 0u);
        ks = phys >= 0 ? C.k_scale[bh] : 0.0f;
    };
    ask(b8, raw, raw_ks);

    // ---- queries as whole numbers, laid out as fragments: eight lanes a row, four rows a warp at a time
    for (int r0 = warp * 4; r0 < S.tiles * 16; r0 += kSelWarps * 4) {
        constexpr int E = D / 8;                                          // values of a lane: E * (lane % 8) ..
        const int r = r0 + (lane >> 3), i = token_of(r), hg = head_of(r), d0 = (lane & 7) * E;
        const bool real = i < n_tok && hg < S.group;
        float x[E];
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = 0.0f;
        if (real) ld_acts<BF16, E>(S.q, (size_t) (s.row + i0 + i) * S.ld_q + (size_t) (h * S.group + hg) * D + d0, S.wide_q, x);
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) amax = fmaxf(amax, fabsf(x[e]));
#pragma unroll
        for (int o = 1; o < 8; o *= 2) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
        const float scale = __fmul_rn(amax, kInv127);
        if ((lane & 7) == 0) qs[r] = real ? scale : __uint_as_float(0x7fc00000u);      // no row: NaN, which no maximum takes
        // round(x / scale) as the exact quotient rounds: a product with the reciprocal, unless one comes near the middle of two numbers
        const float inv = __fdividef(1.0f, scale);
        float c[E], off = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float y = x[e] * inv;
            c[e] = (y + 12582912.0f) - 12582912.0f;
            off = fmaxf(off, fabsf(y - c[e]));
        }
        if (!(off < 0.4998f) || !(scale > 1e-30f && scale < 1e30f)) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float y = scale > 0.0f ? __fdiv_rn(x[e], scale) : 0.0f;
                c[e] = y == y ? fmaxf(-127.0f, fminf(127.0f, rintf(y))) : 0.0f;
            }
        }
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const int d = d0 + e, st = (d >> 5) * 2 + ((d >> 2) & 1);
            *(__half2*) (frag + ((r >> 4) * ST + st) * kFrag + (((r & 7) * 4 + ((d & 31) >> 3)) * 4 + ((d >> 1) & 1) * 2 + ((r >> 3) & 1)) * 4) = __floats2half2_rn(c[e], c[e + 1]);
        }
    }
    if (parts > 1) cluster.sync();                                        // every member runs before one writes to another's memory
    else __syncthreads();

    // ---- scores: eight blocks a warp, their sums straight from memory as fragments
    uint32_t* into = parts > 1 ? cluster.map_shared_rank(keys, 0) : keys;
    auto scores = [&](auto span_) {
        constexpr int span = decltype(span_)::value;
        const bool g0 = g & 1, g1 = g & 2, g2 = g & 4;
        for (; b8 < nb; b8 += stride) {
            uint32_t hi[ST][2], lo[ST][2];
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                digits(raw[i].x, hi[2 * i][0], lo[2 * i][0]); digits(raw[i].y, hi[2 * i][1], lo[2 * i][1]);
                digits(raw[i].z, hi[2 * i + 1][0], lo[2 * i + 1][0]); digits(raw[i].w, hi[2 * i + 1][1], lo[2 * i + 1][1]);
            }
            const float ks = raw_ks;
            if (b8 + stride < nb) ask(b8 + stride, raw, raw_ks);
            float kc[2];                                                  // of columns 2 t, 2 t + 1
            kc[0] = __shfl_sync(0xffffffffu, ks, 8 * t);
            kc[1] = __shfl_sync(0xffffffffu, ks, 8 * t + 4);
            uint32_t* row = into + b8 + 2 * t;                            // of the tile's first token
            int part = 0;                                                 // the tile among its token's
#pragma unroll 2
            for (int tile = 0; tile < S.tiles; ++tile) {
                float ch[4] = {0.0f, 0.0f, 0.0f, 0.0f}, cl[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int st = 0; st < ST; ++st) {
                    const uint4 a = *(const uint4*) (frag + (tile * ST + st) * kFrag + lane * 16);
                    mma_half(ch, a, hi[st][0], hi[st][1]);
                    mma_half(cl, a, lo[st][0], lo[st][1]);
                }
                float sc[4];
                const float q0 = qs[tile * 16 + g], q1 = qs[tile * 16 + g + 8];
#pragma unroll
                for (int e = 0; e < 4; ++e)                               // 256 hi + lo is rounded once, as the whole number would be
                    sc[e] = __fmul_rn(__fmul_rn(fmaf(ch[e], 256.0f, cl[e]), e < 2 ? q0 : q1), kc[e & 1]);
                // the maximum over a token's rows: values are handed over so that every lane is left with what it writes
                auto meet = [&](float keep, float give, int x) { return fmaxf(keep, __shfl_xor_sync(0xffffffffu, give, x)); };
                if constexpr (span == 16) {
                    sc[0] = fmaxf(sc[0], sc[2]); sc[1] = fmaxf(sc[1], sc[3]);
                    float v = meet(g0 ? sc[1] : sc[0], g0 ? sc[0] : sc[1], 4);
                    v = meet(v, v, 8);
                    v = meet(v, v, 16);
                    if (!g1 && !g2) {
                        uint32_t k = key_of(v);
                        if (part > 0) k = max(k, row[g0]);                // a token of more than 16 heads: the same lane's tile before
                        row[g0] = k;
                    }
                    if (++part == S.tiles_per_token) { part = 0; row += S.ld_keys; }
                } else if constexpr (span >= 4) {
                    const float v0 = meet(g0 ? sc[2] : sc[0], g0 ? sc[0] : sc[2], 4), v1 = meet(g0 ? sc[3] : sc[1], g0 ? sc[1] : sc[3], 4);
                    float v = meet(g1 ? v1 : v0, g1 ? v0 : v1, 8);
                    if constexpr (span == 8) v = meet(v, v, 16);
                    if (span == 4 || !g2) row[(span == 8 ? g0 : 2 * g0 + g2) * S.ld_keys + g1] = key_of(v);
                    row += 16 / span * S.ld_keys;
                } else if constexpr (span == 2) {
                    const float v0 = meet(g0 ? sc[2] : sc[0], g0 ? sc[0] : sc[2], 4), v1 = meet(g0 ? sc[3] : sc[1], g0 ? sc[1] : sc[3], 4);
                    *(uint2*) (row + (4 * g0 + (g >> 1)) * S.ld_keys) = make_uint2(key_of(v0), key_of(v1));
                    row += 8 * S.ld_keys;
                } else {
                    *(uint2*) (row + g * S.ld_keys) = make_uint2(key_of(sc[0]), key_of(sc[1]));
                    *(uint2*) (row + (g + 8) * S.ld_keys) = make_uint2(key_of(sc[2]), key_of(sc[3]));
                    row += 16 * S.ld_keys;
                }
            }
        }
    };
    switch (S.span_log2) {
        case 0: scores(std::integral_constant<int, 1>()); break;
        case 1: scores(std::integral_constant<int, 2>()); break;
        case 2: scores(std::integral_constant<int, 4>()); break;
        case 3: scores(std::integral_constant<int, 8>()); break;
        default: scores(std::integral_constant<int, 16>()); break;
    }
    if (parts > 1) {
        cluster.sync();
        if (rank != 0) return;
    } else {
        __syncthreads();
    }

    // ---- the lists: a warp a token, or the whole block for one
    if (n_tok == 1) list_of<kSelWarps>(S.n_sel, S.n_first, S.n_last, keys, nb, first >> 6, S.sel + ((size_t) (s.row + i0) * C.n_kv + h) * S.n_sel, tid);
    else
        for (int i = warp; i < n_tok; i += kSelWarps)
            list_of<1>(S.n_sel, S.n_first, S.n_last, keys + (size_t) i * S.ld_keys, nb, (first + i) >> 6, S.sel + ((size_t) (s.row + i0 + i) * C.n_kv + h) * S.n_sel, lane);
}

template<int D, bool BF16>
int launch_select(const maya_kv_cache& c, const maya_attn_batch& b, const maya_select_args& a, cudaStream_t s) {
    SelView S{};
    S.q = a.q; S.ld_q = a.ld_q; S.n_q = a.n_q; S.group = a.n_q / c.n_kv; S.sel = a.sel;
    S.n_first = a.n_first; S.n_last = a.n_last; S.n_sel = a.n_sel;
    S.wide_q = rows_wide(a.q, a.ld_q, BF16 ? 2 : 4);
    while ((1 << S.span_log2) < S.group && S.span_log2 < 4) ++S.span_log2;
    S.tiles_per_token = S.group > 16 ? (S.group + 15) / 16 : 1;
    const int rows_per_token = S.group > 16 ? S.tiles_per_token * 16 : 1 << S.span_log2;
    S.ld_keys = ((b.max_len + kKvBlock - 1) / kKvBlock + 7) / 8 * 8;      // whole groups of eight blocks
    if (S.ld_keys < 8) S.ld_keys = 8;
    // Tokens a thread block: eight tiles of rows, as far as the tokens reach and their keys fit shared memory.
    auto tiles_of = [&](int n) { return (n * rows_per_token + 15) / 16; };
    auto room_of = [&](int n) { return S.tiles_per_token > 1 ? n : tiles_of(n) << (4 - S.span_log2); };
    auto need = [&](int n) { return (size_t) room_of(n) * S.ld_keys * 4 + (size_t) tiles_of(n) * (D / 16 * kFrag + 64); };
    int tokens = rows_per_token >= 128 ? 1 : 128 / rows_per_token;
    if (tokens > b.max_new) tokens = b.max_new;
    while (tokens > 1 && need(tokens) > kSmemMost) tokens = (tokens + 1) / 2;
    if (need(tokens) > kSmemMost) return refuse(MAYA_ERR_LIMIT);
    S.tokens = tokens;
    S.tiles = tiles_of(tokens);
    S.room = room_of(tokens);
    S.token_tiles = (b.max_new + tokens - 1) / tokens;
    const size_t smem = need(tokens);
    // A sequence's blocks are shared out over a cluster while all thread blocks are on the chip at once (two an SM) and each of their
    // warps has eight cache blocks to score.
    const long long items = (long long) b.n_seq * S.token_tiles;
    int parts = 1;
    while (parts < 8 && items * c.n_kv * parts * 2 <= (long long) sm_count() * 2 && S.ld_keys >= parts * 2 * kSelWarps * 8) parts *= 2;
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
