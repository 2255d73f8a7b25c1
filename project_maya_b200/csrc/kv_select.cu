// kv_select.cu - the blocks each query reads: a cheap score for every block of its sequence, and the n_sel highest.
//
// score(block) = max over the group's heads g of f32(q8_g . k_sum) * s_g * k_scale: the query's dot with the block's mean key (times 64), from 8-bit
// queries and the exact sums of the keys' codes.  Whole-number dots do not depend on the order of their sums, so the lists are
// the same bits whatever the split.  k_sum's 16 bits enter the tensor cores (mma.sync m16n8k16, f16 into f32)
// as two digits, its upper byte signed and its lower byte not: dot = 256 hi + lo, whose sums stay below 2^24 and so are exact in f32.  (m16n8k32
// in 8 bits in its place: 174 us against 160 on a prompt's selection.)
// A block's sums are 2 * head_dim bytes beside its 128 * head_dim bytes of codes, so a decode step's selection reads a 64th of the cache; what bounds it
// there is latency (scores, then the search, one behind the other).
//
// A thread block scores a few tokens of one sequence for one key/value head (their heads fill tiles of eight columns; the sums' fragments are
// loaded once for all) and keeps the scores in shared memory as ordered 32-bit keys; the n_sel-th largest key is sought between the scores, the
// list is written in ascending order.  With few tokens the blocks of a sequence are shared out over a cluster, whose first member gathers the keys.
// Measured, one B200: 16 tokens at 4k..64k, 64 heads over 8, 15.8 us; a chunk of 4096 at 16k, 32 heads over 4, 115 us.
#include <cooperative_groups.h>

#include <type_traits>

#include "maya_kv.cuh"

namespace maya {
namespace {

namespace cg = cooperative_groups;

constexpr int kSelThreads = 256, kSelWarps = kSelThreads / 32;
constexpr uint32_t kForced = 0xffffffffu;         // key of a block that is always taken
constexpr int kFrag = 32 * 16 + 16;                     // bytes of the fragments of eight heads and 32 values, and what moves the next ones' banks on

struct SelView {
    const void* q;
    int64_t ld_q;
    int n_q, group;
    int span_log2, tiles_per_token;              // heads of a tile of eight that are one token's: 1 .. 8; tiles of a token of more than 8 heads, else 1
    int tokens, tiles, room;                     // of a thread block; tiles of eight heads they fill; tokens those have room for
    int token_tiles;                             // thread blocks (clusters) of a sequence
    int n_first, n_last, n_sel, ld_keys, wide_q;
    int* sel;
};

__device__ __forceinline__ void mma_half(float (&d)[4], const uint4 a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
// among them).  The largest number that n_sel keys reach (a forced block's is above all) is sought between the smallest and the largest score,
// by turns where a straight line through the two counts puts it and in the middle; a number that exactly n_sel reach ends the search.  Every warp has
// a stretch of the blocks, a lane every 32nd of it, the first kHeld in registers.  Then the keys above the number and the lowest blocks of those equal to
// it are written in ascending order.
constexpr int kHeld = 8;
template<int WARPS>
__device__ __forceinline__ void list_of(int n_sel, int n_first, int n_last, const uint32_t* keys, int nb, int own, int* out, int at) {
    __shared__ uint2 counts[2][WARPS];
    const int lane = at & 31, warp = at >> 5;
    nb = max(0, min(nb, own + 1));
    const bool all = nb <= n_sel;                                         // (then every block is forced)
    const int lo_b = all ? nb : n_first, hi_b = all ? nb : nb - n_last;   // the blocks in between
    const int share = (nb + 32 * WARPS - 1) / (32 * WARPS) * 32, from = warp * share + lane, to = min(nb, warp * share + share);
    auto key = [&](int b) { return b >= to ? 0u : b < lo_b || b >= hi_b ? kForced : keys[b]; };
    uint32_t held[kHeld];
#pragma unroll
    for (int i = 0; i < kHeld; ++i) held[i] = key(from + 32 * i);
    int round = 0;
    uint32_t lo = 0;                                                      // the result: keys above lo are taken
    int equal = 0;                                                        // and so many of those equal to it, the lowest blocks first
    if (!all) {
        uint32_t hi = 1u, small = 0xffffffffu;                            // over the blocks in between
        auto see = [&](uint32_t k) { hi = max(hi, k + 1u); small = min(small, k - 1u); };      // (forced: 0, so no maximum; none: -1, so no minimum)
#pragma unroll
        for (int i = 0; i < kHeld; ++i) see(held[i]);
        for (int b = from + 32 * kHeld; b < to; b += 32) see(key(b));
        hi = __reduce_max_sync(0xffffffffu, hi);
        small = __reduce_min_sync(0xffffffffu, small);
        if constexpr (WARPS > 1) {
            uint2* c = counts[round++ & 1];
            if (lane == 0) c[warp] = make_uint2(hi, small);
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WARPS; ++w) { hi = max(hi, c[w].x); small = min(small, c[w].y); }
        }
        lo = small + 1u;                                                  // every block reaches it; hi: the forced ones alone
        int n_lo = nb, n_hi = n_first + n_last;
        if (n_hi == n_sel) { lo = hi; n_lo = n_hi; }
        for (int turn = 0; n_lo != n_sel && hi - lo > 1u; ++turn) {
            uint32_t c = lo + ((hi - lo) >> 1);
            if (turn < 12 && (turn & 3) != 3) {                           // by the scores themselves; every fourth turn, and from some point on, halves the keys
                const float f = value_of(lo), w = value_of(hi) - f;
                const float part = turn & 1 ? 0.5f : __fdividef((float) (n_lo - n_sel) + 0.5f, (float) (n_lo - n_hi));
                c = max(lo + 1u, min(key_of(fmaf(w, part, f)), hi - 1u));
            }
            uint32_t n = 0;
#pragma unroll
            for (int i = 0; i < kHeld; ++i) n += held[i] >= c ? 1u : 0u;
            for (int b = from + 32 * kHeld; b < to; b += 32) n += key(b) >= c ? 1u : 0u;
            n = __reduce_add_sync(0xffffffffu, n);
            if constexpr (WARPS > 1) {
                uint2* k = counts[round++ & 1];
                if (lane == 0) k[warp].x = n;
                __syncthreads();
                n = 0;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) n += k[w].x;
            }
            if ((int) n >= n_sel) { lo = c; n_lo = (int) n; }
            else { hi = c; n_hi = (int) n; }
        }
        if (n_lo == n_sel) lo -= 1u;                                      // exactly these
        else equal = n_sel - n_hi;
    }
    int done = 0;
    if constexpr (WARPS > 1) {                                            // what the warps in front of this one write
        uint32_t more = 0, same = 0;
        auto see = [&](uint32_t k) { more += k > lo ? 1u : 0u; same += k == lo ? 1u : 0u; };
#pragma unroll
        for (int i = 0; i < kHeld; ++i) see(held[i]);
        for (int b = from + 32 * kHeld; b < to; b += 32) see(key(b));
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
    const unsigned below = (1u << lane) - 1;
    auto emit = [&](int b, uint32_t k) {
        bool take = k > lo;
        if (equal > 0) {
            const unsigned same = __ballot_sync(0xffffffffu, k == lo);
            take = take || (k == lo && __popc(same & below) < equal);
            equal -= min(equal, __popc(same));
        }
        const unsigned taken = __ballot_sync(0xffffffffu, take);
        if (take) out[done + __popc(taken & below)] = b;
        done += __popc(taken);
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
        if (32 * i < share) emit(from + 32 * i, held[i]);
    for (int i = kHeld; 32 * i < share; ++i) emit(from + 32 * i, key(from + 32 * i));
    if (warp == WARPS - 1)
        for (int e = done + lane; e < n_sel; e += 32) out[e] = -1;
}

template<int D, bool BF16>
__global__ void __launch_bounds__(kSelThreads, D <= 128 ? 2 : 1) select_kernel(const KvView C, const BatchView B, const SelView S) {
    constexpr int ST = D / 16;
    extern __shared__ __align__(16) uint8_t smem[];
    uint32_t* keys = (uint32_t*) smem;                                    // [tokens the tiles have room for][ld_keys]
    uint8_t* frag = smem + (size_t) S.room * S.ld_keys * 4;             // [tiles][ST / 2][kFrag]: f16
    float* qs = (float*) (frag + (size_t) S.tiles * (ST / 2) * kFrag);            // [tiles * 8]; NaN: no row
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
    auto token_of = [&](int r) { return S.tiles_per_token > 1 ? (r >> 3) / S.tiles_per_token : r >> S.span_log2; };
    auto head_of = [&](int r) { return S.tiles_per_token > 1 ? r - token_of(r) * S.tiles_per_token * 8 : r & ((1 << S.span_log2) - 1); };

    // the first cache blocks' sums are asked for before anything else
    const int stride = parts * kSelWarps * 16;
    int b16 = (rank * kSelWarps + warp) * 16;
    uint4 raw[2][D / 32];                                                 // of blocks b16 + g and b16 + g + 8: values 32 i + 8 t ..
    float raw_ks[2];
    int phys[2];
    auto look_up = [&](int at) {
#pragma unroll
        for (int x = 0; x < 2; ++x) phys[x] = at + g + 8 * x < nb ? block_of(C, si, at + g + 8 * x) : -1;
    };
    auto ask = [&]() {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const size_t bh = (size_t) max(phys[x], 0) * C.n_kv + h;
            const uint4* src = (const uint4*) (C.k_sum + bh * D) + t;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) raw[x][i] = phys[x] >= 0 ? src[i * 4] : make_uint4(0u, 0u, 0u, 0u);
            raw_ks[x] = phys[x] >= 0 ? C.k_scale[bh] : -INFINITY;         // (a block that is not there: 0 times this, a NaN, below every score)
        }
    };
    look_up(b16);
    ask();

    // ---- queries as whole numbers, laid out as fragments: eight lanes a row, four rows a warp at a time
    for (int r0 = warp * 4; r0 < S.tiles * 8; r0 += kSelWarps * 4) {
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
        float c[E], off = 0.0f, sum = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float y = x[e] * inv;
            c[e] = (y + 12582912.0f) - 12582912.0f;
            off = fmaxf(off, fabsf(y - c[e]));
            sum += c[e];
        }
        if (!(off < 0.4998f) || sum != sum || !(scale > 1e-30f && scale < 1e30f)) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float y = scale > 0.0f ? __fdiv_rn(x[e], scale) : 0.0f;
                c[e] = y == y ? fmaxf(-127.0f, fminf(127.0f, rintf(y))) : 0.0f;
            }
        }
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const int d = d0 + e, st = (d >> 5) * 2 + ((d >> 2) & 1);      // two steps of a 32 lie side by side: one 16-byte load a lane
            *(__half2*) (frag + ((r >> 3) * (ST / 2) + (st >> 1)) * kFrag + (((r & 7) * 4 + ((d & 31) >> 3)) * 4 + (st & 1) * 2 + ((d >> 1) & 1)) * 4) = __floats2half2_rn(c[e], c[e + 1]);
        }
    }
    if (parts > 1) cluster.sync();                                        // every member runs before one writes to another's memory
    else __syncthreads();

    // ---- scores: sixteen blocks a warp as rows, their sums straight from memory as fragments; eight heads as columns
    uint32_t* into = parts > 1 ? cluster.map_shared_rank(keys, 0) : keys;
    auto scores = [&](auto span_) {
        constexpr int span = decltype(span_)::value;
        const bool t0 = t & 1, t1 = t & 2;
        for (; b16 < nb; b16 += stride) {
            uint4 hi[ST], lo[ST];
#pragma unroll
            for (int i = 0; i < D / 32; ++i) {
                digits(raw[0][i].x, hi[2 * i].x, lo[2 * i].x); digits(raw[1][i].x, hi[2 * i].y, lo[2 * i].y);
                digits(raw[0][i].y, hi[2 * i].z, lo[2 * i].z); digits(raw[1][i].y, hi[2 * i].w, lo[2 * i].w);
                digits(raw[0][i].z, hi[2 * i + 1].x, lo[2 * i + 1].x); digits(raw[1][i].z, hi[2 * i + 1].y, lo[2 * i + 1].y);
                digits(raw[0][i].w, hi[2 * i + 1].z, lo[2 * i + 1].z); digits(raw[1][i].w, hi[2 * i + 1].w, lo[2 * i + 1].w);
            }
            const float ks0 = raw_ks[0], ks1 = raw_ks[1];
            uint32_t* row = into + b16 + g;                               // of the tile's first token
            look_up(b16 + stride);
            int part = 0;                                                 // the tile among its token's
            float m0 = -INFINITY, m1 = -INFINITY;                         // the maxima over a token's tiles so far
#pragma unroll 2
            for (int tile = 0; tile < S.tiles; ++tile) {
                float ch[4] = {0.0f, 0.0f, 0.0f, 0.0f}, cl[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int i = 0; i < ST / 2; ++i) {
                    const uint4 b = *(const uint4*) (frag + (tile * (ST / 2) + i) * kFrag + lane * 16);
                    mma_half(ch, hi[2 * i], b.x, b.y);
                    mma_half(cl, lo[2 * i], b.x, b.y);
                    mma_half(ch, hi[2 * i + 1], b.z, b.w);
                    mma_half(cl, lo[2 * i + 1], b.z, b.w);
                }
                const float2 q = *(const float2*) (qs + tile * 8 + 2 * t);
                // (256 hi + lo is rounded once, as the whole number would be; the key's scale is not negative, so it may be multiplied behind the maximum)
                const float s00 = __fmul_rn(fmaf(ch[0], 256.0f, cl[0]), q.x), s01 = __fmul_rn(fmaf(ch[1], 256.0f, cl[1]), q.y);
                const float s10 = __fmul_rn(fmaf(ch[2], 256.0f, cl[2]), q.x), s11 = __fmul_rn(fmaf(ch[3], 256.0f, cl[3]), q.y);
                // values are handed over so that every lane is left with what it writes
                auto meet = [&](float keep, float give, int x) { return fmaxf(keep, __shfl_xor_sync(0xffffffffu, give, x)); };
                if constexpr (span == 8) {
                    m0 = fmaxf(m0, fmaxf(s00, s01));
                    m1 = fmaxf(m1, fmaxf(s10, s11));
                    if (++part == S.tiles_per_token) {
                        float v = meet(t0 ? m1 : m0, t0 ? m0 : m1, 1);
                        v = meet(v, v, 2);
                        if (!t1) row[8 * t0] = key_of(__fmul_rn(v, t0 ? ks1 : ks0));
                        part = 0;
                        m0 = m1 = -INFINITY;
                        row += S.ld_keys;
                    }
                } else if constexpr (span == 4) {
                    const float v0 = fmaxf(s00, s01), v1 = fmaxf(s10, s11), v = meet(t0 ? v1 : v0, t0 ? v0 : v1, 1);
                    row[t1 * S.ld_keys + 8 * t0] = key_of(__fmul_rn(v, t0 ? ks1 : ks0));
                    row += 2 * S.ld_keys;
                } else if constexpr (span == 2) {
                    row[t * S.ld_keys] = key_of(__fmul_rn(fmaxf(s00, s01), ks0));
                    row[t * S.ld_keys + 8] = key_of(__fmul_rn(fmaxf(s10, s11), ks1));
                    row += 4 * S.ld_keys;
                } else {
                    row[2 * t * S.ld_keys] = key_of(__fmul_rn(s00, ks0));
                    row[(2 * t + 1) * S.ld_keys] = key_of(__fmul_rn(s01, ks0));
                    row[2 * t * S.ld_keys + 8] = key_of(__fmul_rn(s10, ks1));
                    row[(2 * t + 1) * S.ld_keys + 8] = key_of(__fmul_rn(s11, ks1));
                    row += 8 * S.ld_keys;
                }
            }
            ask();                                                        // (in registers that the fragments have left: two thread blocks an SM)
        }
    };
    switch (S.span_log2) {
        case 0: scores(std::integral_constant<int, 1>()); break;
        case 1: scores(std::integral_constant<int, 2>()); break;
        case 2: scores(std::integral_constant<int, 4>()); break;
        default: scores(std::integral_constant<int, 8>()); break;
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
    while ((1 << S.span_log2) < S.group && S.span_log2 < 3) ++S.span_log2;
    S.tiles_per_token = (S.group + 7) / 8;
    S.ld_keys = ((b.max_len + kKvBlock - 1) / kKvBlock + 15) / 16 * 16 + 4;      // whole groups of 16 blocks; + 4: the tokens' keys in other banks
    if (S.ld_keys < 20) S.ld_keys = 20;
    // Tokens a thread block: 16 tiles of heads, as far as the tokens reach and their keys fit shared memory (128 heads).
    auto rows_of = [&]() { return S.group > 8 ? S.tiles_per_token * 8 : 1 << S.span_log2; };      // of a token
    auto tiles_of = [&](int n) { return (n * rows_of() + 7) / 8; };
    auto room_of = [&](int n) { return S.tiles_per_token > 1 ? n : tiles_of(n) << (3 - S.span_log2); };
    auto need = [&](int n) { return (size_t) room_of(n) * S.ld_keys * 4 + (size_t) tiles_of(n) * (D / 32 * kFrag + 32); };
    // (tiles are whole, and every token they have room for gets keys: one token of a group of one head has eight times its own.  Where that is beyond shared
    // memory, from 404k tokens on, a token takes more rows than it has heads, a tile by itself in the end.  Guards at the stores instead cost every call
    // registers: 16.1 us where this takes 15.7, 16 tokens at up to 64k.)
    while (S.span_log2 < 3 && need(1) > kSmemMost) ++S.span_log2;
    int tokens = rows_of() >= 128 ? 1 : 128 / rows_of();
    if (tokens > b.max_new) tokens = b.max_new;
    while (tokens > 1 && need(tokens) > kSmemMost) tokens = (tokens + 1) / 2;
    // (fewer while that leaves the chip's two thread blocks an SM unfilled: 100 tokens of two sequences at 26k, 3 key/value heads of 2: 70 us, so 27)
    while (tokens > 1 && (long long) b.n_seq * ((b.max_new + tokens - 1) / tokens) * c.n_kv < 2ll * sm_count()) tokens = (tokens + 1) / 2;
    if (need(tokens) > kSmemMost) return refuse(MAYA_ERR_LIMIT);
    S.tokens = tokens;
    S.tiles = tiles_of(tokens);
    S.room = room_of(tokens);
    S.token_tiles = (b.max_new + tokens - 1) / tokens;
    const size_t smem = need(tokens);
    // A sequence's blocks are shared out over a cluster while all thread blocks are on the chip at once (two an SM) and each of their
    // warps has 16 cache blocks to score.
    const long long items = (long long) b.n_seq * S.token_tiles;
    int parts = 1;
    while (parts < 8 && items * c.n_kv * parts * 2 <= (long long) sm_count() * 2 && S.ld_keys >= parts * 2 * kSelWarps * 16) parts *= 2;
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
