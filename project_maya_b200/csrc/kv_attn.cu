// kv_attn.cu - attention over the paged 8-bit cache for single tokens, windows and short prompts, on mma.sync (m16n8k16, f16 into f32).
//
// What bounds it is the cache's bytes: 2 * head_dim bytes a token and key/value head, read once for the group of query heads
// that shares them.  So everything is made to keep copies in flight: a thread block is four warps with rings of 4 KB pieces (64 tokens of 64 key
// values, or 64 values of 64 tokens: contiguous in the cache, one bulk copy each), three thread blocks an SM.  Measured, one B200: 64
// tokens at 1k..16k, 64 heads over 8 of 128: 145 to 151 us, 5.1 to 5.3 TB/s of cache (the copies alone 135 us; f32 154); one at 131071 56 us, 4.8 TB/s (f32 63).
//   RW warps share a ring and take 8 NT rows each; BW = 4 / RW rings take every BW-th cache block.  One token of up to 8 (16) heads a
//   group: RW = 1, NT = 1 (2), every warp on its own; 17..32 rows: 2 x 2; more: one ring, 64 rows.
//
// The codes are the first operand of both products, the queries and P the second: S^T = K Q^T and O^T = V^T P^T.  Rows are then tokens (values), of which
// there are always enough, and columns come in eights, so that a group of 8 heads wastes nothing (with queries as rows of 16 it took twice the
// products, exponentials and registers; the products of a batch of 64 at up to 16k alone 131 us, so 100).  Between HBM and the tensor cores a code costs a byte permute and half
// a subtraction (codes_to_half).
//
// Fragments.  The contraction index of m16n8k16 may be permuted as long as both operands agree, and the cache's layout is chosen for
// it: lane (g, t) of a warp owns values 16 t .. 16 t + 15 of every 64 in a key row (four K = 16 steps of four values from one
// 16-byte load), and tokens 16 t .. 16 t + 15 of the block in a value row.  Row g of S^T's tile s is token 16 (g >> 1) + 4 s + (g & 1), row g + 8 the
// token two further: turned over by movmatrix, P^T's columns are the tokens of V's step s.  Every shared-memory load is 16 bytes a lane, a
// quarter warp on 128 consecutive bytes.
//
// Long sequences are cut into pieces of a few dozen blocks, and the resident thread blocks take one after the other, whatever the sequences' lengths (they
// are known on the device only).  The pieces of a (tile, head) leave (m, l, O) parts, which a second launch joins in order, a warp or a thread block a
// row, so that the bits do not depend on who worked on what.  With more than kTilesMost tiles, or more (tile, head)s than there is room for parts of, none is cut: a
// call then ends with its longest sequence (257 tokens, one at 131k, one key/value head: 968 us, 256 of them 33).
#include <cuda_fp16.h>

#include "kv_attn.cuh"

namespace maya {
namespace {

constexpr int kJoinWarps = 4;
template<bool F32> constexpr float kBias = F32 ? 12.0f : 4.0f;                  // P is kept as 2^bias p
constexpr int kMeta = 128;                        // cache blocks looked up at a time
constexpr int kPiece = 4096;                      // bytes of a ring's slot: 64 tokens x 64 values of K or of V
constexpr long long kWarm = 1 << 20;              // bytes of queries, and of the table, that are asked into L2 ahead
constexpr int kTilesMost = 256;                   // tiles whose blocks a thread block adds up

struct Meta {
    int bh, lb;                                   // block and head in the cache (-1: none); place in the sequence
    float ks, vs;
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint4 a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*) &h;
}
__device__ __forceinline__ uint32_t turned(uint32_t x) {      // an 8 x 8 matrix of f16, a row's pair a lane
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// what f16 left of a and b
__device__ __forceinline__ uint32_t pack_rest(uint32_t hi, float a, float b) {
    const float2 f = __half22float2(*(const __half2*) &hi);
    return pack_half(a - f.x, b - f.y);
}

template<int D, bool F32, int NT, int RW, int NW> struct Cfg {
    static constexpr int BW = NW / RW;
    static constexpr int rows = 8 * NT * RW;
    static constexpr int ctas = NW == 1 ? (D == 64 ? 14 : D == 128 ? (F32 ? 8 : 12) : 7) : D == 64 ? (F32 && NT == 2 ? 2 : 3) : D == 128 ? (F32 || NT == 2 ? 2 : 3) : F32 ? 1 : 2;   // thread blocks an SM
    static constexpr int room = NW == 1 ? 228 * 1024 / ctas - 4800 : ctas == 3 ? 71680 : ctas == 2 ? 108544 : 212992; // and shared memory of each
    static constexpr int frag = RW * NT * (D / 64) * 2 * 512;                    // queries as fragments
    static constexpr int wide = D + 4;                                           // floats of a row where the rings' outputs meet, over the rings
    static constexpr int merge = NW * 8 * NT * wide * 4;
    static constexpr int desk = (F32 ? 2 : 1) * frag;
    static constexpr int slots = (room - desk) / kPiece / BW;                    // of a ring
    static constexpr int body = BW * slots * kPiece;
    static_assert(merge <= body, "outputs meet in the rings' memory");
    static constexpr size_t smem = (size_t) body + desk;
};

// Cache blocks that a tile's rows see, from block b_lo on; rows r0 .. of unit `unit`.
struct Tile {
    Seq s;
    int si, i0, r0, n_rows, first, pos_lo, pos_hi, b_lo, n_blocks;
};
__device__ __forceinline__ Tile tile_of(const BatchView& B, const AttnView& A, int tile, int rows) {
    Tile t;
    const int unit = tile / A.row_tiles;
    t.r0 = (A.row_tiles - 1 - tile % A.row_tiles) * rows;                        // the longest rows of a prompt first
    t.si = A.sel != nullptr ? seq_of_row(B, unit) : unit;
    t.s = seq_of(B, t.si);
    t.i0 = A.sel != nullptr ? unit - t.s.row : 0;                                // the unit's first new token
    t.n_rows = A.sel != nullptr ? (t.i0 < t.s.n_new ? A.group : 0) : t.s.n_new * A.group;
    t.first = t.s.len - t.s.n_new;
    t.pos_lo = t.first + t.i0 + t.r0 / A.group;
    t.pos_hi = t.first + t.i0 + (min(t.r0 + rows, t.n_rows) - 1) / A.group;
    t.b_lo = A.sel != nullptr || A.window <= 0 ? 0 : max(0, t.pos_lo - A.window + 1) / kKvBlock;
    // (a tile whose rows see nothing has one block to look at, which is none: its zeros have to be written all the same)
    t.n_blocks = t.r0 >= t.n_rows ? 0 : A.sel != nullptr ? A.n_sel : t.pos_hi < 0 ? 1 : max(1, t.pos_hi / kKvBlock + 1 - t.b_lo);
    return t;
}
__device__ __forceinline__ size_t out_row(const AttnView& A, const Tile& T, int h, int r) {      // row r of the tile in `out`
    const int row = T.r0 + r;
    return (size_t) (T.s.row + T.i0 + row / A.group) * A.n_q + h * A.group + row % A.group;
}

// A (tile, head)'s cache blocks are cut into pieces of about `q`, of which a thread block works on one at a time: about four a thread block where there are
// many blocks (the SMs are not equally fast: with even shares fixed beforehand the last of 444 thread blocks ended at 147 us, the middle one at 113), none
// below 24 blocks for that, or more than there is room for parts of.
__device__ __forceinline__ unsigned piece_of(const AttnView& A, unsigned blocks, int bw) {
    const unsigned turns = max(1u, min(4u, blocks / A.grid / 24)), share = A.grid * turns;
    const unsigned q = max((blocks + share - 1) / share, blocks / (A.parts_most - A.pairs) + 1);
    return (q + bw - 1) / bw * bw;
}
__device__ __forceinline__ unsigned pieces_of(unsigned nb, unsigned q) { return (nb + q - 1) / q; }

template<int D, bool F32, int NT, int RW, int NW>
__global__ void __launch_bounds__(32 * NW, Cfg<D, F32, NT, RW, NW>::ctas) attn_kernel(const KvView C, const BatchView B, const AttnView A) {
    using K = Cfg<D, F32, NT, RW, NW>;
    constexpr int kWarps = NW, kThreads = 32 * NW;
    constexpr int BW = K::BW, P = D / 64, V = D / 32, TF = F32 ? 2 : 1;
    constexpr float bias = kBias<F32>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Meta meta[kMeta];
    __shared__ __align__(8) uint64_t full[BW][K::slots], empty[BW][K::slots];
    __shared__ float qinv[K::rows], sm_m[kWarps][8 * NT], sm_l[kWarps][8 * NT];
    __shared__ int pre[NW == 1 ? 1 : kTilesMost + 1];
    __shared__ unsigned sums[kWarps], upcoming;
    __shared__ int lost;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int bw = warp / RW, rw = warp % RW;
    uint8_t* ring = smem + (size_t) bw * K::slots * kPiece;
    uint8_t* desk = smem + K::body;

    if (tid == 0) {
        for (int b = 0; b < BW; ++b)
            for (int i = 0; i < K::slots; ++i) { mbar_init(&full[b][i], 1); mbar_init(&empty[b][i], RW); }
        lost = 0;
        mbar_fence_init();
    }
    grid_launch_dependents();
    // what the way to the first copies reads, asked into L2 (the launch in front may still be writing some of it: nothing is read)
    for (unsigned i = blockIdx.x * kThreads + tid; i < A.warm_q + A.warm_table; i += gridDim.x * kThreads) {
        const char* p = i < A.warm_q ? (const char*) A.q + (size_t) i * 128 : (const char*) C.table + (size_t) (i - A.warm_q) * 128;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(p));
    }
    if (tid < 2) asm volatile("prefetch.global.L2 [%0];" ::"l"(tid == 0 ? B.start : B.kv_len));
    grid_dependency_wait();

    // ---- the pieces in front of each tile (of one head)
    unsigned units = 0;
    if (NW == 1 || A.direct) {
        __syncthreads();
    } else if (A.sel != nullptr) {
        units = (unsigned) A.tiles * pieces_of((unsigned) A.n_sel, piece_of(A, (unsigned) A.tiles * (unsigned) C.n_kv * (unsigned) A.n_sel, BW));
        __syncthreads();
    } else {
        if constexpr (NW > 1) {
            const int each = (A.tiles + kThreads - 1) / kThreads;
            unsigned nb[kTilesMost / kThreads], sum = 0;
#pragma unroll
            for (int i = 0; i < kTilesMost / kThreads; ++i) {
                nb[i] = i < each && tid * each + i < A.tiles ? (unsigned) tile_of(B, A, tid * each + i, K::rows).n_blocks : 0u;
                sum += nb[i];
            }
            sum = __reduce_add_sync(0xffffffffu, sum);
            if (lane == 0) sums[warp] = sum;
            __syncthreads();
            unsigned all = 0;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) all += sums[w];
            const unsigned q = piece_of(A, all * (unsigned) C.n_kv, BW);
            sum = 0;
#pragma unroll
            for (int i = 0; i < kTilesMost / kThreads; ++i) sum += pieces_of(nb[i], q);
            unsigned up = sum;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) { const unsigned y = __shfl_up_sync(0xffffffffu, up, o); if (lane >= o) up += y; }
            __syncthreads();
            if (lane == 31) sums[warp] = up;
            __syncthreads();
            unsigned before = up - sum;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) { if (w < warp) before += sums[w]; units += sums[w]; }
#pragma unroll
            for (int i = 0; i < kTilesMost / kThreads; ++i)
                if (i < each && tid * each + i < A.tiles) { pre[tid * each + i] = (int) before; before += pieces_of(nb[i], q); }
            if (tid == 0) pre[A.tiles] = (int) units;
            __syncthreads();
            if (blockIdx.x == 0)                                                     // for the join
                for (int i = tid; i <= A.tiles; i += kThreads) A.pre[i] = pre[i];
        }
    }
    units *= (unsigned) C.n_kv;

    float o[NT][D / 16][4], m[NT][2], l[NT][2];                                  // columns 2 t, 2 t + 1
    int pos[NT][2];
    unsigned u_put = 0, put_phase = 0, get_phase = 0;                            // pieces this ring has asked for; the phases of
    int put_slot = 0, get_slot = 0;                                              // the slots that the next one goes into, and is taken from
    bool ok = true;
    // ---- one piece after the other: the thread block's own number first, then whichever is next
    for (unsigned unit = blockIdx.x;;) {
        if (!A.direct && unit >= units) break;
        unsigned next = 0xffffffffu, pieces = 1, piece = 0;
        if (tid == 0 && !A.direct) next = gridDim.x + atomicAdd(A.taken, 1u);        // (its number arrives meanwhile)
        int tile, h;
        if (A.direct) {
            tile = (int) (unit / (unsigned) C.n_kv);
            h = (int) (unit % (unsigned) C.n_kv);
        } else {
            unsigned in;
            if (A.sel != nullptr) {
                pieces = units / ((unsigned) A.tiles * (unsigned) C.n_kv);
                tile = (int) (unit / (pieces * (unsigned) C.n_kv));
                in = unit % (pieces * (unsigned) C.n_kv);
            } else {
                int lo = 0, hi = A.tiles - 1;                                        // the last tile whose first piece is not behind it
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if ((unsigned) pre[mid] * (unsigned) C.n_kv <= unit) lo = mid; else hi = mid - 1;
                }
                tile = lo;
                pieces = (unsigned) (pre[lo + 1] - pre[lo]);
                in = unit - (unsigned) pre[lo] * (unsigned) C.n_kv;
            }
            h = (int) (in / pieces);
            piece = in % pieces;
        }
        const Tile T = tile_of(B, A, tile, K::rows);
        const unsigned base = (unsigned) T.n_blocks / pieces, rest = (unsigned) T.n_blocks % pieces;
        const int w0 = (int) (piece * base + min(piece, rest)), w1 = w0 + (int) (base + (piece < rest ? 1u : 0u));
        constexpr int U = K::rows / kWarps < 4 ? K::rows / kWarps : 4;               // query rows of a warp in flight
        float qx[U][V];
        auto ask_rows = [&](int r4) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int row = T.r0 + r4 + u * kWarps;
#pragma unroll
                for (int e = 0; e < V; ++e) qx[u][e] = 0.0f;
                if (row < T.n_rows)
                    ld_acts<!F32, V>(A.q, (size_t) (T.s.row + T.i0 + row / A.group) * A.ld_q + (size_t) (h * A.group + row % A.group) * D + lane * V, A.wide_q, qx[u]);
            }
        };
        ask_rows(warp);                                                              // (in front of the copies, behind which they would have to wait)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][i][e] = 0.0f;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m[n][e] = kNone;
                l[n][e] = 0.0f;
                const int row = T.r0 + (rw * NT + n) * 8 + 2 * t + e;                // last visible position (rows beyond the tile's: all, not kept)
                pos[n][e] = row < T.n_rows ? T.first + T.i0 + row / A.group : 0x3fffffff;
            }
        }
        int low = min(pos[0][0], pos[0][1]);
        if constexpr (NT == 2) low = min(low, min(pos[NT - 1][0], pos[NT - 1][1]));
        const int wpos_lo = __reduce_min_sync(0xffffffffu, low);                     // over the warp's rows
        const int wpos_hi = T.first + T.i0 + min(min(T.r0 + K::rows, T.n_rows) - 1, T.r0 + (rw + 1) * NT * 8 - 1) / A.group;

        for (int c0 = w0; c0 < w1; c0 += kMeta) {
            const int nc = min(kMeta, w1 - c0);
            if (c0 > w0) __syncthreads();                                            // everybody is done with meta
            if (lost) break;
            for (int i = tid; i < nc; i += kThreads) {
                const int lb = A.sel != nullptr ? T.n_rows > 0 ? A.sel[((size_t) (tile / A.row_tiles) * C.n_kv + h) * A.n_sel + c0 + i] : -1 : T.b_lo + c0 + i;
                const int phys = lb >= 0 && T.pos_hi >= 0 && lb <= T.pos_hi / kKvBlock ? block_of(C, T.si, lb) : -1;
                meta[i].lb = lb;
                meta[i].bh = phys >= 0 ? phys * C.n_kv + h : -1;
            }
            __syncthreads();

            // copies of this ring's blocks: the pieces of a block's keys, then of its values, as many ahead as there are slots
            int put = bw, put_at = 0;                                                // next block to ask for, and its next piece
            const uint8_t* src = nullptr;                                            // the piece
            auto ask = [&]() {                                                       // one piece, by the ring's first warp
                if (put_at == 0) {
                    while (put < nc && meta[put].bh < 0) put += BW;
                    if (put < nc) src = C.k + (size_t) meta[put].bh * (P * kPiece);
                }
                if (put >= nc) return;
                if (RW > 1 && u_put >= K::slots && !mbar_wait(&empty[bw][put_slot], put_phase ^ 1u)) { ok = false; return; }
                if (lane == 0) {
                    mbar_expect_tx(&full[bw][put_slot], kPiece);
                    bulk_load(ring + put_slot * kPiece, src, kPiece, &full[bw][put_slot]);
                }
                ++u_put;
                if (++put_slot == K::slots) { put_slot = 0; put_phase ^= 1u; }
                src += kPiece;
                if (++put_at == P) src += C.v - C.k - P * kPiece;
                if (put_at == 2 * P) { put_at = 0; put += BW; }
            };
            auto take = [&]() -> const uint8_t* {                                    // the ring's next piece, once it is there
                if (!mbar_wait(&full[bw][get_slot], get_phase)) { ok = false; return nullptr; }
                return ring + get_slot * kPiece;
            };
            auto leave = [&]() {                                                     // and its room for another
                __syncwarp();
                if (RW > 1 && lane == 0) mbar_arrive_one(&empty[bw][get_slot]);
                if (++get_slot == K::slots) { get_slot = 0; get_phase ^= 1u; }
                if (rw == 0) ask();
            };
            if (rw == 0)
                for (int i = 0; i < K::slots && ok; ++i) ask();
            for (int i = tid; i < nc; i += kThreads) {                               // the scales, behind the first copies
                const int bh = meta[i].bh;
                meta[i].ks = bh >= 0 ? C.k_scale[bh] : 0.0f;
                meta[i].vs = bh >= 0 ? C.v_scale[bh] : 0.0f;
            }
            if (c0 == w0) {
                // scaled by a power of two, rounded to f16 (f32: two terms), laid out as fragments
                for (int r4 = warp; r4 < K::rows; r4 += kWarps * U) {
                    if (r4 != warp) ask_rows(r4);
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const int r = r4 + u * kWarps;
                        float amax = 0.0f;
#pragma unroll
                        for (int e = 0; e < V; ++e) amax = fmaxf(amax, fabsf(qx[u][e]));
                        amax = warp_max(amax);
                        const int exp2_ = up_of_row(amax);   // amax * 2^e in [2^11, 2^12)
                        const float up = __uint_as_float((uint32_t) (127 + exp2_) << 23);
                        if (lane == 0) qinv[r] = scale_of_row(amax, __uint_as_float((uint32_t) (127 - exp2_) << 23) * A.scale_log2);
#pragma unroll
                        for (int e = 0; e < V; e += 2) {
                            const int d = lane * V + e, dd = d & 63, tt = dd >> 4, st = (dd >> 2) & 3, w = dd & 3;
                            uint8_t* f = desk + ((((r >> 3) * P + (d >> 6)) * 2 + (st >> 1)) * 32 + (r & 7) * 4 + tt) * 16 + ((st & 1) * 2 + (w >> 1)) * 4;
                            const uint32_t hi = pack_half(qx[u][e] * up, qx[u][e + 1] * up);
                            *(uint32_t*) f = hi;
                            if constexpr (F32) *(uint32_t*) (f + K::frag) = pack_rest(hi, qx[u][e] * up, qx[u][e + 1] * up);
                        }
                    }
                }
            }
            __syncthreads();

            for (int b = bw; b < nc && ok; b += BW) {
                const Meta x = meta[b];
                if (x.bh < 0) continue;
                // ---- S^T = K Q^T: rows of tile s are tokens, columns the queries
                float sc[NT][4][4];
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int s = 0; s < 4; ++s)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sc[n][s][e] = 0.0f;
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const uint8_t* kp = take();
                    if (!ok) break;
                    kp += (16 * (g >> 1) + (g & 1)) * 64 + t * 16;
                    uint4 q[TF][NT][2];
#pragma unroll
                    for (int f = 0; f < TF; ++f)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
                                q[f][n][i] = *(const uint4*) (desk + f * K::frag + ((((rw * NT + n) * P + p) * 2 + i) * 32 + lane) * 16);
                    constexpr int SG = NT == 1 ? 4 : 2;                          // tiles side by side: one's wait for the product before is another's turn
#pragma unroll
                    for (int s0 = 0; s0 < 4; s0 += SG) {
                        uint32_t wa[SG][4], wb[SG][4];
#pragma unroll
                        for (int i = 0; i < SG; ++i) {
                            *(uint4*) wa[i] = *(const uint4*) (kp + 4 * (s0 + i) * 64);
                            *(uint4*) wb[i] = *(const uint4*) (kp + (4 * (s0 + i) + 2) * 64);
                        }
                        // (f32: 64 values' products are summed by themselves and added with a rounded add - the tensor cores cut what falls off a sum,
                        // always towards zero, and over a long axis that adds up)
                        float part[NT][SG][4];
                        if constexpr (F32)
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int i = 0; i < SG; ++i)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) part[n][i][e] = 0.0f;
#pragma unroll
                        for (int st = 0; st < 4; ++st)
#pragma unroll
                            for (int i = 0; i < SG; ++i) {
                                uint4 a;
                                codes_to_half(wa[i][st], a.x, a.z);
                                codes_to_half(wb[i][st], a.y, a.w);
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int f = TF - 1; f >= 0; --f) {
                                        const uint4 y = q[f][n][st >> 1];
                                        mma16816(F32 ? part[n][i] : sc[n][s0 + i], a, st & 1 ? y.z : y.x, st & 1 ? y.w : y.y);
                                    }
                            }
                        if constexpr (F32)
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int i = 0; i < SG; ++i)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) sc[n][s0 + i][e] += part[n][i][e];
                    }
                    leave();
                }
                if (!ok) break;

                // ---- running maximum, P^T
                const int tb = x.lb * kKvBlock;
                const bool cut = tb + kKvBlock - 1 > wpos_lo || (A.window > 0 && tb <= wpos_hi - A.window);      // not visible to every row in whole
                // V's scale is in P's exponent (m is then of s + log2 vs, and l takes it out again): bf16: all of it; f32, where a logarithm would cost
                // bits: its power of two, the rest (1 .. 2) a factor
                float wv = 1.0f, lv, ivs;
                if constexpr (F32) {
                    const uint32_t e = min(max(__float_as_uint(x.vs) >> 23, kVsExpLeast), 253u);
                    lv = (float) ((int) e - 127);
                    ivs = __uint_as_float((254u - e) << 23);
                    wv = x.vs * ivs;
                } else {
                    const float vs = fmaxf(x.vs, kVsLeast);
                    lv = __log2f(vs);
                    ivs = __fdividef(1.0f, vs);
                }
                float alpha[NT][2];
                bool moved = false;
                uint32_t pb[TF][NT][4][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    float off[2], c[2], sum[2] = {0.0f, 0.0f};
#pragma unroll
                    for (int e = 0; e < 2; ++e) c[e] = qinv[(rw * NT + n) * 8 + 2 * t + e] * x.ks;
                    if (cut) {
#pragma unroll
                        for (int s = 0; s < 4; ++s)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int at = tb + 16 * (g >> 1) + 4 * s + (g & 1) + (e & 2), to = pos[n][e & 1];
                                sc[n][s][e] = at <= to && (A.window <= 0 || at > to - A.window || to == 0x3fffffff) ? sc[n][s][e] * c[e & 1] : kNone;
                            }
                        c[0] = c[1] = 1.0f;
                    }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(sc[n][0][e], sc[n][0][e + 2]);
#pragma unroll
                        for (int s = 1; s < 4; ++s) mx = fmaxf(mx, fmaxf(sc[n][s][e], sc[n][s][e + 2]));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        const float top = fmaf(mx, c[e], lv);
                        if constexpr (F32) {
                            const float mn = fmaxf(m[n][e], top), use = mn == kNone ? 0.0f : mn, al = ex2(m[n][e] - use);
                            off[e] = bias + lv - use;
                            m[n][e] = mn;
                            l[n][e] *= al;
                            alpha[n][e] = al;
                        } else {                                                 // m is raised only when it is passed by more than kRise: P stays below 2^12
                            alpha[n][e] = 1.0f;
                            if (top > m[n][e] + kRise) {
                                alpha[n][e] = ex2(m[n][e] - top);
                                l[n][e] *= alpha[n][e];
                                m[n][e] = top;
                                moved = true;
                            }
                            off[e] = m[n][e] == kNone ? kNone : bias + lv - m[n][e];
                        }
                    }
#pragma unroll
                    for (int s = 0; s < 4; ++s)
#pragma unroll
                        for (int hh = 0; hh < 2; ++hh) {                         // rows g, g + 8
                            const float p0 = ex2(fmaf(sc[n][s][2 * hh], c[0], off[0])), p1 = ex2(fmaf(sc[n][s][2 * hh + 1], c[1], off[1]));
                            sum[0] += p0;
                            sum[1] += p1;
                            if constexpr (F32) {
                                const uint32_t hi = pack_half(p0 * wv, p1 * wv);
                                pb[0][n][s][hh] = turned(hi);
                                pb[TF - 1][n][s][hh] = turned(pack_rest(hi, p0 * wv, p1 * wv));
                            } else {
                                pb[0][n][s][hh] = turned(pack_half(p0, p1));
                            }
                        }
#pragma unroll
                    for (int e = 0; e < 2; ++e) l[n][e] = fmaf(sum[e], ivs, l[n][e]);
                }
                if (!F32 && __any_sync(0xffffffffu, moved))
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < D / 16; ++i)
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[n][i][e] *= alpha[n][e & 1];

                // ---- O^T += V^T P^T: rows are values
#pragma unroll
                for (int p = 0; p < P; ++p) {
                    const uint8_t* vp = take();
                    if (!ok) break;
                    vp += g * kKvBlock + t * 16;
#pragma unroll
                    for (int i0 = 0; i0 < 4; i0 += 2) {
                        uint32_t wa[2][4], wb[2][4];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            *(uint4*) wa[i] = *(const uint4*) (vp + 16 * (i0 + i) * kKvBlock);
                            *(uint4*) wb[i] = *(const uint4*) (vp + (16 * (i0 + i) + 8) * kKvBlock);
                        }
                        float part[NT][2][4];
                        if constexpr (F32)
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int i = 0; i < 2; ++i)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) part[n][i][e] = 0.0f;
#pragma unroll
                        for (int st = 0; st < 4; ++st)
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                uint4 a;
                                codes_to_half(wa[i][st], a.x, a.z);
                                codes_to_half(wb[i][st], a.y, a.w);
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int f = TF - 1; f >= 0; --f)
                                        mma16816(F32 ? part[n][i] : o[n][4 * p + i0 + i], a, pb[f][n][st][0], pb[f][n][st][1]);
                            }
                        if constexpr (F32)
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int i = 0; i < 2; ++i)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) {
                                        float& y = o[n][4 * p + i0 + i][e];
                                        y = fmaf(y, alpha[n][e & 1], part[n][i][e]);
                                    }
                    }
                    leave();
                }
                if (!ok) break;
            }
            if (!ok) lost = 1;
        }

        // ---- the rings' results meet in the rings' memory (nothing is on its way into it), a thread four values of a row
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int x = 4; x < 32; x *= 2) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], x);
        if (g == 0) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) { sm_m[warp][n * 8 + 2 * t + e] = m[n][e]; sm_l[warp][n * 8 + 2 * t + e] = l[n][e]; }
        }
        __syncthreads();                                                     // every ring is empty
        float* buf = (float*) smem;                                          // [warp][8 NT][wide]
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) buf[((warp * NT + n) * 8 + 2 * t + (e & 1)) * K::wide + 16 * i + g + (e & 2) * 4] = o[n][i][e];
        __syncthreads();
        if (lost) break;
        const bool whole = pieces == 1;
        const size_t part_at = (size_t) unit * K::rows;
        for (int i = tid; i < K::rows * (D / 4); i += kThreads) {
            const int r = i / (D / 4), d = (i % (D / 4)) * 4, rr = r % (8 * NT), x0 = r / (8 * NT);      // the row's warps: x0 + RW * b
            if (T.r0 + r >= T.n_rows) break;
            float mm = kNone, total = 0.0f;
#pragma unroll
            for (int b = 0; b < BW; ++b) mm = fmaxf(mm, sm_m[x0 + RW * b][rr]);
            const float use = mm == kNone ? 0.0f : mm;
            float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int b = 0; b < BW; ++b) {
                const int x = x0 + RW * b;
                const float f = ex2(sm_m[x][rr] - use);
                total += sm_l[x][rr] * f;
                const float4 z = *(const float4*) (buf + (x * 8 * NT + rr) * K::wide + d);
                y.x += z.x * f; y.y += z.y * f; y.z += z.z * f; y.w += z.w * f;
            }
            if (!whole) {
                *(float4*) (A.part_o + (part_at + r) * D + d) = y;
                if (d == 0) A.part_ml[part_at + r] = make_float2(mm, total);
                continue;
            }
            const float inv = total == 0.0f ? 0.0f : 1.0f / total;
            y.x *= inv; y.y *= inv; y.z *= inv; y.w *= inv;
            const size_t at = out_row(A, T, h, r);
            if constexpr (F32) *(float4*) ((float*) A.out + at * D + d) = y;
            else {
                const __nv_bfloat162 a = __floats2bfloat162_rn(y.x, y.y), b = __floats2bfloat162_rn(y.z, y.w);
                *(uint2*) ((uint16_t*) A.out + at * D + d) = make_uint2(*(const uint32_t*) &a, *(const uint32_t*) &b);
            }
            if (d == 0 && A.lse != nullptr) A.lse[at] = lse_of(mm, total, kBias<F32>);
        }
        fence_proxy_async();                                                 // the next copies write where this was read
        if (A.direct) break;
        if (tid == 0) upcoming = next;
        __syncthreads();
        unit = upcoming;
    }
    if (!ok && rw == 0)                                                          // a copy that did not land in time: none may land after the end
        for (unsigned u = u_put > K::slots ? u_put - K::slots : 0; u < u_put; ++u) mbar_wait(&full[bw][u % K::slots], (u / K::slots) & 1);
    __syncthreads();
    if (tid == 0) {
        if (lost) atomicExch(A.error, 1u);
        if (!A.direct) {                                                         // the last to leave sets the counters back
            __threadfence();
            if (atomicAdd(A.taken + 1, 1u) == gridDim.x - 1) A.taken[0] = A.taken[1] = 0u;
        }
    }
}

// The rows of (tile, head)s that were cut into pieces, from their parts in order: a thread block a row (WIDE: few rows, each of many
// parts), or a warp.
template<int D, bool F32, bool WIDE>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const KvView C, const BatchView B, const AttnView A, int rows, int bw) {
    constexpr int V = D / 32, W = WIDE ? kJoinWarps : 1;
    __shared__ float acc_of[WIDE ? kJoinWarps : 1][D], l_of[kJoinWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = WIDE ? warp : 0;
    const long long id = WIDE ? (long long) blockIdx.x : (long long) blockIdx.x * kJoinWarps + warp;
    const int r = (int) (id % rows), h = (int) (id / rows % C.n_kv), tile = (int) (id / rows / C.n_kv);
    grid_launch_dependents();
    grid_dependency_wait();
    if (tile >= A.tiles) return;
    unsigned pieces, s0;
    if (A.fixed > 0) {
        pieces = A.fixed;
        s0 = ((unsigned) tile * (unsigned) C.n_kv + h) * pieces;
    } else if (A.sel != nullptr) {
        pieces = pieces_of((unsigned) A.n_sel, piece_of(A, (unsigned) A.tiles * (unsigned) C.n_kv * (unsigned) A.n_sel, bw));
        s0 = ((unsigned) tile * (unsigned) C.n_kv + h) * pieces;
    } else {
        const unsigned p0 = (unsigned) A.pre[tile];
        pieces = (unsigned) A.pre[tile + 1] - p0;
        s0 = p0 * (unsigned) C.n_kv + h * pieces;
    }
    if (pieces <= 1) return;
    const unsigned s1 = s0 + pieces - 1;
    const Tile T = tile_of(B, A, tile, rows);
    if (T.r0 + r >= T.n_rows) return;
    auto slot_of = [&](unsigned c) { return (size_t) c * rows + r; };
    float mm = kNone, total = 0.0f;
    for (unsigned c = s0 + lane; c <= s1; c += 32) mm = fmaxf(mm, A.part_ml[slot_of(c)].x);
    mm = warp_max(mm);
    const float use = mm == kNone ? 0.0f : mm;
    float acc[V];
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] = 0.0f;
    for (unsigned c32 = s0 + part * 32; c32 <= s1; c32 += 32 * W) {
        float f = 0.0f;
        if (c32 + lane <= s1) {
            const float2 x = A.part_ml[slot_of(c32 + lane)];
            f = ex2(x.x - use);
            total += x.y * f;
        }
#pragma unroll
        for (int k0 = 0; k0 < 32; k0 += 16) {                                    // sixteen parts in flight
            if (c32 + k0 > s1) break;
            float y[16][V];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const float* src = A.part_o + slot_of(min(c32 + k0 + k, s1)) * D + lane * V;
#pragma unroll
                for (int e = 0; e < V; e += 2) *(float2*) &y[k][e] = *(const float2*) (src + e);
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const float fk = __shfl_sync(0xffffffffu, f, k0 + k);            // (0 behind the last)
#pragma unroll
                for (int e = 0; e < V; ++e) acc[e] = fmaf(y[k][e], fk, acc[e]);
            }
        }
    }
    total = warp_sum(total);
    if constexpr (WIDE) {
#pragma unroll
        for (int e = 0; e < V; ++e) acc_of[warp][lane * V + e] = acc[e];
        if (lane == 0) l_of[warp] = total;
        __syncthreads();
        if (warp != 0) return;
        total = 0.0f;
#pragma unroll
        for (int x = 0; x < kJoinWarps; ++x) total += l_of[x];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            acc[e] = 0.0f;
#pragma unroll
            for (int x = 0; x < kJoinWarps; ++x) acc[e] += acc_of[x][lane * V + e];
        }
    }
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    const size_t at = out_row(A, T, h, r);
#pragma unroll
    for (int e = 0; e < V; ++e) st_act<!F32>(A.out, at * D + lane * V + e, acc[e] * inv);
    if (A.lse != nullptr && lane == 0) A.lse[at] = lse_of(mm, total, kBias<F32>);
}

template<int D, bool F32>
int launch_join(const maya_kv_cache& c, const maya_attn_batch& b, const AttnView& A, int rows, int bw, cudaStream_t s) {
    const long long all = (long long) A.tiles * c.n_kv * rows;
    if (all <= 4 * sm_count()) launch_dependent(join_kernel<D, F32, true>, dim3((unsigned) all), dim3(32 * kJoinWarps), 0, s, kv_view(c), batch_view(b), A, rows, bw);
    else launch_dependent(join_kernel<D, F32, false>, dim3((unsigned) ((all + kJoinWarps - 1) / kJoinWarps)), dim3(32 * kJoinWarps), 0, s, kv_view(c), batch_view(b), A, rows, bw);
    return note_launch("attn_q8 join");
}

template<int D, bool F32, int NT, int RW, int NW = 4>
int launch_attn(const maya_kv_cache& c, const maya_attn_batch& b, const maya_attn_args& a, AttnView A, cudaStream_t s) {
    using K = Cfg<D, F32, NT, RW, NW>;
    static_assert(K::slots >= 2, "a ring holds a piece in use and one on its way");
    const long long rows = a.sel ? A.group : (long long) b.max_new * A.group;
    A.row_tiles = (int) ((rows + K::rows - 1) / K::rows);
    const long long tiles = (long long) A.row_tiles * (a.sel ? b.n_tokens : b.n_seq);
    long long most = a.sel ? a.n_sel : (b.max_len + kKvBlock - 1) / kKvBlock;    // cache blocks of the longest tile
    if (!a.sel && A.window > 0) {
        const long long reach = (A.window + (K::rows + A.group - 1) / A.group + 2 * kKvBlock) / kKvBlock;
        if (reach < most) most = reach;
    }
    if (most < 1) most = 1;
    // As many thread blocks as are on the chip at once, each with an even share of the cache blocks; none with less than a round of its rings.
    // With more tiles than a thread block adds up in one go, one a (tile, head): there are enough of them to fill the chip.
    A.tiles = (int) tiles;
    A.direct = (!a.sel && tiles > kTilesMost) || tiles * most * c.n_kv >= 0x7fffffffll;
    long long grid = tiles * c.n_kv;
    if (grid > 0x7fffffffll) return refuse(MAYA_ERR_LIMIT);
    if (!A.direct) {
        const long long rounds = (tiles * most * c.n_kv + K::BW - 1) / K::BW;
        grid = (long long) sm_count() * K::ctas;
        if (grid > kCtasMost) grid = kCtasMost;
        if (grid > rounds) grid = rounds;
    }
    A.grid = (unsigned) grid;
    A.pairs = (unsigned) (tiles * c.n_kv);
    A.parts_most = (unsigned) (kPartRows / K::rows);
    if (A.pairs >= A.parts_most / 2) A.direct = true;                            // many (tile, head)s: whole ones, as many thread blocks
    if (NW == 1) A.direct = true;
    if (A.direct) grid = tiles * c.n_kv;
    if (grid > 0x7fffffffll) return refuse(MAYA_ERR_LIMIT);
    const long long q_bytes = ((long long) (b.n_tokens - 1) * a.ld_q + (long long) a.n_q * D) * (F32 ? 4 : 2), table_bytes = (long long) b.n_seq * c.table_ld * 4;
    A.warm_q = (unsigned) ((q_bytes < kWarm ? q_bytes : kWarm) / 128);
    A.warm_table = (unsigned) ((table_bytes < kWarm ? table_bytes : kWarm) / 128);
    static SmemLimit limit;
    if (!limit.raise((const void*) attn_kernel<D, F32, NT, RW, NW>, K::smem)) return note_launch("kv attention smem attribute");
    launch_dependent(attn_kernel<D, F32, NT, RW, NW>, dim3((unsigned) grid), dim3(32 * NW), K::smem, s, kv_view(c), batch_view(b), A);
    const int st = note_launch("attn_q8");
    if (st != MAYA_OK || A.direct || grid == 1) return st;
    return launch_join<D, F32>(c, b, A, K::rows, K::BW, s);
}

template<int D, bool F32>
int by_rows(const maya_kv_cache& c, const maya_attn_batch& b, const maya_attn_args& a, const AttnView& A, cudaStream_t s) {
    const long long rows = (long long) (a.sel ? 1 : b.max_new) * (a.n_q / c.n_kv);
    // Lists of many tokens, 8 heads a group or fewer: a warp a (token, head), by itself - no barrier, nothing to meet - once there are enough of them to
    // fill the chip several times (a chunk of 4096 tokens, 4 key/value heads, 16 blocks each: four warps a list 608 us, one 515).
    if (a.sel && rows <= 8 && (long long) b.n_tokens * c.n_kv >= 48ll * sm_count()) return launch_attn<D, F32, 1, 1, 1>(c, b, a, A, s);
    if (rows <= 8) return launch_attn<D, F32, 1, 1>(c, b, a, A, s);
    if constexpr (D <= 128) {
        if (rows <= 16) return launch_attn<D, F32, 2, 1>(c, b, a, A, s);
        if (rows <= 32) return launch_attn<D, F32, 2, 2>(c, b, a, A, s);
        return launch_attn<D, F32, 2, 4>(c, b, a, A, s);
    } else {                                                                     // (two columns of outputs of these sizes do not fit the registers)
        if (rows <= 16) return launch_attn<D, F32, 1, 2>(c, b, a, A, s);
        return launch_attn<D, F32, 1, 4>(c, b, a, A, s);
    }
}

}  // namespace

int attn_join(const maya_kv_cache& c, const maya_attn_batch& b, const AttnView& A, int rows, cudaStream_t s) {
    return c.head_dim == 64 ? launch_join<64, false>(c, b, A, rows, 1, s) : launch_join<128, false>(c, b, A, rows, 1, s);
}

}  // namespace maya

using namespace maya;

extern "C" size_t maya_attn_scratch_bytes(const maya_kv_cache* c, int n_q, int max_tokens) {
    if (kv_check(c) != MAYA_OK || n_q <= 0 || n_q % c->n_kv != 0 || max_tokens <= 0) return 0;
    return kAttnHead + kAttnPre + (size_t) kPartRows * (c->head_dim + 2) * 4;
}

extern "C" int maya_attn_q8(const maya_kv_cache* c, const maya_attn_batch* b, const maya_attn_args* a, void* scratch, size_t scratch_bytes,
                            void* stream) {
    int st = kv_check(c);
    if (st == MAYA_OK) st = batch_check(c, b);
    if (st == MAYA_OK && !a) st = MAYA_ERR_ARG;
    if (st != MAYA_OK) return refuse(st);
    if (b->n_tokens == 0) return MAYA_OK;
    if (!a->q || !a->out || a->n_q <= 0 || a->n_q % c->n_kv != 0 || !(a->scale > 0.0f) || a->window < 0) return refuse(MAYA_ERR_ARG);
    if (a->ld_q < (int64_t) a->n_q * c->head_dim || !aligned16(a->out)) return refuse(MAYA_ERR_ARG);
    if (a->sel && a->n_sel <= 0) return refuse(MAYA_ERR_ARG);
    if ((a->sel && a->n_sel > MAYA_MAX_SELECTED) || c->n_kv > 65535) return refuse(MAYA_ERR_LIMIT);
    if ((long long) b->max_new * (a->n_q / c->n_kv) > 0x7fffff00ll) return refuse(MAYA_ERR_LIMIT);      // (rows of a sequence are ints)
    if (!scratch || ((uintptr_t) scratch & 255u) || scratch_bytes < maya_attn_scratch_bytes(c, a->n_q, 1)) return refuse(MAYA_ERR_ARG);
    cudaStream_t s = as_stream(stream);
    AttnView A{};
    A.q = a->q; A.ld_q = a->ld_q; A.out = a->out; A.lse = a->lse; A.sel = a->sel; A.n_sel = a->n_sel; A.n_q = a->n_q; A.group = a->n_q / c->n_kv;
    A.window = a->window < b->max_len ? a->window : 0;                           // (wider than any sequence: none; what is left keeps int arithmetic in range)
    A.wide_q = rows_wide(a->q, a->ld_q, a->is_bf16 ? 2 : 4);
    A.scale_log2 = a->scale * 1.4426950408889634f;
    A.error = (unsigned*) scratch;
    A.taken = (unsigned*) ((uint8_t*) scratch + 16);
    A.pre = (int*) ((uint8_t*) scratch + kAttnHead);
    A.part_ml = (float2*) ((uint8_t*) scratch + kAttnHead + kAttnPre);
    A.part_o = (float*) (A.part_ml + kPartRows);
    st = attn_prompt(*c, *b, A, a->is_bf16 != 0, s);
    if (st != kNotTaken) return st;
#define ATTN(D) a->is_bf16 ? by_rows<D, false>(*c, *b, *a, A, s) : by_rows<D, true>(*c, *b, *a, A, s)
    switch (c->head_dim) {
        case 64: return ATTN(64);
        case 128: return ATTN(128);
        case 192: return ATTN(192);
        default: return ATTN(256);
    }
#undef ATTN
}

extern "C" int maya_attn_error(const void* scratch, void* stream) {
    unsigned word = 0;
    if (!scratch) return MAYA_ERR_ARG;
    if (cudaMemcpyAsync(&word, scratch, sizeof(word), cudaMemcpyDeviceToHost, as_stream(stream)) != cudaSuccess ||
        cudaStreamSynchronize(as_stream(stream)) != cudaSuccess) {
        note_launch("attn_error");
        return MAYA_ERR_LAUNCH;
    }
    return (int) word;
}
