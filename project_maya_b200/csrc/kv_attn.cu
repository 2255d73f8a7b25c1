// kv_attn.cu - attention over the paged 8-bit cache for single tokens, windows and short prompts, on mma.sync (m16n8k16, f16 into f32).
//
// What bounds it is the cache's bytes: 2 * head_dim bytes a token and key/value head, read once for the group of query heads
// that shares them.  So everything is made to keep copies in flight: a thread block is four warps with a ring of half-block slots
// (64 tokens of keys, 64 tokens of values: 64 * D contiguous bytes each, one bulk copy), two thread blocks an SM.
//   RW warps share a ring and take 16 rows each; BW = 4 / RW rings take every BW-th cache block.  One token of up to 16 heads a
//   group: RW = 1, every warp on its own; 17..32 rows: 2 x 2; more: one ring, 64 rows.
// Between HBM and the tensor cores a code costs a byte permute and half a subtraction (codes_to_half); no value is written back.
//
// Fragments.  The contraction index of m16n8k16 may be permuted as long as both operands agree, and the cache's layout is chosen for
// it: lane (g, t) of a warp owns values 16 t .. 16 t + 15 of every 64 in a key row (four K = 16 steps of four values from one
// 16-byte load), and tokens 16 t .. 16 t + 15 of the block in a value column.  Keys enter as columns in the order that leaves the
// scores where P wants its tokens: column n of tile j is token 16 (n >> 1) + 4 (j >> 1) + 2 (j & 1) + (n & 1).  Every shared-memory
// load is 16 bytes a lane, a quarter warp on 128 consecutive bytes.
//
// A tile whose cache blocks are split over several thread blocks leaves (m, l, O) partials; the last of them to arrive joins
// all in the order of the splits, so the bits do not depend on who was last.
#include <cuda_fp16.h>

#include "kv_attn.cuh"

namespace maya {
namespace {

constexpr int kThreads = 128, kWarps = 4;
constexpr int kMeta = 256;                        // cache blocks looked up at a time

struct Meta {
    int phys, lb;
    float ks, vs;
};

__device__ __forceinline__ void mma16816(float (&d)[4], const uint4 a, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
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
// what f16 left of a and b
__device__ __forceinline__ uint32_t pack_rest(uint32_t hi, float a, float b) {
    const float2 f = __half22float2(*(const __half2*) &hi);
    return pack_half(a - f.x, b - f.y);
}

template<int D, bool F32, int RW> struct Cfg {
    static constexpr int BW = kWarps / RW;
    static constexpr int rows = 16 * RW;
    static constexpr int slot = kKvBlock * D;                                    // bytes: keys or values of one block
    // slots of a ring: 96 KB a thread block; D = 256: one thread block an SM, what the queries leave of its shared memory
    static constexpr int slots = D == 64 ? 6 * RW : D == 128 ? 3 * RW : D == 192 ? 2 * RW : RW == 1 ? 3 : RW == 2 ? 5 : 9;
    static constexpr int ctas = D == 256 ? 1 : 2;                                // thread blocks an SM
    static constexpr int ring = BW * slots * slot;
    static constexpr int merge = kWarps * 16 * D * 4;                            // the warps' outputs, over the ring's bytes
    static constexpr int frag = RW * (D / 64) * 4 * 512;                         // queries as fragments
    static constexpr int body = ring > merge ? ring : merge;
    static constexpr size_t smem = (size_t) body + (F32 ? 2 : 1) * frag;
};

template<int D, bool F32, int RW>
__global__ void __launch_bounds__(kThreads, Cfg<D, F32, RW>::ctas) attn_kernel(const KvView C, const BatchView B, const AttnView A) {
    using K = Cfg<D, F32, RW>;
    constexpr int BW = K::BW, P = D / 64, V = D / 32;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Meta meta[kMeta];
    __shared__ __align__(8) uint64_t full[BW][K::slots], empty[BW][K::slots];
    __shared__ float qinv[K::rows], sm_m[kWarps][16], sm_l[kWarps][16], sm_vr[kWarps];
    __shared__ int lost, arrived;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int bw = warp / RW, rw = warp % RW;
    uint8_t* ring = smem + (size_t) bw * K::slots * K::slot;
    uint8_t* fragq = smem + K::body;

    if (tid == 0) {
        for (int b = 0; b < BW; ++b)
            for (int i = 0; i < K::slots; ++i) { mbar_init(&full[b][i], 1); mbar_init(&empty[b][i], RW); }
        lost = 0;
        mbar_fence_init();
    }
    grid_launch_dependents();
    grid_dependency_wait();

    // ---- the tile: rows r0 .. of (new token, head of the group) pairs of one sequence, or of one token with a list
    const int split = blockIdx.z, h = blockIdx.y;
    const int unit = blockIdx.x / A.row_tiles, r0 = (A.row_tiles - 1 - blockIdx.x % A.row_tiles) * K::rows;   // the longest rows of a prompt first
    const int si = A.sel != nullptr ? seq_of_row(B, unit) : unit;
    const Seq s = seq_of(B, si);
    const int i0 = A.sel != nullptr ? unit - s.row : 0;                          // the unit's first new token
    const int n_rows = A.sel != nullptr ? A.group : s.n_new * A.group;
    if (r0 >= n_rows || i0 >= s.n_new) return;
    const int first = s.len - s.n_new;
    const int last_row = min(r0 + K::rows, n_rows) - 1;
    const int pos_lo = first + i0 + r0 / A.group, pos_hi = first + i0 + last_row / A.group;
    const int* list = A.sel != nullptr ? A.sel + ((size_t) unit * C.n_kv + h) * A.n_sel : nullptr;
    const int b_lo = list != nullptr || A.window <= 0 ? 0 : max(0, pos_lo - A.window + 1) / kKvBlock;
    const int n_blocks = list != nullptr ? A.n_sel : max(0, (pos_hi < 0 ? -1 : pos_hi / kKvBlock) + 1 - b_lo);
    const int block_hi = pos_hi < 0 ? -1 : pos_hi / kKvBlock;
    const int my0 = split * A.split_blocks, my1 = min(my0 + A.split_blocks, n_blocks);
    const int splits = max(1, (n_blocks + A.split_blocks - 1) / A.split_blocks);  // of this tile
    if (split >= splits) return;

    // ---- queries: scaled by a power of two, rounded to f16 (f32: two terms), laid out as fragments
    for (int r = warp; r < K::rows; r += kWarps) {
        const int row = r0 + r, i = i0 + row / A.group, hq = h * A.group + row % A.group;
        float x[V];
#pragma unroll
        for (int e = 0; e < V; ++e) x[e] = 0.0f;
        if (row < n_rows) ld_acts<!F32, V>(A.q, (size_t) (s.row + i) * A.ld_q + (size_t) hq * D + lane * V, A.wide_q, x);
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) amax = fmaxf(amax, fabsf(x[e]));
        amax = warp_max(amax);
        const int exp2_ = amax > 0.0f ? max(-100, min(100, 138 - (int) (__float_as_uint(amax) >> 23))) : 0;   // amax * 2^e in [2^11, 2^12)
        const float up = __uint_as_float((uint32_t) (127 + exp2_) << 23);
        if (lane == 0) qinv[r] = __uint_as_float((uint32_t) (127 - exp2_) << 23) * A.scale_log2;
#pragma unroll
        for (int e = 0; e < V; e += 2) {
            const int d = lane * V + e, dd = d & 63, tt = dd >> 4, st = (dd >> 2) & 3, w = dd & 3;
            uint8_t* f = fragq + ((((r >> 4) * P + (d >> 6)) * 4 + st) * 32 + (r & 7) * 4 + tt) * 16 + (((w >> 1) * 2) + ((r >> 3) & 1)) * 4;
            const uint32_t hi = pack_half(x[e] * up, x[e + 1] * up);
            *(uint32_t*) f = hi;
            if constexpr (F32) *(uint32_t*) (f + K::frag) = pack_rest(hi, x[e] * up, x[e + 1] * up);
        }
    }

    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[i][e] = 0.0f;
    float m[2] = {kNone, kNone}, l[2] = {0.0f, 0.0f}, vr = 0.0f;
    int pos[2];                                                                  // last visible position of rows g, g + 8 (rows beyond the tile's: all, not kept)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const int row = r0 + rw * 16 + g + 8 * e;
        pos[e] = row < n_rows ? first + i0 + row / A.group : 0x3fffffff;
    }
    const int wpos_lo = __reduce_min_sync(0xffffffffu, min(pos[0], pos[1]));     // over the warp's rows
    const int wpos_hi = first + i0 + min(last_row, r0 + rw * 16 + 15) / A.group;

    unsigned u_put = 0, u_get = 0;                                               // half-block slots asked for and taken so far by this ring
    bool ok = true;
    for (int c0 = my0; c0 < my1 && ok; c0 += kMeta) {
        const int nc = min(kMeta, my1 - c0);
        __syncthreads();                                                         // queries (first round); everybody is done with meta
        if (lost) break;
        for (int i = tid; i < nc; i += kThreads) {
            Meta x;
            x.lb = list != nullptr ? list[c0 + i] : b_lo + c0 + i;
            x.phys = x.lb >= 0 && x.lb <= block_hi ? block_of(C, si, x.lb) : -1;
            x.ks = x.vs = 0.0f;
            if (x.phys >= 0) {
                const size_t bh = (size_t) x.phys * C.n_kv + h;
                x.ks = C.k_scale[bh];
                x.vs = C.v_scale[bh];
            }
            meta[i] = x;
        }
        __syncthreads();

        // copies of this ring's blocks: keys and values by turns, as many half blocks ahead as there are slots
        int put = bw;                                                            // next block to ask for
        bool put_v = false;
        auto ask = [&](unsigned limit) {                                         // by the ring's first warp, until `limit` halves are asked for
            while (put < nc && u_put < limit) {
                const Meta x = meta[put];
                if (x.phys < 0) { put += BW; continue; }
                const unsigned sl = u_put % K::slots;
                if (u_put >= K::slots && RW > 1 && !mbar_wait(&empty[bw][sl], ((u_put / K::slots) - 1) & 1)) { ok = false; return; }
                if (lane == 0) {
                    mbar_expect_tx(&full[bw][sl], K::slot);
                    bulk_load(ring + sl * K::slot, (put_v ? C.v : C.k) + ((size_t) x.phys * C.n_kv + h) * K::slot, K::slot, &full[bw][sl]);
                }
                ++u_put;
                if (put_v) put += BW;
                put_v = !put_v;
            }
        };
        if (rw == 0) ask(u_get + K::slots);

        for (int b = bw; b < nc && ok; b += BW) {
            const Meta x = meta[b];
            if (x.phys < 0) continue;
            // ---- S = Q K^T
            unsigned sl = u_get % K::slots;
            if (!mbar_wait(&full[bw][sl], (u_get / K::slots) & 1)) { ok = false; break; }
            float sc[8][4];
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[j][e] = 0.0f;
            const uint8_t* kp = ring + sl * K::slot + (16 * (g >> 1) + (g & 1)) * 64 + t * 16;
#pragma unroll
            for (int p = 0; p < P; ++p) {
                uint4 a[4], a2[F32 ? 4 : 1];
#pragma unroll
                for (int st = 0; st < 4; ++st) {
                    a[st] = *(const uint4*) (fragq + (((rw * P + p) * 4 + st) * 32 + lane) * 16);
                    if constexpr (F32) a2[st] = *(const uint4*) (fragq + K::frag + (((rw * P + p) * 4 + st) * 32 + lane) * 16);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint4 w = *(const uint4*) (kp + p * (kKvBlock * 64) + (4 * (j >> 1) + 2 * (j & 1)) * 64);
                    const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
                    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int st = 0; st < 4; ++st) {
                        uint32_t b0, b1;
                        codes_to_half(ww[st], b0, b1);
                        if constexpr (F32) {
                            mma16816(part, a2[st], b0, b1);
                            mma16816(part, a[st], b0, b1);
                        } else {
                            mma16816(sc[j], a[st], b0, b1);
                        }
                    }
                    if constexpr (F32)
#pragma unroll
                        for (int e = 0; e < 4; ++e) sc[j][e] += part[e];
                }
            }
            __syncwarp();
            if (RW > 1 && lane == 0) mbar_arrive_one(&empty[bw][sl]);
            ++u_get;
            if (rw == 0) ask(u_get + K::slots);

            // ---- running maximum, P
            const int tb = x.lb * kKvBlock;
            float c[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) c[e] = qinv[rw * 16 + g + 8 * e] * x.ks;
            if (tb + kKvBlock - 1 > wpos_lo || (A.window > 0 && tb <= wpos_hi - A.window)) {      // the block is not visible to every row in whole
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int at = tb + 16 * t + 4 * (j >> 1) + 2 * (j & 1) + (e & 1), to = pos[e >> 1];
                        sc[j][e] = at <= to && (A.window <= 0 || at > to - A.window || to == 0x3fffffff) ? sc[j][e] * c[e >> 1] : kNone;
                    }
                c[0] = c[1] = 1.0f;
            }
            float mx[2] = {kNone, kNone};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                mx[0] = fmaxf(mx[0], fmaxf(sc[j][0], sc[j][1]));
                mx[1] = fmaxf(mx[1], fmaxf(sc[j][2], sc[j][3]));
            }
            const bool vgrew = x.vs > vr;
            float beta = 1.0f;
            if (vgrew) { beta = __fdividef(vr, x.vs); vr = x.vs; }
            const float wv = vr > 0.0f ? x.vs == vr ? 1.0f : __fdiv_rn(x.vs, vr) : 0.0f;
            float alpha[2], off[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 1));
                mx[e] = fmaxf(mx[e], __shfl_xor_sync(0xffffffffu, mx[e], 2));
                const float mn = fmaxf(m[e], mx[e] * c[e]);
                const float use = mn == kNone ? 0.0f : mn;
                alpha[e] = ex2(m[e] - use);
                off[e] = kPBias - use;
                m[e] = mn;
                l[e] *= alpha[e];
                alpha[e] *= beta;
            }
            if (!F32 && __any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    o[i][0] *= alpha[0]; o[i][1] *= alpha[0];
                    o[i][2] *= alpha[1]; o[i][3] *= alpha[1];
                }
            }
            uint4 pa[4], pr[F32 ? 4 : 1];
#pragma unroll
            for (int st = 0; st < 4; ++st) {
                uint32_t hi[4], rest[4];
#pragma unroll
                for (int e = 0; e < 2; ++e) {                                    // rows g, g + 8
#pragma unroll
                    for (int q2 = 0; q2 < 2; ++q2) {                             // tokens + {0, 1}, + {2, 3}
                        const float p0 = ex2(fmaf(sc[2 * st + q2][2 * e], c[e], off[e])), p1 = ex2(fmaf(sc[2 * st + q2][2 * e + 1], c[e], off[e]));
                        l[e] += p0 + p1;
                        hi[q2 * 2 + e] = pack_half(p0 * wv, p1 * wv);
                        if constexpr (F32) rest[q2 * 2 + e] = pack_rest(hi[q2 * 2 + e], p0 * wv, p1 * wv);
                    }
                }
                pa[st] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                if constexpr (F32) pr[st] = make_uint4(rest[0], rest[1], rest[2], rest[3]);
            }

            // ---- O += P V
            sl = u_get % K::slots;
            if (!mbar_wait(&full[bw][sl], (u_get / K::slots) & 1)) { ok = false; break; }
            const uint8_t* vp = ring + sl * K::slot + g * kKvBlock + t * 16;
#pragma unroll
            for (int i = 0; i < D / 8; ++i) {
                const uint4 w = *(const uint4*) (vp + i * 8 * kKvBlock);
                const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
                // f32: a block's products are summed by themselves and added with a rounded add - the tensor cores cut what falls off a
                // sum, always towards zero, and over a long axis that adds up (so do those of 64 values of a score)
                float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int st = 0; st < 4; ++st) {
                    uint32_t b0, b1;
                    codes_to_half(ww[st], b0, b1);
                    if constexpr (F32) {
                        mma16816(part, pr[st], b0, b1);
                        mma16816(part, pa[st], b0, b1);
                    } else {
                        mma16816(o[i], pa[st], b0, b1);
                    }
                }
                if constexpr (F32)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[i][e] = fmaf(o[i][e], alpha[e >> 1], part[e]);
            }
            __syncwarp();
            if (RW > 1 && lane == 0) mbar_arrive_one(&empty[bw][sl]);
            ++u_get;
            if (rw == 0) ask(u_get + K::slots);
        }
        if (!ok) lost = 1;
    }
    if (!ok) {                                                                   // a copy that did not land in time: none may land after the end
        lost = 1;
        if (rw == 0)
            for (unsigned u = u_put > K::slots ? u_put - K::slots : 0; u < u_put; ++u) mbar_wait(&full[bw][u % K::slots], (u / K::slots) & 1);
    }

    // ---- the warps' results meet in shared memory (the ring is done with)
    __syncthreads();
    if (lost) {
        if (tid == 0) atomicExch(A.error, 1u);
        return;
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
        if (t == 0) { sm_m[warp][g + 8 * e] = m[e]; sm_l[warp][g + 8 * e] = l[e]; }
    }
    if (lane == 0) sm_vr[warp] = vr;
    float* mo = (float*) smem;                                                   // [warp][16][D]
#pragma unroll
    for (int i = 0; i < D / 8; ++i) {
        *(float2*) (mo + (warp * 16 + g) * D + 8 * i + 2 * t) = make_float2(o[i][0], o[i][1]);
        *(float2*) (mo + (warp * 16 + g + 8) * D + 8 * i + 2 * t) = make_float2(o[i][2], o[i][3]);
    }
    __syncthreads();
    const size_t slot_id = (size_t) blockIdx.x * C.n_kv + h;
    const int tile_rows = min(K::rows, n_rows - r0);
    auto put_row = [&](int r, int d, float4 v, float total) {                    // four values of row r, divided by the sum
        const int row = r0 + r, i = i0 + row / A.group, hq = h * A.group + row % A.group;
        const size_t at = ((size_t) (s.row + i) * A.n_q + hq) * D + d;
        const float inv = total > 0.0f ? 1.0f / total : 0.0f;
        v.x *= inv; v.y *= inv; v.z *= inv; v.w *= inv;
        if constexpr (F32) *(float4*) ((float*) A.out + at) = v;
        else {
            const __nv_bfloat162 x = __floats2bfloat162_rn(v.x, v.y), y = __floats2bfloat162_rn(v.z, v.w);
            *(uint2*) ((uint16_t*) A.out + at) = make_uint2(*(const uint32_t*) &x, *(const uint32_t*) &y);
        }
    };
    auto put_lse = [&](int r, float mm, float total) {
        const int row = r0 + r, i = i0 + row / A.group, hq = h * A.group + row % A.group;
        if (A.lse != nullptr) A.lse[(size_t) (s.row + i) * A.n_q + hq] = total > 0.0f ? (mm + log2f(total) - kPBias) * 0.69314718055994531f : kNone;
    };
    for (int i = tid; i < tile_rows * (D / 4); i += kThreads) {
        const int r = i / (D / 4), d = (i % (D / 4)) * 4, rr = r & 15, w0 = r >> 4;      // the row's warps: w0 + RW * b
        float mm = kNone, total = 0.0f;
#pragma unroll
        for (int b = 0; b < BW; ++b) mm = fmaxf(mm, sm_m[w0 + RW * b][rr]);
        const float use = mm == kNone ? 0.0f : mm;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int b = 0; b < BW; ++b) {
            const int w = w0 + RW * b;
            const float f = ex2(sm_m[w][rr] - use), fv = f * sm_vr[w];
            total += sm_l[w][rr] * f;
            const float4 y = *(const float4*) (mo + (w * 16 + rr) * D + d);
            v.x += y.x * fv; v.y += y.y * fv; v.z += y.z * fv; v.w += y.w * fv;
        }
        if (splits == 1) {
            put_row(r, d, v, total);
            if (d == 0) put_lse(r, mm, total);
        } else {
            const size_t at = (slot_id * A.n_split + split) * K::rows + r;
            *(float4*) (A.part_o + at * D + d) = v;
            if (d == 0) A.part_ml[at] = make_float2(mm, total);
        }
    }
    if (splits == 1) return;

    // ---- the last of the tile's splits joins them
    __threadfence();
    __syncthreads();
    if (tid == 0) {
        arrived = (int) atomicAdd(A.counters + slot_id, 1u);
        __threadfence();
    }
    __syncthreads();
    if (arrived != splits - 1) return;
    if (tid == 0) A.counters[slot_id] = 0;
    for (int i = tid; i < tile_rows * (D / 4); i += kThreads) {
        const int r = i / (D / 4), d = (i % (D / 4)) * 4;
        const size_t at = slot_id * A.n_split * K::rows + r;
        float mm = kNone, total = 0.0f;
        for (int k = 0; k < splits; ++k) mm = fmaxf(mm, __ldcg(A.part_ml + at + (size_t) k * K::rows).x);
        const float use = mm == kNone ? 0.0f : mm;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int k = 0; k < splits; ++k) {
            const float2 ml = __ldcg(A.part_ml + at + (size_t) k * K::rows);
            const float f = ex2(ml.x - use);
            const float4 y = __ldcg((const float4*) (A.part_o + (at + (size_t) k * K::rows) * D + d));
            total += ml.y * f;
            v.x += y.x * f; v.y += y.y * f; v.z += y.z * f; v.w += y.w * f;
        }
        put_row(r, d, v, total);
        if (d == 0) put_lse(r, mm, total);
    }
}

template<int D, bool F32, int RW>
int launch_attn(const maya_kv_cache& c, const maya_attn_batch& b, const maya_attn_args& a, AttnView A, uint8_t* scratch, size_t scratch_bytes, cudaStream_t s) {
    using K = Cfg<D, F32, RW>;
    const long long rows = a.sel ? A.group : (long long) b.max_new * A.group;
    A.row_tiles = (int) ((rows + K::rows - 1) / K::rows);
    const long long tiles = (long long) A.row_tiles * (a.sel ? b.n_tokens : b.n_seq);
    if (tiles > 0x7fffffffll) return refuse(MAYA_ERR_LIMIT);
    // cache blocks of the longest tile
    long long most = a.sel ? a.n_sel : (b.max_len + kKvBlock - 1) / kKvBlock;
    if (!a.sel && a.window > 0) {
        const long long reach = (a.window + (K::rows + A.group - 1) / A.group + 2 * kKvBlock) / kKvBlock;
        if (reach < most) most = reach;
    }
    if (most < 1) most = 1;
    // Splits: as many as fill the chip once with the longest tiles, none below one block a ring or, to keep ragged batches even, above 64.
    const long long room = (long long) sm_count() * K::ctas, pairs = tiles * c.n_kv;
    long long per = (most * pairs + room - 1) / room;
    if (per < K::BW) per = K::BW;
    if (per > 64) per = 64;
    long long n_split = (most + per - 1) / per;
    const size_t parts = scratch_bytes > kAttnHead + kCountersMost * 4 ? (scratch_bytes - kAttnHead - kCountersMost * 4) / ((D + 2) * 4) : 0;
    if (pairs > kCountersMost || pairs * n_split * K::rows > (long long) parts) {   // no room for the partials: as many as there is room for
        n_split = pairs > kCountersMost ? 1 : (long long) parts / (pairs * K::rows);
        if (n_split < 1) n_split = 1;
        per = (most + n_split - 1) / n_split;
        n_split = (most + per - 1) / per;
    }
    A.split_blocks = (int) per;
    A.n_split = (int) n_split;
    A.counters = (unsigned*) (scratch + kAttnHead);
    A.part_ml = (float2*) (scratch + kAttnHead + kCountersMost * 4);
    A.part_o = (float*) (A.part_ml + pairs * n_split * K::rows);
    static SmemLimit limit;
    if (!limit.raise((const void*) attn_kernel<D, F32, RW>, K::smem)) return note_launch("kv attention smem attribute");
    launch_dependent(attn_kernel<D, F32, RW>, dim3((unsigned) tiles, (unsigned) c.n_kv, (unsigned) n_split), dim3(kThreads), K::smem, s, kv_view(c),
                     batch_view(b), A);
    return note_launch("attn_q8");
}

template<int D, bool F32>
int by_rows(const maya_kv_cache& c, const maya_attn_batch& b, const maya_attn_args& a, const AttnView& A, uint8_t* scratch, size_t bytes,
            cudaStream_t s) {
    const long long rows = (long long) (a.sel ? 1 : b.max_new) * (a.n_q / c.n_kv);
    if (rows <= 16) return launch_attn<D, F32, 1>(c, b, a, A, scratch, bytes, s);
    if (rows <= 32) return launch_attn<D, F32, 2>(c, b, a, A, scratch, bytes, s);
    return launch_attn<D, F32, 4>(c, b, a, A, scratch, bytes, s);
}

}  // namespace
}  // namespace maya

using namespace maya;

extern "C" size_t maya_attn_scratch_bytes(const maya_kv_cache* c, int n_q, int max_tokens) {
    if (kv_check(c) != MAYA_OK || n_q <= 0 || n_q % c->n_kv != 0 || max_tokens <= 0) return 0;
    return kAttnHead + (size_t) kCountersMost * 4 + (size_t) kPartRows * (c->head_dim + 2) * 4;
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
    if (!scratch || ((uintptr_t) scratch & 255u) || scratch_bytes < kAttnHead + kCountersMost * 4) return refuse(MAYA_ERR_ARG);
    cudaStream_t s = as_stream(stream);
    AttnView A{};
    A.q = a->q; A.ld_q = a->ld_q; A.out = a->out; A.lse = a->lse; A.sel = a->sel; A.n_sel = a->n_sel; A.n_q = a->n_q; A.group = a->n_q / c->n_kv;
    A.window = a->window;
    A.wide_q = rows_wide(a->q, a->ld_q, a->is_bf16 ? 2 : 4);
    A.scale_log2 = a->scale * 1.4426950408889634f;
    A.error = (unsigned*) scratch;
    st = attn_prompt(*c, *b, A, a->is_bf16 != 0, s);
    if (st != kNotTaken) return st;
#define ATTN(D) a->is_bf16 ? by_rows<D, false>(*c, *b, *a, A, (uint8_t*) scratch, scratch_bytes, s) : by_rows<D, true>(*c, *b, *a, A, (uint8_t*) scratch, scratch_bytes, s)
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
