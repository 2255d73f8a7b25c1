// kv_append.cu - what stands between a layer's projections and its attention: the RMS norm of every query and key head, their
// rotation, and the rounding of keys and values into the blocks of the 8-bit cache, in one launch; and blocks read back as values.
//
// A block's scale is that of its largest value, so the tokens a pass adds to one block have to be seen together: a thread block
// owns (sequence, touched block, key/value head, keys or values), makes the new rows in shared memory (f32), takes their
// largest value, moves the codes that are there to the larger scale if it grew, and writes.  Nobody else writes to that block,
// so nothing is atomic across thread blocks and a call's bits do not depend on how they run.  Query rows are independent: a warp each, and
// the same launch (thread blocks behind the cache's).
//
// Bounds: a decode step is one launch's latency (one dependent chain: lengths, table, scale, rows); a prompt is bytes - the rows read once,
// queries written, a byte a value into the cache.  Measured, one B200: a step of 64
// sequences, 64 heads over 8, 8 us; prompts of 5352 tokens, 48 heads over 8, 75 us (1.7 TB/s; issue 55 % busy).
#include "maya_kv.cuh"

namespace maya {
namespace {

// Two forms: FEW (a step of decode: at most four new tokens a sequence) of 128 threads, with what a block holds already on its way from the start; and
// for prompts 256 threads with two rows of a warp in flight.
template<bool FEW> struct Form {
    static constexpr int threads = FEW ? 128 : 256, warps = threads / 32, rows = FEW ? 1 : 2;
    static constexpr int blocks(int D) { return FEW ? (D <= 128 ? 8 : 4) : (D <= 128 ? 4 : 2); }      // an SM
};

struct RopeView {
    const void *q, *k, *v;
    int64_t ld_q, ld_k, ld_v;
    int n_q;
    const float *q_w, *k_w;
    float eps;
    const float *cos, *sin;
    const int* pos;
    int n_pos, rot, pairs;
    void* q_out;
    int wide_q, wide_k, wide_v, wide_out, heads;          // heads: of a warp's query rows
};

// A lane's part of the rotation at one position: V = D / 32 consecutive values from lane * V on; value d becomes x c + partner s.
template<int D> struct Turn {
    static constexpr int V = D / 32;
    float c[V], s[V];
    __device__ __forceinline__ void at(const RopeView& R, int pos, int lane) {
        const int half = R.rot >> 1;
        const size_t row = (size_t) max(0, min(pos, R.n_pos - 1)) * half;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int d = lane * V + i, j = R.pairs ? d >> 1 : d < half ? d : d - half;
            const bool turns = d < R.rot, second = R.pairs ? d & 1 : d >= half;
            c[i] = turns ? __ldg(R.cos + row + j) : 1.0f;
            s[i] = turns ? __ldg(R.sin + row + j) : 0.0f;
            if (!second) s[i] = -s[i];
        }
    }
};
// One head's row: the norm (w: the lane's weights, NORM or not), then the rotation.  A partner is the lane's own neighbour (pairs) or half / V lanes away;
// where halves begin inside a lane's values, partners change hands through `buf`, D floats of this warp's own.
template<int D>
__device__ __forceinline__ void norm_rotate(float (&x)[D / 32], bool norm, const float (&w)[D / 32], const RopeView& R, const Turn<D>& T, float* buf, int lane) {
    constexpr int V = D / 32;
    if (norm) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) ss += x[i] * x[i];
        ss = warp_sum(ss);
        const float inv = rsqrtf(ss * (1.0f / D) + R.eps);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = x[i] * inv * w[i];
    }
    if (R.rot == 0) return;
    float y[V];
    const int half = R.rot >> 1;
    if (R.pairs) {
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = x[i ^ 1];
    } else if (half % V == 0) {
        const int from = lane * V < half ? lane + half / V : lane - half / V;
#pragma unroll
        for (int i = 0; i < V; ++i) y[i] = __shfl_sync(0xffffffffu, x[i], from & 31);
    } else {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < V; ++i) buf[lane * V + i] = x[i];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int d = lane * V + i;
            y[i] = d < R.rot ? buf[d < half ? d + half : d - half] : 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = x[i] * T.c[i] + y[i] * T.s[i];
}
template<int V, bool BF16> __device__ __forceinline__ void st_acts(void* p, size_t i, const float (&x)[V], bool wide) {
    if (!wide) {
#pragma unroll
        for (int e = 0; e < V; ++e) st_act<BF16>(p, i + e, x[e]);
    } else if constexpr (BF16) {
        uint32_t w[V / 2];
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
            const __nv_bfloat162 y = __floats2bfloat162_rn(x[2 * e], x[2 * e + 1]);
            w[e] = *(const uint32_t*) &y;
        }
        uint32_t* to = (uint32_t*) ((uint16_t*) p + i);
        if constexpr (V == 8) *(uint4*) to = *(const uint4*) w;
        else if constexpr (V == 4) *(uint2*) to = *(const uint2*) w;
        else {
#pragma unroll
            for (int e = 0; e < V / 2; ++e) to[e] = w[e];
        }
    } else {
        float* to = (float*) p + i;
        if constexpr (V % 4 == 0) {
#pragma unroll
            for (int e = 0; e < V; e += 4) *(float4*) (to + e) = *(const float4*) &x[e];
        } else {
#pragma unroll
            for (int e = 0; e < V; e += 2) *(float2*) (to + e) = *(const float2*) &x[e];
        }
    }
}

// A value as its code: nearest (by the scale's reciprocal: within 2^-15 of a step), +-127, NaN 0.
__device__ __forceinline__ int code_of(float x, float inv) {
    const float r = rintf(x * inv);
    return r == r ? (int) fmaxf(-127.0f, fminf(127.0f, r)) : 0;
}
__device__ __forceinline__ int code_moved(uint32_t code, float ratio) { return (int) rintf((float) ((int) code - 128) * ratio); }

template<int D, bool BF16, bool FEW>
__global__ void __launch_bounds__(Form<FEW>::threads, Form<FEW>::blocks(D)) append_kernel(const KvView C, const BatchView B, const RopeView R, int touched, int kv_items) {
    constexpr int V = D / 32, kAppendThreads = Form<FEW>::threads, kAppendWarps = Form<FEW>::warps, U = Form<FEW>::rows;
    extern __shared__ __align__(16) float rows[];                 // [tokens of the block][D], then a D-float buffer a warp
    __shared__ float swarp[kAppendWarps];
    __shared__ int ssum[D];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float* buf = rows + (size_t) min(kKvBlock, B.max_new) * D + warp * D;
    grid_launch_dependents();
    grid_dependency_wait();

    if ((int) blockIdx.x >= kv_items) {                           // query rows: R.heads heads of one token a warp, U in flight
        const long long job = (long long) (blockIdx.x - kv_items) * kAppendWarps + warp;
        const int of = (R.n_q + R.heads - 1) / R.heads, n = (int) (job / of), h0 = (int) (job % of) * R.heads, h1 = min(h0 + R.heads, R.n_q);
        if (n >= B.n_tokens) return;
        int pos;
        if (R.pos != nullptr) pos = R.pos[n];
        else {
            const Seq s = seq_of(B, seq_of_row(B, n));
            pos = s.len - s.n_new + (n - s.row);
        }
        float w[V];
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = R.q_w != nullptr ? R.q_w[lane * V + i] : 1.0f;
        Turn<D> T;
        if (R.rot > 0) T.at(R, pos, lane);
        for (int h = h0; h < h1; h += U) {
            float x[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (h + u < h1) ld_acts<BF16, V>(R.q, (size_t) n * R.ld_q + (size_t) (h + u) * D + lane * V, R.wide_q, x[u]);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (h + u < h1) {
                    norm_rotate<D>(x[u], R.q_w != nullptr, w, R, T, buf, lane);
                    st_acts<V, BF16>(R.q_out, ((size_t) n * R.n_q + h + u) * D + lane * V, x[u], R.wide_out);
                }
        }
        return;
    }

    int item = blockIdx.x;
    const bool val = item & 1;
    item >>= 1;
    const int h = item % C.n_kv;
    item /= C.n_kv;
    const int j = item % touched, si = item / touched;
    const Seq s = seq_of(B, si);
    const int first = s.len - s.n_new;                            // position of the first new token (below 0: those have no place)
    const int lb = max(first, 0) / kKvBlock + j;
    if (s.n_new == 0 || lb * kKvBlock >= s.len) return;
    const int t0 = max(max(first, 0) - lb * kKvBlock, 0), t1 = min(s.len - lb * kKvBlock, kKvBlock);   // new tokens of the block
    float wk[V];
#pragma unroll
    for (int i = 0; i < V; ++i) wk[i] = !val && R.k_w != nullptr ? R.k_w[lane * V + i] : 1.0f;
    const int phys = block_of(C, si, lb);
    const size_t bh = (size_t) max(phys, 0) * C.n_kv + h;
    uint8_t* codes = (val ? C.v : C.k) + bh * (size_t) (kKvBlock * D);
    float* scale = (val ? C.v_scale : C.k_scale) + bh;
    const float s0 = t0 > 0 && phys >= 0 ? *scale : 0.0f;
    // keys: [D / 64][64 tokens][64 values], a word is 4 values of a token, a thread's are of the same four
    constexpr int quads = D / 4, step = kAppendThreads / quads, held = FEW ? (kKvBlock + step - 1) / step : 1;
    const int dq = tid % quads * 4;
    uint8_t* k_at = codes + (dq / 64) * (kKvBlock * 64) + (dq % 64);
    uint32_t old[held];
    if (FEW && !val && phys >= 0 && C.k_sum != nullptr && tid < step * quads)
#pragma unroll
        for (int i = 0; i < held; ++i) old[i] = tid / quads + i * step < t0 ? *(const uint32_t*) (k_at + (tid / quads + i * step) * 64) : 0u;
    // rows (U of a warp in flight), and the largest value
    float amax = 0.0f;
    for (int t = t0 + warp; t < t1; t += U * kAppendWarps) {
        float x[U][V];
        Turn<D> T[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int at = lb * kKvBlock + t + u * kAppendWarps, n = s.row + at - first;
            if (t + u * kAppendWarps >= t1) continue;
            if (val) ld_acts<BF16, V>(R.v, (size_t) n * R.ld_v + (size_t) h * D + lane * V, R.wide_v, x[u]);
            else {
                ld_acts<BF16, V>(R.k, (size_t) n * R.ld_k + (size_t) h * D + lane * V, R.wide_k, x[u]);
                if (R.rot > 0) T[u].at(R, R.pos != nullptr ? R.pos[n] : at, lane);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (t + u * kAppendWarps >= t1) continue;
            if (!val) norm_rotate<D>(x[u], R.k_w != nullptr, wk, R, T[u], buf, lane);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                amax = fmaxf(amax, fabsf(x[u][i]));
                rows[(t + u * kAppendWarps - t0) * D + lane * V + i] = x[u][i];
            }
        }
    }
    amax = warp_max(amax);
    if (lane == 0) swarp[warp] = amax;
    for (int d = tid; d < D; d += kAppendThreads) ssum[d] = 0;
    __syncthreads();
    if (phys < 0) return;
#pragma unroll
    for (int i = 0; i < kAppendWarps; ++i) amax = fmaxf(amax, swarp[i]);
    const float s1 = fmaxf(s0, amax > 0.0f ? fmaxf(kScaleLeast, fminf(amax * kInv127, kScaleMost)) : 0.0f), inv = s1 > 0.0f ? __fdiv_rn(1.0f, s1) : 0.0f;
    const bool grew = t0 > 0 && s1 > s0;
    const float ratio = grew ? __fdiv_rn(s0, s1) : 1.0f;

    if (!val) {
        int sum[4] = {0, 0, 0, 0};
        if (tid < step * quads) {
            // k_sum is made from the codes each time: tokens that were taken back (a shorter kv_len than before) are in no sum
            auto one = [&](int t, uint32_t w) {
                uint32_t r = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int c = grew ? code_moved((w >> (8 * e)) & 255u, ratio) : (int) ((w >> (8 * e)) & 255u) - 128;
                    r |= (uint32_t) (c + 128) << (8 * e);
                    sum[e] += c;
                }
                if (grew) *(uint32_t*) (k_at + t * 64) = r;
            };
            if (FEW && C.k_sum != nullptr) {
#pragma unroll
                for (int i = 0; i < held; ++i)
                    if (tid / quads + i * step < t0) one(tid / quads + i * step, old[i]);
            } else if (grew || C.k_sum != nullptr) {
#pragma unroll 4
                for (int t = tid / quads; t < t0; t += step) one(t, *(const uint32_t*) (k_at + t * 64));
            }
            for (int t = t0 + tid / quads; t < t1; t += step) {
                const float4 y = *(const float4*) (rows + (t - t0) * D + dq);
                const int c[4] = {code_of(y.x, inv), code_of(y.y, inv), code_of(y.z, inv), code_of(y.w, inv)};
                uint32_t r = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    r |= (uint32_t) (c[e] + 128) << (8 * e);
                    sum[e] += c[e];
                }
                *(uint32_t*) (k_at + t * 64) = r;
            }
            if (C.k_sum != nullptr)
#pragma unroll
                for (int e = 0; e < 4; ++e) atomicAdd(&ssum[dq + e], sum[e]);
        }
        __syncthreads();
        if (C.k_sum != nullptr)
            for (int x = tid; x < D; x += kAppendThreads) C.k_sum[bh * D + x] = (int16_t) ssum[x];
    } else {                                                      // [D][64 tokens]: neighbours have neighbouring values, 16 tokens of each
        const int g0 = grew ? 0 : t0 / 16, g1 = (t1 + 15) / 16;
        for (int i = tid; i < D * (g1 - g0); i += kAppendThreads) {
            const int d = i % D, t = (g0 + i / D) * 16;
            uint32_t* p = (uint32_t*) (codes + d * kKvBlock + t);
            if (t >= t0 && t + 16 <= t1) {
                uint4 r;
                uint32_t* rw = (uint32_t*) &r;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    rw[w] = 0;
#pragma unroll
                    for (int e = 0; e < 4; ++e) rw[w] |= (uint32_t) (code_of(rows[(t + 4 * w + e - t0) * D + d], inv) + 128) << (8 * e);
                }
                *(uint4*) p = r;
                continue;
            }
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const int tw = t + 4 * w;
                if (tw >= t1 || (tw + 4 <= t0 && !grew)) continue;
                uint32_t r = tw < t0 || tw + 4 > t1 ? p[w] : 0u;  // codes of others in the word
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at = tw + e;
                    if (at >= t1 || (at < t0 && !grew)) continue;
                    const int c = at < t0 ? code_moved((r >> (8 * e)) & 255u, ratio) : code_of(rows[(at - t0) * D + d], inv);
                    r = (r & ~(255u << (8 * e))) | (uint32_t) (c + 128) << (8 * e);
                }
                p[w] = r;
            }
        }
    }
    if (tid == 0 && (t0 == 0 || grew)) *scale = s1;
}

template<int D, bool BF16, bool FEW>
int launch_form(const maya_kv_cache& c, const maya_attn_batch& b, const maya_rope_args& a, cudaStream_t s) {
    constexpr int es = BF16 ? 2 : 4, kAppendThreads = Form<FEW>::threads, kAppendWarps = Form<FEW>::warps;
    // heads a warp: as many as leave every SM two dozen warps, so that a token's angles are read once for them
    int heads = 16;
    while (heads > 1 && (long long) b.n_tokens * ((a.n_q + heads - 1) / heads) < 24ll * sm_count()) heads /= 2;
    const RopeView R{a.q, a.k, a.v, a.ld_q, a.ld_k, a.ld_v, a.n_q, a.q_w, a.k_w, a.eps, a.cos, a.sin, a.pos, a.n_pos, a.rot_dim, a.pairs,
                     a.q_out, rows_wide(a.q, a.ld_q, es), rows_wide(a.k, a.ld_k, es), rows_wide(a.v, a.ld_v, es), aligned16(a.q_out), heads};
    const int touched = a.k ? (b.max_new + kKvBlock - 2) / kKvBlock + 1 : 0;     // blocks that max_new tokens fall into at most
    const long long kv_items = (long long) b.n_seq * touched * c.n_kv * 2;
    const long long q_blocks = ((long long) b.n_tokens * ((a.n_q + heads - 1) / heads) + kAppendWarps - 1) / kAppendWarps;
    if (kv_items + q_blocks > 0x7fffffffll) return refuse(MAYA_ERR_LIMIT);
    const size_t smem = ((size_t) (b.max_new < kKvBlock ? b.max_new : kKvBlock) + kAppendWarps) * D * sizeof(float);
    static SmemLimit limit;
    if (smem > kSmemNoLimit && !limit.raise((const void*) append_kernel<D, BF16, FEW>, kSmemMost)) return note_launch("kv append smem attribute");
    launch_dependent(append_kernel<D, BF16, FEW>, dim3((unsigned) (kv_items + q_blocks)), dim3(kAppendThreads), smem, s, kv_view(c), batch_view(b), R,
                     touched, (int) kv_items);
    return note_launch("qk_norm_rope_append");
}
template<int D, bool BF16>
int launch_append(const maya_kv_cache& c, const maya_attn_batch& b, const maya_rope_args& a, cudaStream_t s) {
    return b.max_new <= 4 ? launch_form<D, BF16, true>(c, b, a, s) : launch_form<D, BF16, false>(c, b, a, s);
}

// ---------------------------------------------------------------- blocks as values
// A thread block is one (block, head).  All its codes are asked for at once, 16 bytes a load; keys are rows already, values turn through shared memory, four
// tokens of four values at a time.
template<int D, bool BF16>
__global__ void __launch_bounds__(256) read_kernel(const KvView C, const int* blocks, const int* counts, void* k_out, void* v_out, void* mean) {
    constexpr int wide = kKvBlock + 4, loads = kKvBlock * D / 16 / 256;
    __shared__ __align__(16) uint8_t vt[D * wide];
    const int i = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
    grid_launch_dependents();
    grid_dependency_wait();
    const int phys = blocks[i];
    const bool real = phys >= 0 && phys < C.n_blocks;
    const int count = real ? counts != nullptr ? max(0, min(counts[i], kKvBlock)) : kKvBlock : 0;
    const size_t bh = real ? (size_t) phys * C.n_kv + h : 0;
    uint4 kw[loads], vw[loads];
#pragma unroll
    for (int x = 0; x < loads; ++x) {
        kw[x] = vw[x] = make_uint4(0u, 0u, 0u, 0u);
        if (real && k_out != nullptr) kw[x] = ((const uint4*) (C.k + bh * (size_t) (kKvBlock * D)))[x * 256 + tid];
        if (real && v_out != nullptr) vw[x] = ((const uint4*) (C.v + bh * (size_t) (kKvBlock * D)))[x * 256 + tid];
    }
    const float ks = real ? C.k_scale[bh] : 0.0f, vs = real ? C.v_scale[bh] : 0.0f;
    auto put = [&](void* out, int t, int d, uint32_t w, float s) {           // 4 values of token t
        const size_t at = (((size_t) i * kKvBlock + t) * C.n_kv + h) * D + d;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = t < count ? (float) ((int) ((w >> (8 * e)) & 255u) - 128) * s : 0.0f;
        st_acts<4, BF16>(out, at, x, true);
    };
    if (v_out != nullptr)
#pragma unroll
        for (int x = 0; x < loads; ++x) {                                    // 16 tokens of value d
            const int at = x * 256 + tid, d = at / 4, t = at % 4 * 16;
            uint32_t* to = (uint32_t*) (vt + d * wide + t);
            to[0] = vw[x].x; to[1] = vw[x].y; to[2] = vw[x].z; to[3] = vw[x].w;
        }
    if (k_out != nullptr)
#pragma unroll
        for (int x = 0; x < loads; ++x) {                                    // 16 values of token t
            const int at = x * 256 + tid, t = at / 4 % kKvBlock, d = at / (4 * kKvBlock) * 64 + at % 4 * 16;
            put(k_out, t, d, kw[x].x, ks); put(k_out, t, d + 4, kw[x].y, ks); put(k_out, t, d + 8, kw[x].z, ks); put(k_out, t, d + 12, kw[x].w, ks);
        }
    if (v_out != nullptr) {
        __syncthreads();
        for (int x = tid; x < kKvBlock * D / 16; x += 256) {                 // tokens t .. t + 3 of values d .. d + 3
            const int d = x % (D / 4) * 4, t = x / (D / 4) * 4;
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) w[e] = *(const uint32_t*) (vt + (d + e) * wide + t);
            const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140), c = __byte_perm(w[0], w[1], 0x7362), e = __byte_perm(w[2], w[3], 0x7362);
            put(v_out, t, d, __byte_perm(a, b, 0x5410), vs);
            put(v_out, t + 1, d, __byte_perm(a, b, 0x7632), vs);
            put(v_out, t + 2, d, __byte_perm(c, e, 0x5410), vs);
            put(v_out, t + 3, d, __byte_perm(c, e, 0x7632), vs);
        }
    }
    if (mean != nullptr)
        for (int d = tid; d < D; d += 256)
            st_act<BF16>(mean, ((size_t) i * C.n_kv + h) * D + d,
                         count > 0 ? __fdiv_rn((float) C.k_sum[bh * D + d] * ks, (float) count) : 0.0f);
}

template<int D, bool BF16>
int launch_read(const maya_kv_cache& c, const int32_t* blocks, const int32_t* counts, int n, void* k, void* v, void* mean, cudaStream_t s) {
    launch_dependent(read_kernel<D, BF16>, dim3((unsigned) n, (unsigned) c.n_kv), dim3(256), 0, s, kv_view(c), blocks, counts, k, v, mean);
    return note_launch("kv_read");
}

}  // namespace
}  // namespace maya

using namespace maya;

#define KV_BY_DIM(D, CALL)                 \
    switch (D) {                           \
        case 64: return CALL(64);          \
        case 128: return CALL(128);        \
        case 192: return CALL(192);        \
        default: return CALL(256);         \
    }

extern "C" int maya_qk_norm_rope_append(const maya_kv_cache* c, const maya_attn_batch* b, const maya_rope_args* a, void* stream) {
    int st = kv_check(c);
    if (st == MAYA_OK) st = batch_check(c, b);
    if (st == MAYA_OK && !a) st = MAYA_ERR_ARG;
    if (st != MAYA_OK) return refuse(st);
    if (b->n_tokens == 0) return MAYA_OK;
    if (!a->q || !a->q_out || a->n_q <= 0 || (a->k == nullptr) != (a->v == nullptr) || !(a->eps >= 0.0f)) return refuse(MAYA_ERR_ARG);
    if (a->rot_dim < 0 || a->rot_dim % 2 != 0 || a->rot_dim > c->head_dim) return refuse(MAYA_ERR_ARG);
    if (a->rot_dim > 0 && (!a->cos || !a->sin || a->n_pos <= 0)) return refuse(MAYA_ERR_ARG);
    if (a->ld_q < (int64_t) a->n_q * c->head_dim) return refuse(MAYA_ERR_ARG);
    if (a->k && (a->ld_k < (int64_t) c->n_kv * c->head_dim || a->ld_v < (int64_t) c->n_kv * c->head_dim)) return refuse(MAYA_ERR_ARG);
    if (a->q_out == a->q && a->ld_q != (int64_t) a->n_q * c->head_dim) return refuse(MAYA_ERR_ARG);
    cudaStream_t s = as_stream(stream);
#define APPEND(D) a->is_bf16 ? launch_append<D, true>(*c, *b, *a, s) : launch_append<D, false>(*c, *b, *a, s)
    KV_BY_DIM(c->head_dim, APPEND)
#undef APPEND
}

extern "C" int maya_kv_read(const maya_kv_cache* c, const int32_t* blocks, const int32_t* counts, int n, int out_is_bf16, void* k, void* v,
                            void* mean, void* stream) {
    const int st = kv_check(c);
    if (st != MAYA_OK) return refuse(st);
    if (n == 0) return MAYA_OK;
    if (!blocks || n < 0 || (mean && !c->k_sum) || (k && !aligned16(k)) || (v && !aligned16(v))) return refuse(MAYA_ERR_ARG);
    if (c->n_kv > 65535) return refuse(MAYA_ERR_LIMIT);
    if (!k && !v && !mean) return MAYA_OK;
    cudaStream_t s = as_stream(stream);
#define READ(D) out_is_bf16 ? launch_read<D, true>(*c, blocks, counts, n, k, v, mean, s) : launch_read<D, false>(*c, blocks, counts, n, k, v, mean, s)
    KV_BY_DIM(c->head_dim, READ)
#undef READ
}
