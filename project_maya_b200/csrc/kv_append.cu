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
// queries written, a byte a value into the cache.
#include "maya_kv.cuh"

namespace maya {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / 32;

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
    int wide_q, wide_k, wide_v;
};

// One head's row, V = D / 32 consecutive values a lane: the norm, then the rotation (partners change lanes through `buf`, D
// floats of this warp's own).
template<int D>
__device__ __forceinline__ void norm_rotate(float (&x)[D / 32], const float* w, const RopeView& R, int pos, float* buf, int lane) {
    constexpr int V = D / 32;
    if (w != nullptr) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) ss += x[i] * x[i];
        ss = warp_sum(ss);
        const float inv = rsqrtf(ss * (1.0f / D) + R.eps);
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = x[i] * inv * w[lane * V + i];
    }
    if (R.rot == 0) return;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < V; ++i) buf[lane * V + i] = x[i];
    __syncwarp();
    const int half = R.rot >> 1;
    const size_t row = (size_t) max(0, min(pos, R.n_pos - 1)) * half;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int d = lane * V + i;
        if (d >= R.rot) continue;
        const int j = R.pairs ? d >> 1 : d < half ? d : d - half;             // the angle
        const bool second = R.pairs ? d & 1 : d >= half;
        const float c = __ldg(R.cos + row + j), s = __ldg(R.sin + row + j);
        const float other = buf[R.pairs ? d ^ 1 : second ? d - half : d + half];
        x[i] = second ? x[i] * c + other * s : x[i] * c - other * s;
    }
}

// A value as its code: nearest, +-127, NaN 0.
__device__ __forceinline__ int code_of(float x, float scale) {
    if (!(scale > 0.0f)) return 0;
    const float r = rintf(__fdiv_rn(x, scale));
    return r == r ? (int) fmaxf(-127.0f, fminf(127.0f, r)) : 0;
}
__device__ __forceinline__ int code_moved(uint32_t code, float ratio) { return (int) rintf((float) ((int) code - 128) * ratio); }

template<int D, bool BF16>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const KvView C, const BatchView B, const RopeView R, int touched, int kv_items) {
    constexpr int V = D / 32;
    extern __shared__ __align__(16) float rows[];                 // [tokens of the block][D], then a D-float buffer a warp
    __shared__ float swarp[kAppendWarps];
    __shared__ int ssum[D];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    grid_launch_dependents();
    grid_dependency_wait();
    float* buf = rows + (size_t) min(kKvBlock, B.max_new) * D + warp * D;

    if ((int) blockIdx.x >= kv_items) {                           // query rows
        const long long row = (long long) (blockIdx.x - kv_items) * kAppendWarps + warp;
        if (row >= (long long) B.n_tokens * R.n_q) return;
        const int n = (int) (row / R.n_q), h = (int) (row % R.n_q);
        int pos;
        if (R.pos != nullptr) pos = R.pos[n];
        else {
            const Seq s = seq_of(B, seq_of_row(B, n));
            pos = s.len - s.n_new + (n - s.row);
        }
        float x[V];
        ld_acts<BF16, V>(R.q, (size_t) n * R.ld_q + (size_t) h * D + lane * V, R.wide_q, x);
        norm_rotate<D>(x, R.q_w, R, pos, buf, lane);
#pragma unroll
        for (int i = 0; i < V; ++i) st_act<BF16>(R.q_out, (size_t) row * D + lane * V + i, x[i]);
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
    const int phys = block_of(C, si, lb);
    if (phys < 0) return;
    const int t0 = max(max(first, 0) - lb * kKvBlock, 0), t1 = min(s.len - lb * kKvBlock, kKvBlock);   // new tokens of the block
    const size_t bh = (size_t) phys * C.n_kv + h;
    float* scale = (val ? C.v_scale : C.k_scale) + bh;
    const float s0 = t0 > 0 ? *scale : 0.0f;

    float amax = 0.0f;
    for (int t = t0 + warp; t < t1; t += kAppendWarps) {
        const int at = lb * kKvBlock + t, n = s.row + at - first;
        float x[V];
        if (val) ld_acts<BF16, V>(R.v, (size_t) n * R.ld_v + (size_t) h * D + lane * V, R.wide_v, x);
        else {
            ld_acts<BF16, V>(R.k, (size_t) n * R.ld_k + (size_t) h * D + lane * V, R.wide_k, x);
            norm_rotate<D>(x, R.k_w, R, R.pos != nullptr ? R.pos[n] : at, buf, lane);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            amax = fmaxf(amax, fabsf(x[i]));
            rows[(t - t0) * D + lane * V + i] = x[i];
        }
    }
    amax = warp_max(amax);
    if (lane == 0) swarp[warp] = amax;
    for (int d = tid; d < D; d += kAppendThreads) ssum[d] = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kAppendWarps; ++i) amax = fmaxf(amax, swarp[i]);
    const float s1 = fmaxf(s0, fminf(amax * kInv127, kScaleMost));
    const bool grew = t0 > 0 && s1 > s0;
    const float ratio = grew ? __fdiv_rn(s0, s1) : 1.0f;
    uint8_t* codes = (val ? C.v : C.k) + bh * (size_t) (kKvBlock * D);

    if (!val) {                                                   // [D / 64][64 tokens][64 values]: a word is 4 values of a token
        // k_sum is made from the codes each time: tokens that were taken back (a shorter kv_len than before) are in no sum
        for (int i = tid; i < (grew || C.k_sum != nullptr ? t0 : 0) * (D / 4); i += kAppendThreads) {
            const int t = i / (D / 4), d = (i % (D / 4)) * 4;
            uint32_t* p = (uint32_t*) (codes + (d / 64) * (kKvBlock * 64) + t * 64 + (d % 64));
            const uint32_t w = *p;
            uint32_t r = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = grew ? code_moved((w >> (8 * e)) & 255u, ratio) : (int) ((w >> (8 * e)) & 255u) - 128;
                r |= (uint32_t) (c + 128) << (8 * e);
                atomicAdd(&ssum[d + e], c);
            }
            if (grew) *p = r;
        }
        for (int i = tid; i < (t1 - t0) * (D / 4); i += kAppendThreads) {
            const int t = i / (D / 4), d = (i % (D / 4)) * 4;
            uint32_t r = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = code_of(rows[t * D + d + e], s1);
                r |= (uint32_t) (c + 128) << (8 * e);
                atomicAdd(&ssum[d + e], c);
            }
            *(uint32_t*) (codes + (d / 64) * (kKvBlock * 64) + (t0 + t) * 64 + (d % 64)) = r;
        }
        __syncthreads();
        if (C.k_sum != nullptr)
            for (int d = tid; d < D; d += kAppendThreads) C.k_sum[bh * D + d] = (int16_t) ssum[d];
    } else {                                                      // [D][64 tokens]: a word is 4 tokens of a value
        const int w0 = grew ? 0 : t0 / 4, w1 = (t1 + 3) / 4, nw = w1 - w0;
        for (int i = tid; i < D * nw; i += kAppendThreads) {
            const int d = i / nw, t = (w0 + i % nw) * 4;
            uint8_t* p = codes + d * kKvBlock + t;
            uint32_t r = t < t0 || t + 4 > t1 ? *(const uint32_t*) p : 0u;       // codes of others in the word
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int at = t + e;
                if (at >= t1 || (at < t0 && !grew)) continue;
                const int c = at < t0 ? code_moved((r >> (8 * e)) & 255u, ratio) : code_of(rows[(at - t0) * D + d], s1);
                r = (r & ~(255u << (8 * e))) | (uint32_t) (c + 128) << (8 * e);
            }
            *(uint32_t*) p = r;
        }
    }
    if (tid == 0 && (t0 == 0 || grew)) *scale = s1;
}

template<int D, bool BF16>
int launch_append(const maya_kv_cache& c, const maya_attn_batch& b, const maya_rope_args& a, cudaStream_t s) {
    constexpr int es = BF16 ? 2 : 4;
    const RopeView R{a.q, a.k, a.v, a.ld_q, a.ld_k, a.ld_v, a.n_q, a.q_w, a.k_w, a.eps, a.cos, a.sin, a.pos, a.n_pos, a.rot_dim, a.pairs,
                     a.q_out, rows_wide(a.q, a.ld_q, es), rows_wide(a.k, a.ld_k, es), rows_wide(a.v, a.ld_v, es)};
    const int touched = a.k ? (b.max_new + kKvBlock - 2) / kKvBlock + 1 : 0;     // blocks that max_new tokens fall into at most
    const long long kv_items = (long long) b.n_seq * touched * c.n_kv * 2;
    const long long q_blocks = ((long long) b.n_tokens * a.n_q + kAppendWarps - 1) / kAppendWarps;
    if (kv_items + q_blocks > 0x7fffffffll) return refuse(MAYA_ERR_LIMIT);
    const size_t smem = ((size_t) (b.max_new < kKvBlock ? b.max_new : kKvBlock) + kAppendWarps) * D * sizeof(float);
    static SmemLimit limit;
    if (smem > kSmemNoLimit && !limit.raise((const void*) append_kernel<D, BF16>, kSmemMost)) return note_launch("kv append smem attribute");
    launch_dependent(append_kernel<D, BF16>, dim3((unsigned) (kv_items + q_blocks)), dim3(kAppendThreads), smem, s, kv_view(c), batch_view(b), R,
                     touched, (int) kv_items);
    return note_launch("qk_norm_rope_append");
}

// ---------------------------------------------------------------- blocks as values
// A thread block is one (block, head): keys are rows already; values turn through shared memory.
template<int D, bool BF16>
__global__ void __launch_bounds__(256) read_kernel(const KvView C, const int* blocks, const int* counts, void* k_out, void* v_out, void* mean) {
    __shared__ __align__(16) uint8_t vt[D * (kKvBlock + 4)];
    const int i = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
    grid_launch_dependents();
    grid_dependency_wait();
    const int phys = blocks[i];
    const bool real = phys >= 0 && phys < C.n_blocks;
    const int count = real ? counts != nullptr ? max(0, min(counts[i], kKvBlock)) : kKvBlock : 0;
    const size_t bh = real ? (size_t) phys * C.n_kv + h : 0;
    const float ks = count > 0 ? C.k_scale[bh] : 0.0f, vs = count > 0 ? C.v_scale[bh] : 0.0f;
    auto put = [&](void* out, int t, int d, uint32_t w, float s) {           // 4 values of token t
        const size_t at = (((size_t) i * kKvBlock + t) * C.n_kv + h) * D + d;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = t < count ? (float) ((int) ((w >> (8 * e)) & 255u) - 128) * s : 0.0f;
        if constexpr (BF16) {
            const __nv_bfloat162 a = __floats2bfloat162_rn(x[0], x[1]), b = __floats2bfloat162_rn(x[2], x[3]);
            *(uint2*) ((uint16_t*) out + at) = make_uint2(*(const uint32_t*) &a, *(const uint32_t*) &b);
        } else {
            *(float4*) ((float*) out + at) = make_float4(x[0], x[1], x[2], x[3]);
        }
    };
    if (k_out != nullptr) {
        const uint8_t* codes = C.k + bh * (size_t) (kKvBlock * D);
        for (int w = tid; w < kKvBlock * D / 4; w += 256) {
            const int t = w / (D / 4), d = (w % (D / 4)) * 4;
            put(k_out, t, d, t < count ? *(const uint32_t*) (codes + (d / 64) * (kKvBlock * 64) + t * 64 + (d % 64)) : 0u, ks);
        }
    }
    if (v_out != nullptr) {
        const uint8_t* codes = C.v + bh * (size_t) (kKvBlock * D);
        if (count > 0)
            for (int w = tid; w < kKvBlock * D / 4; w += 256)
                *(uint32_t*) (vt + (w / 16) * (kKvBlock + 4) + (w % 16) * 4) = ((const uint32_t*) codes)[w];
        __syncthreads();
        for (int w = tid; w < kKvBlock * D / 4; w += 256) {
            const int t = w / (D / 4), d = (w % (D / 4)) * 4;
            uint32_t r = 0;
            if (t < count)
#pragma unroll
                for (int e = 0; e < 4; ++e) r |= (uint32_t) vt[(d + e) * (kKvBlock + 4) + t] << (8 * e);
            put(v_out, t, d, r, vs);
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
