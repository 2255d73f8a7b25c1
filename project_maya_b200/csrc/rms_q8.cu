// rms_q8.cu - what stands in front of a product: residual add, RMS norm and the rounding of the normed rows to 8 bits with scales, in one
// launch; and the 8-bit rows read back as the values they stand for.
//
// Reference counterpart: glmf::rms_q8 (include/strata/kernels/glm_fast.hpp:534, src/kernels/cuda/glm_fast.cu:5669-5697) for one f32 token
// and q8_1 blocks; here any number of rows, bf16 rows, and the prompt path's image as well.
//
//   t = h + add                            f32; h_out = t, rounded once when the stream is bf16
//   x = t * (1 / sqrt(mean(t^2) + eps)) * w   f32, of the unrounded t; x_out rounded once
//   xq = x as maya_quantize_q8_1 or maya_mmq_quantize rounds it, byte for byte
//
// Bounds: a prompt is bytes (4096 x 6144 f32 rows with add and h_out into the image: 66 us, 5.4 TB/s of the 354 MB it moves; with streaming loads and stores 65, with
// two runs a thread instead of four 68), a token one launch with its chain of loads, reduction and stores (3 us, 2 more to read it back).
//
// One thread block a row.  A thread holds runs of 8 consecutive values (32 bytes of f32: two 16-byte loads) in registers across the
// reduction, so the row is read once; four neighbouring lanes hold a 32-value group, whose amax is two shuffles away.  The group's sum keeps
// the quantizers' order of additions - theirs is a butterfly over single values, distances 16, 8, 4, 2, 1, here the first two between lanes and the
// rest inside one - so that the bytes are those of the separate launches.
#include "maya_mmq_image.cuh"

namespace maya {
namespace {

struct RmsRows {
    const void* h;
    const void* add;
    const float* w;
    void* h_out;
    void* x_out;
    uint8_t* xq;
    int64_t ld_h, ld_add, ld_h_out, ld_x;
    int n;
    float eps;
    int add_is_bf16, x_is_bf16, image;
};

constexpr int kRunsMost = 8;                       // runs of 8 values a thread holds at most
constexpr int kRmsWarpsMost = 32;
constexpr int kRmsMost = 32768;                    // values of a row: 512 threads of 8 runs

__device__ __forceinline__ float bf16_at(const void* p, int64_t i) { return __uint_as_float((uint32_t) ((const uint16_t*) p)[i] << 16); }
__device__ __forceinline__ uint32_t bf16_pair(float a, float b) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
    return r;
}
__device__ __forceinline__ void load8(const void* p, int64_t at, bool bf16, float (&v)[8]) {
    if (bf16) {
        const uint4 u = *(const uint4*) ((const uint16_t*) p + at);
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u); }
    } else {
        const float4 a = *(const float4*) ((const float*) p + at), b = *(const float4*) ((const float*) p + at + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
}
__device__ __forceinline__ void store8(void* p, int64_t at, bool bf16, const float (&v)[8]) {
    if (bf16) {
        *(uint4*) ((uint16_t*) p + at) = make_uint4(bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7]));
    } else {
        *(float4*) ((float*) p + at) = make_float4(v[0], v[1], v[2], v[3]);
        *(float4*) ((float*) p + at + 4) = make_float4(v[4], v[5], v[6], v[7]);
    }
}

// 8 values of a 32-value group to its q8_1 block (blk: the block; part: which of its four runs).  Every lane of the warp calls.
__device__ __forceinline__ void q8_1_run(const float (&v)[8], uint8_t* blk, int part, bool live) {
    float amax = fabsf(v[0]);                    // (not 0: a group of nothing but NaN has no largest value)
#pragma unroll
    for (int i = 1; i < 8; ++i) amax = fmaxf(amax, fabsf(v[i]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    float s[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] = v[i] + __shfl_xor_sync(0xffffffffu, v[i], 2);        // values 16 apart
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] += __shfl_xor_sync(0xffffffffu, s[i], 1);              // 8 apart
    const float sum = ((s[0] + s[4]) + (s[2] + s[6])) + ((s[1] + s[5]) + (s[3] + s[7]));    // 4, 2, 1
    const float d = fminf(__fdiv_rn(amax, 127.0f), 65504.0f);
    uint32_t q[2] = {0u, 0u};
    if (amax != 0.0f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = (int) fmaxf(-127.0f, fminf(127.0f, roundf(__fdiv_rn(v[i], d))));
            q[i >> 2] |= (uint32_t) (c & 0xFF) << (8 * (i & 3));
        }
    }
    if (!live) return;
    *(uint32_t*) (blk + 4 + 8 * part) = q[0];
    *(uint32_t*) (blk + 8 + 8 * part) = q[1];
    if (part == 0) *(__half2*) blk = __floats2half2_rn(d, fmaxf(-65504.0f, fminf(65504.0f, sum)));
}

// Run c (values 8 c ..) of row `row` to the 8-bit image.  Every lane of the warp calls; live: the run exists.
__device__ __forceinline__ void emit_run(const RmsRows& A, int64_t row, int c, const float (&x)[8], bool live) {
    if (A.image == MAYA_XQ_Q8_1) {
        q8_1_run(x, A.xq + (row * (A.n >> 5) + (c >> 2)) * kQ81Bytes, c & 3, live);
    } else if (A.image == MAYA_XQ_MMQ) {
        uint32_t o[4];
        const __half xa = q8_1_round8(x, o);
        if (!live) return;
        __half* d = (__half*) A.xq + row * xq_ld(A.n);
        *(uint4*) (d + (int64_t) c * 8) = make_uint4(o[0], o[1], o[2], o[3]);
        if ((c & 3) == 0) d[A.n + (c >> 2)] = xa;
    }
}
// The zeros behind a row's sum corrections.
__device__ __forceinline__ void pad_image(const RmsRows& A, int64_t row, int tid) {
    if (A.image != MAYA_XQ_MMQ) return;
    __half* d = (__half*) A.xq + row * xq_ld(A.n) + A.n;
    for (int i = A.n / 32 + tid; i < (int) xq_tail(A.n); i += blockDim.x) d[i] = __float2half_rn(0.0f);
}

// (never contracted into the sums behind it: the quantizers round the x that is stored)
__device__ __forceinline__ float scaled(float t, float inv, float w) { return __fmul_rn(__fmul_rn(t, inv), w); }

__device__ __forceinline__ float block_sum(float v, float* s, int tid, int nt) {
    v = warp_sum(v);
    if ((tid & 31) == 0) s[tid >> 5] = v;
    __syncthreads();
    float tot = 0.0f;
    for (int i = 0; i < nt >> 5; ++i) tot += s[i];
    return tot;
}

// HB: h and h_out are bf16.  R: runs a thread holds.  Everything 16-byte aligned, n a multiple of 8 (of 32 with an image).
template<bool HB, int R>
__global__ void __launch_bounds__(R > 2 ? 512 : 1024) rms_q8_kernel(const RmsRows A) {
    __shared__ float sred[kRmsWarpsMost];
    const int tid = threadIdx.x, nt = blockDim.x, runs = A.n >> 3;
    const int64_t row = blockIdx.x;
    grid_launch_dependents();
    for (int e = tid * 32; e < A.n; e += nt * 32) asm volatile("prefetch.global.L2 [%0];" ::"l"(A.w + e));
    grid_dependency_wait();
    float t[R][8];
    float ss = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = tid + r * nt;
#pragma unroll
        for (int i = 0; i < 8; ++i) t[r][i] = 0.0f;
        if (c < runs) load8(A.h, row * A.ld_h + c * 8, HB, t[r]);
    }
    if (A.add != nullptr) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int c = tid + r * nt;
            float a[8];
            if (c < runs) {
                load8(A.add, row * A.ld_add + c * 8, A.add_is_bf16 != 0, a);
#pragma unroll
                for (int i = 0; i < 8; ++i) t[r][i] += a[i];
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i) ss += t[r][i] * t[r][i];
    const float inv = rsqrtf(block_sum(ss, sred, tid, nt) / (float) A.n + A.eps);
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int c = tid + r * nt;
        if (c - (tid & 31) >= runs) break;               // the whole warp is behind the row's end
        const bool live = c < runs;
        float x[8];
        if (live) {
            if (A.h_out != nullptr) store8(A.h_out, row * A.ld_h_out + c * 8, HB, t[r]);
            load8(A.w, c * 8, false, x);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = live ? scaled(t[r][i], inv, x[i]) : 0.0f;
        if (live && A.x_out != nullptr) store8(A.x_out, row * A.ld_x + c * 8, A.x_is_bf16 != 0, x);
        emit_run(A, row, c, x, live);
    }
    pad_image(A, row, tid);
}

// Any alignment and any n: single elements, the row in shared memory.
template<bool HB>
__global__ void __launch_bounds__(512) rms_q8_any_kernel(const RmsRows A) {
    extern __shared__ __align__(16) float xs[];
    __shared__ float sred[kRmsWarpsMost];
    const int tid = threadIdx.x, nt = blockDim.x;
    const int64_t row = blockIdx.x;
    grid_launch_dependents();
    grid_dependency_wait();
    float ss = 0.0f;
    for (int e = tid; e < A.n; e += nt) {
        float t = HB ? bf16_at(A.h, row * A.ld_h + e) : ((const float*) A.h)[row * A.ld_h + e];
        if (A.add != nullptr) t += A.add_is_bf16 ? bf16_at(A.add, row * A.ld_add + e) : ((const float*) A.add)[row * A.ld_add + e];
        xs[e] = t;
        ss += t * t;
    }
    const float inv = rsqrtf(block_sum(ss, sred, tid, nt) / (float) A.n + A.eps);
    for (int e = tid; e < A.n; e += nt) {                // a thread's own elements
        const float t = xs[e], x = scaled(t, inv, A.w[e]);
        xs[e] = x;
        if (A.h_out != nullptr) {
            if (HB) ((uint16_t*) A.h_out)[row * A.ld_h_out + e] = (uint16_t) bf16_pair(t, 0.0f);
            else ((float*) A.h_out)[row * A.ld_h_out + e] = t;
        }
        if (A.x_out != nullptr) {
            if (A.x_is_bf16) ((uint16_t*) A.x_out)[row * A.ld_x + e] = (uint16_t) bf16_pair(x, 0.0f);
            else ((float*) A.x_out)[row * A.ld_x + e] = x;
        }
    }
    if (A.image == 0) return;
    __syncthreads();
    const int runs = A.n >> 3;
    for (int c0 = 0; c0 < runs; c0 += nt) {
        const int c = c0 + tid;
        const bool live = c < runs;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = live ? xs[c * 8 + i] : 0.0f;
        emit_run(A, row, c, x, live);
    }
    pad_image(A, row, tid);
}

// Threads and runs a thread, by rule: with no more rows than SMs a row's latency counts - as many threads as there are runs; with more, a
// row's blocks share an SM and a thread with four runs has eight (f32, with add: sixteen) loads in flight.
template<bool HB> int launch_rms(const RmsRows& A, int64_t rows, cudaStream_t s) {
    const int runs = A.n >> 3;
    const int least = rows <= sm_count() ? 1 : 4;
    int r = least;
    while ((runs + r - 1) / r > (r > 2 ? 512 : 1024)) r *= 2;
    const dim3 block((unsigned) (((runs + r - 1) / r + 31) & ~31)), grid((unsigned) rows);
    switch (r) {
        case 1: launch_dependent(rms_q8_kernel<HB, 1>, grid, block, 0, s, A); break;
        case 2: launch_dependent(rms_q8_kernel<HB, 2>, grid, block, 0, s, A); break;
        case 4: launch_dependent(rms_q8_kernel<HB, 4>, grid, block, 0, s, A); break;
        default: launch_dependent(rms_q8_kernel<HB, kRunsMost>, grid, block, 0, s, A); break;
    }
    return note_launch("rms_q8");
}
template<bool HB> int launch_rms_any(const RmsRows& A, int64_t rows, cudaStream_t s) {
    static SmemLimit limit;
    const size_t smem = (size_t) A.n * sizeof(float);
    if (smem > kSmemNoLimit && !limit.raise((const void*) rms_q8_any_kernel<HB>, kSmemMost)) return note_launch("rms_q8 smem attribute");
    launch_dependent(rms_q8_any_kernel<HB>, dim3((unsigned) rows), dim3(512), smem, s, A);
    return note_launch("rms_q8");
}

// Values and group sums of 8-bit rows.  A thread takes 8 values; four neighbours share a group.
template<bool MMQ, bool OB>
__global__ void __launch_bounds__(256) q8_read_kernel(const uint8_t* __restrict__ xq, int64_t n_runs, int n, void* __restrict__ values,
                                                      __half* __restrict__ sums) {
    const int64_t c = (int64_t) blockIdx.x * 256 + threadIdx.x;
    grid_launch_dependents();
    grid_dependency_wait();
    const bool live = c < n_runs;                        // (a multiple of 4: a group's lanes live together)
    float v[8] = {};
    float tail = 0.0f;
    if (live) {
        if constexpr (MMQ) {
            const int per = n >> 3;
            const int64_t row = c / per;
            const int at = (int) (c - row * per);
            const __half* p = (const __half*) xq + row * xq_ld(n);
            const uint4 u = *(const uint4*) (p + at * 8);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 f = __half22float2(*(const __half2*) &w[i]);
                v[2 * i] = f.x; v[2 * i + 1] = f.y;
            }
            tail = __half2float(p[n + (at >> 2)]);
        } else {
            const uint8_t* b = xq + (c >> 2) * kQ81Bytes;
            const __half2 ds = *(const __half2*) b;
            const float d = __low2float(ds);
            tail = __high2float(ds);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const uint32_t q = *(const uint32_t*) (b + 4 + 8 * (c & 3) + 4 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * i + j] = d * (float) (int8_t) (q >> (8 * j));
            }
        }
    }
    if constexpr (MMQ) {                                  // the image keeps the sum less that of the stored values, which is exact in f32
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += v[i];
        s += __shfl_xor_sync(0xffffffffu, s, 1);
        s += __shfl_xor_sync(0xffffffffu, s, 2);
        tail += s;
    }
    if (!live) return;
    if (values != nullptr) store8(values, c * 8, OB, v);
    if (sums != nullptr && (c & 3) == 0) sums[c >> 2] = __float2half_rn(tail);
}

}  // namespace
}  // namespace maya

using namespace maya;

extern "C" int maya_rms_q8(const maya_rms_args* a, void* stream) {
    if (!a) return refuse(MAYA_ERR_ARG);
    if (a->n_rows <= 0) return MAYA_OK;
    if (!a->h || !a->w || a->n <= 0 || !(a->eps >= 0.0f) || (!a->h_out && !a->x_out && !a->xq)) return refuse(MAYA_ERR_ARG);
    if (a->image != MAYA_XQ_NONE && a->image != MAYA_XQ_Q8_1 && a->image != MAYA_XQ_MMQ) return refuse(MAYA_ERR_ARG);
    if ((a->image != MAYA_XQ_NONE) != (a->xq != nullptr)) return refuse(MAYA_ERR_ARG);
    if (a->image != MAYA_XQ_NONE && (a->n % 32 || !aligned16(a->xq))) return refuse(MAYA_ERR_ARG);
    if (a->n > kRmsMost || a->n_rows > 0x7FFFFFFF) return refuse(MAYA_ERR_LIMIT);
    if (a->ld_h < a->n || (a->add && a->ld_add < a->n) || (a->h_out && a->ld_h_out < a->n) || (a->x_out && a->ld_x < a->n)) return refuse(MAYA_ERR_ARG);
    // in place where every thread writes what it has read itself: the same rows, the same type
    if (a->h_out && a->h_out == a->h && a->ld_h_out != a->ld_h) return refuse(MAYA_ERR_ARG);
    if (a->h_out && a->h_out == a->add && (a->ld_h_out != a->ld_add || !a->add_is_bf16 != !a->h_is_bf16)) return refuse(MAYA_ERR_ARG);
    if (a->x_out && (a->x_out == a->h_out || a->x_out == a->xq)) return refuse(MAYA_ERR_ARG);
    if (a->x_out && a->x_out == a->h && (a->ld_x != a->ld_h || !a->x_is_bf16 != !a->h_is_bf16)) return refuse(MAYA_ERR_ARG);
    if (a->x_out && a->x_out == a->add && (a->ld_x != a->ld_add || !a->x_is_bf16 != !a->add_is_bf16)) return refuse(MAYA_ERR_ARG);
    const RmsRows A{a->h, a->add, a->w, a->h_out, a->x_out, (uint8_t*) a->xq, a->ld_h, a->ld_add, a->ld_h_out, a->ld_x, a->n, a->eps,
                    a->add_is_bf16, a->x_is_bf16, a->image};
    auto whole = [](const void* p, int64_t ld, int bf16) { return !p || (aligned16(p) && ld % (bf16 ? 8 : 4) == 0); };
    const bool vec = a->n % 8 == 0 && aligned16(a->w) && whole(a->h, a->ld_h, a->h_is_bf16) && whole(a->add, a->ld_add, a->add_is_bf16) &&
                     whole(a->h_out, a->ld_h_out, a->h_is_bf16) && whole(a->x_out, a->ld_x, a->x_is_bf16);
    cudaStream_t s = as_stream(stream);
    if (vec) return a->h_is_bf16 ? launch_rms<true>(A, a->n_rows, s) : launch_rms<false>(A, a->n_rows, s);
    return a->h_is_bf16 ? launch_rms_any<true>(A, a->n_rows, s) : launch_rms_any<false>(A, a->n_rows, s);
}

extern "C" int maya_q8_read(const void* xq, int image, int64_t rows, int n, int out_is_bf16, void* values, uint16_t* sums, void* stream) {
    if (rows <= 0) return MAYA_OK;
    if (!xq || (!values && !sums) || n <= 0 || n % 32 || (image != MAYA_XQ_Q8_1 && image != MAYA_XQ_MMQ)) return refuse(MAYA_ERR_ARG);
    if (!aligned16(xq) || (values && !aligned16(values)) || (((uintptr_t) sums) & 1u)) return refuse(MAYA_ERR_ARG);
    const int64_t runs = rows * (n >> 3), blocks = (runs + 255) / 256;
    if (rows > 0x7FFFFFFFll || blocks > 0x7FFFFFFFll) return refuse(MAYA_ERR_LIMIT);
    const dim3 grid((unsigned) blocks), block(256);
    cudaStream_t s = as_stream(stream);
    __half* hs = (__half*) sums;
    if (image == MAYA_XQ_MMQ) {
        if (out_is_bf16) launch_dependent(q8_read_kernel<true, true>, grid, block, 0, s, (const uint8_t*) xq, runs, n, values, hs);
        else launch_dependent(q8_read_kernel<true, false>, grid, block, 0, s, (const uint8_t*) xq, runs, n, values, hs);
    } else {
        if (out_is_bf16) launch_dependent(q8_read_kernel<false, true>, grid, block, 0, s, (const uint8_t*) xq, runs, n, values, hs);
        else launch_dependent(q8_read_kernel<false, false>, grid, block, 0, s, (const uint8_t*) xq, runs, n, values, hs);
    }
    return note_launch("q8_read");
}
