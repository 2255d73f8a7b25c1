// lora.cu - low-rank adapters of many requests beside a projection that all of them share:
//
//   out[t] = y[t] + scale_i * B_i (A_i x[t]),  i = idx[t];  idx[t] outside 0 .. n_adapters - 1: out[t] = y[t]
//
// A [n_adapters][rank][n_in], B [n_adapters][n_out][rank] in bf16 or f16, x f32 or bf16, y and out f32.  Products and sums in f32.
//
// Two launches: z = A x over pieces of n_in, the pieces' sums left side by side in the scratch (nothing is added in an order that depends on how blocks
// run), then out = y + scale * B z.  The second waits for nothing but z: the first lets it start once what stood in front of both is done, so that its rows of
// B and y are on their way while z is made.
//
// Few tokens (lora_z_kernel, lora_out_kernel): each token reads its adapter's matrices, out of L2 where tokens share one.  What bounds a step of decode
// is latency - two launches, two round trips each: 3.2 us for one token of rank 16, 4096 -> 6144 - and, for some dozens, what comes out of L2: 9.1 us for 64
// tokens, 21 MB.  Many tokens: lora_prompt.cu, 67 us for 4096 of rank 64; which of the two serves a call is said there.
#include "maya_lora.cuh"

namespace maya {
namespace {

constexpr int kLoraRows = 4;                   // rows of A a warp multiplies: x is read once for them
constexpr int kLoraPiece = 512;                // values of n_in a warp takes: two 16-byte loads of each row a lane
constexpr int kLoraWarps = 8;
constexpr size_t kLoraWords = 256;             // bytes of the scratch in front of z: the error word of the prompts' kernels

// z of one token: a warp takes four rows of A over one piece of n_in.  blockIdx.y: the token.
template<bool XB, bool F16>
__global__ void __launch_bounds__(32 * kLoraWarps) lora_z_kernel(const Lora A) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    grid_dependency_wait();
    grid_launch_dependents();                  // (behind the wait: what the next launch reads ahead of its own is finished)
    const int job = blockIdx.x * kLoraWarps + warp, quads = A.rank / kLoraRows;
    if (job >= quads * A.pieces) return;
    const int piece = job / quads, r0 = (job - piece * quads) * kLoraRows, t = blockIdx.y;
    const int i = A.idx[t];
    if (i < 0 || i >= A.n_adapters) return;
    const uint16_t* rows = (const uint16_t*) A.a + ((size_t) i * A.rank + r0) * A.n_in;
    float acc[kLoraRows] = {};
    uint4 w[2][kLoraRows];
    float x[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int c = piece * kLoraPiece + h * 256 + lane * 8;
        const bool live = c < A.n_in;
#pragma unroll
        for (int r = 0; r < kLoraRows; ++r) {
            w[h][r] = make_uint4(0u, 0u, 0u, 0u);
            if (live) w[h][r] = __ldg((const uint4*) (rows + (size_t) r * A.n_in + c));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[h][j] = 0.0f;
        if (live) {
            if constexpr (XB) {
                weights8<false>(*(const uint4*) ((const uint16_t*) A.x + t * A.ld_x + c), x[h]);
            } else {
                const float4 u = *(const float4*) ((const float*) A.x + t * A.ld_x + c), v = *(const float4*) ((const float*) A.x + t * A.ld_x + c + 4);
                x[h][0] = u.x; x[h][1] = u.y; x[h][2] = u.z; x[h][3] = u.w; x[h][4] = v.x; x[h][5] = v.y; x[h][6] = v.z; x[h][7] = v.w;
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < kLoraRows; ++r) {
            float f[8];
            weights8<F16>(w[h][r], f);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[r] = __fmaf_rn(f[j], x[h][j], acc[r]);
        }
#pragma unroll
    for (int r = 0; r < kLoraRows; ++r) acc[r] = warp_sum(acc[r]);
    if (lane == 0) *(float4*) (A.z + ((size_t) piece * A.n_tokens + t) * A.rank + r0) = make_float4(acc[0], acc[1], acc[2], acc[3]);
}

// out of one token: a thread an output.  The first 32 values of its row of B and its y are asked for ahead of z (out of L2: L1 may hold what an earlier call
// left there).
template<bool F16>
__global__ void __launch_bounds__(256) lora_out_kernel(const Lora A) {
    extern __shared__ __align__(16) float zs[];
    const int tid = threadIdx.x, n = blockIdx.x * 256 + tid, t = blockIdx.y;
    const int i = __ldcg(A.idx + t);
    const bool has = i >= 0 && i < A.n_adapters, live = n < A.n_out;
    const uint4* row = (const uint4*) ((const uint16_t*) A.b + ((size_t) (has ? i : 0) * A.n_out + (live ? n : 0)) * A.rank);
    const int eights = A.rank >> 3;
    uint4 w[4];
    float y = 0.0f, s = 1.0f;
    if (live && A.y != nullptr) y = __ldcg(A.y + t * A.ld_y + n);
    if (has) {
        if (A.scale != nullptr) s = __ldcg(A.scale + i);
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (q < eights) w[q] = __ldcg(row + q);
    }
    grid_launch_dependents();
    grid_dependency_wait();
    if (!has) {                                // the whole block: one token
        if (live) A.out[t * A.ld_out + n] = y;
        return;
    }
    for (int r = tid; r < A.rank; r += 256) {
        float v = 0.0f;
#pragma unroll 8
        for (int p = 0; p < A.pieces; ++p) v += A.z[((size_t) p * A.n_tokens + t) * A.rank + r];
        zs[r] = v;
    }
    __syncthreads();
    float acc = 0.0f;
    auto add = [&](const uint4 u, int q) {
        float f[8];
        weights8<F16>(u, f);
        const float4 a = *(const float4*) (zs + 8 * q), b = *(const float4*) (zs + 8 * q + 4);
        acc = __fmaf_rn(f[0], a.x, acc); acc = __fmaf_rn(f[1], a.y, acc); acc = __fmaf_rn(f[2], a.z, acc); acc = __fmaf_rn(f[3], a.w, acc);
        acc = __fmaf_rn(f[4], b.x, acc); acc = __fmaf_rn(f[5], b.y, acc); acc = __fmaf_rn(f[6], b.z, acc); acc = __fmaf_rn(f[7], b.w, acc);
    };
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (q < eights) add(w[q], q);
    for (int q = 4; q < eights; ++q) add(__ldcg(row + q), q);
    if (live) A.out[t * A.ld_out + n] = __fmaf_rn(s, acc, y);
}

int lora_pieces(int n_in) { return (n_in + kLoraPiece - 1) / kLoraPiece; }

template<bool F16> int lora_launch(const Lora& A, int x_is_bf16, cudaStream_t s) {
    const int jobs = A.rank / kLoraRows * A.pieces;
    const dim3 gz((unsigned) ((jobs + kLoraWarps - 1) / kLoraWarps), (unsigned) A.n_tokens);
    if (x_is_bf16) launch_dependent(lora_z_kernel<true, F16>, gz, dim3(32 * kLoraWarps), 0, s, A);
    else launch_dependent(lora_z_kernel<false, F16>, gz, dim3(32 * kLoraWarps), 0, s, A);
    const int st = note_launch("lora z");
    if (st != MAYA_OK) return st;
    launch_dependent(lora_out_kernel<F16>, dim3((unsigned) ((A.n_out + 255) / 256), (unsigned) A.n_tokens), dim3(256), (size_t) A.rank * sizeof(float), s, A);
    return note_launch("lora out");
}

}  // namespace
}  // namespace maya

using namespace maya;

extern "C" size_t maya_lora_scratch_bytes(int n_in, int rank, int n_adapters, int max_tokens) {
    if (n_in <= 0 || n_in % 32 || rank <= 0 || rank % 16 || rank > MAYA_MAX_LORA_RANK || n_adapters <= 0 || max_tokens <= 0 || max_tokens > MAYA_MAX_LORA_TOKENS) return 0;
    const size_t few = kLoraWords + (size_t) lora_pieces(n_in) * max_tokens * rank * sizeof(float);
    const size_t many = lora_many_fits(max_tokens, n_adapters, rank) ? lora_prompt_bytes(max_tokens, n_adapters, rank) : 0;
    return few > many ? few : many;
}

extern "C" int maya_lora_error(const void* scratch, void* stream) {
    if (!scratch) return refuse(MAYA_ERR_ARG);
    int word = 0;
    cudaStream_t s = as_stream(stream);
    if (cudaMemcpyAsync(&word, scratch, sizeof(word), cudaMemcpyDeviceToHost, s) != cudaSuccess || cudaStreamSynchronize(s) != cudaSuccess) return note_launch("lora error");
    return word;
}

extern "C" int maya_lora(const maya_lora_args* a, void* stream) {
    if (!a) return refuse(MAYA_ERR_ARG);
    if (a->n_tokens <= 0) return MAYA_OK;
    if (!a->x || !a->out || !a->a || !a->b || !a->idx || !a->scratch || a->n_adapters <= 0 || a->n_in <= 0 || a->n_out <= 0) return refuse(MAYA_ERR_ARG);
    if (a->n_in % 32 || a->rank <= 0 || a->rank % 16) return refuse(MAYA_ERR_ARG);
    if (a->rank > MAYA_MAX_LORA_RANK || a->n_tokens > MAYA_MAX_LORA_TOKENS) return refuse(MAYA_ERR_LIMIT);
    if (a->ld_x < a->n_in || (a->y && a->ld_y < a->n_out) || a->ld_out < a->n_out) return refuse(MAYA_ERR_ARG);
    if (a->ld_x > 0x7FFFFFFFll || (a->y && a->ld_y > 0x7FFFFFFFll) || a->ld_out > 0x7FFFFFFFll) return refuse(MAYA_ERR_LIMIT);
    if (a->y == a->out && a->ld_y != a->ld_out) return refuse(MAYA_ERR_ARG);
    if (!aligned16(a->x) || !aligned16(a->a) || !aligned16(a->b) || (((uintptr_t) a->scratch) & 255u) || a->ld_x % (a->x_is_bf16 ? 8 : 4)) return refuse(MAYA_ERR_ARG);
    if (a->kernel < MAYA_LORA_CHOICE || a->kernel > MAYA_LORA_MANY) return refuse(MAYA_ERR_ARG);
    bool many = a->kernel == MAYA_LORA_MANY;
    if (a->kernel == MAYA_LORA_CHOICE) many = lora_many_better(a->n_tokens, a->n_adapters, a->rank, a->n_in + a->n_out);
    if (many && a->n_adapters > kLoraAdaptersMost) return refuse(MAYA_ERR_LIMIT);
    const size_t need = many ? lora_prompt_bytes(a->n_tokens, a->n_adapters, a->rank) : kLoraWords + (size_t) lora_pieces(a->n_in) * a->n_tokens * a->rank * sizeof(float);
    if (a->scratch_bytes < need) return refuse(MAYA_ERR_LIMIT);
    const Lora A{a->x, a->y, a->out, a->a, a->b, a->scale, a->idx, (float*) ((uint8_t*) a->scratch + kLoraWords), a->ld_x, a->ld_y, a->ld_out, a->n_adapters, a->n_in, a->n_out,
                 a->rank, a->n_tokens, lora_pieces(a->n_in)};
    if (many) return lora_prompt(A, a->x_is_bf16, a->w_is_f16, a->scratch, as_stream(stream));
    return a->w_is_f16 ? lora_launch<true>(A, a->x_is_bf16, as_stream(stream)) : lora_launch<false>(A, a->x_is_bf16, as_stream(stream));
}
