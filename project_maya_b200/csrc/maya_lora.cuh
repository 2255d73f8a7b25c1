// maya_lora.cuh - a call of the low-rank adapters as its kernels take it (lora.cu: few tokens; lora_prompt.cu: prompts).
#pragma once

#include "maya_common.cuh"

namespace maya {

struct Lora {
    const void* x;
    const float* y;
    float* out;
    const void* a;
    const void* b;
    const float* scale;
    const int* idx;
    float* z;                    // [pieces][n_tokens][rank]
    int64_t ld_x, ld_y, ld_out;
    int n_adapters, n_in, n_out, rank, n_tokens, pieces;
};

// 8 weights of 16 bits as f32.
template<bool F16> __device__ __forceinline__ void weights8(const uint4 u, float (&w)[8]) {
    const uint32_t p[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (F16) {
            const float2 f = __half22float2(*(const __half2*) &p[i]);
            w[2 * i] = f.x; w[2 * i + 1] = f.y;
        } else {
            w[2 * i] = __uint_as_float(p[i] << 16); w[2 * i + 1] = __uint_as_float(p[i] & 0xFFFF0000u);
        }
    }
}

// ---- prompts (lora_prompt.cu): tokens of one adapter in tiles of kLoraTile rows
constexpr int kLoraTile = 128;
constexpr int kLoraAdaptersMost = 4096;        // whose tokens one thread block counts
bool lora_many_fits(int n_tokens, int n_adapters, int rank);                         // the scratch has room for it
bool lora_many_better(int n_tokens, int n_adapters, int rank, int width);            // width: n_in + n_out
size_t lora_prompt_bytes(int n_tokens, int n_adapters, int rank);
int lora_prompt(const Lora& A, int x_is_bf16, int w_is_f16, void* scratch, cudaStream_t s);

}  // namespace maya
