// maya_kv.cuh - the paged 8-bit cache on the device: geometry, checked look-ups, codes to 16-bit values; host checks.
#pragma once

#include <cuda_bf16.h>

#include "maya_attn.h"
#include "maya_common.cuh"

namespace maya {

constexpr int kKvBlock = MAYA_KV_BLOCK;
constexpr float kInv127 = 1.0f / 127.0f;
constexpr float kScaleLeast = 0x1p-126f;  // of a block with a value that is not 0: its reciprocal is finite
constexpr float kScaleMost = 1e30f;       // of a block that was given an infinity: 127 * kScaleMost is finite

// The cache and the batch as the kernels take them.
struct KvView {
    uint8_t* k;
    uint8_t* v;
    float* k_scale;
    float* v_scale;
    int16_t* k_sum;
    const int* table;
    int table_ld, n_blocks, n_kv;
};
struct BatchView {
    const int* start;
    const int* kv_len;
    int n_seq, n_tokens, max_new, max_len;
};
inline KvView kv_view(const maya_kv_cache& c) {
    return {(uint8_t*) c.k, (uint8_t*) c.v, c.k_scale, c.v_scale, c.k_sum, c.table, c.table_ld, c.n_blocks, c.n_kv};
}
inline BatchView batch_view(const maya_attn_batch& b) { return {b.start, b.kv_len, b.n_seq, b.n_tokens, b.max_new, b.max_len}; }

inline int kv_check(const maya_kv_cache* c) {
    if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale || !c->table || c->table_ld <= 0 || c->n_blocks <= 0 || c->n_kv <= 0) return MAYA_ERR_ARG;
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 192 && c->head_dim != 256) return MAYA_ERR_LIMIT;
    if (!aligned16(c->k) || !aligned16(c->v) || (c->k_sum && !aligned16(c->k_sum))) return MAYA_ERR_ARG;
    return MAYA_OK;
}
inline int batch_check(const maya_kv_cache* c, const maya_attn_batch* b) {
    if (!b || !b->start || !b->kv_len || b->n_seq < 0 || b->n_tokens < 0 || b->max_new < 0 || b->max_len < 0) return MAYA_ERR_ARG;
    if (b->n_tokens > 0 && (b->n_seq == 0 || b->max_new == 0 || b->max_new > b->n_tokens)) return MAYA_ERR_ARG;
    if ((long long) b->n_seq * b->max_new < b->n_tokens) return MAYA_ERR_ARG;
    if (b->n_seq > 65535 || b->n_tokens > (1 << 24)) return MAYA_ERR_LIMIT;
    if (b->max_len > (long long) c->table_ld * kKvBlock) return MAYA_ERR_ARG;
    return MAYA_OK;
}

// Sequence s of a batch: its first packed row, its new tokens and its tokens in all, held to what the batch says at most.
struct Seq {
    int row, n_new, len;
};
__device__ __forceinline__ Seq seq_of(const BatchView& B, int s) {
    Seq q;
    q.row = max(0, min(B.start[s], B.n_tokens));
    q.n_new = max(0, min(min(B.start[s + 1], B.n_tokens) - q.row, B.max_new));
    q.len = max(0, min(B.kv_len[s], B.max_len));
    return q;
}
// The sequence a packed row belongs to: the last s with start[s] <= row.
__device__ __forceinline__ int seq_of_row(const BatchView& B, int row) {
    int lo = 0, hi = B.n_seq - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (B.start[mid] <= row) lo = mid; else hi = mid - 1;
    }
    return lo;
}
// The block that holds tokens 64 b .. of sequence s, or -1.
__device__ __forceinline__ int block_of(const KvView& C, int s, int b) {
    if (b < 0 || b >= C.table_ld) return -1;
    const int p = C.table[(size_t) s * C.table_ld + b];
    return p >= 0 && p < C.n_blocks ? p : -1;
}

// Four codes (one byte each, value + 128) -> two f16 pairs of the values, exactly: 0x64xx is 1024 + xx in f16.
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
    const __half2 bias = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));     // 1152
    uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*(__half2*) &a, bias), y = __hsub2(*(__half2*) &b, bias);
    lo = *(const uint32_t*) &x;
    hi = *(const uint32_t*) &y;
}

template<bool BF16> __device__ __forceinline__ float ld_act(const void* p, size_t i) {
    if constexpr (BF16) return __uint_as_float((uint32_t) ((const uint16_t*) p)[i] << 16);
    return ((const float*) p)[i];
}
template<bool BF16> __device__ __forceinline__ void st_act(void* p, size_t i, float v) {
    if constexpr (BF16) ((__nv_bfloat16*) p)[i] = __float2bfloat16_rn(v);
    else ((float*) p)[i] = v;
}
// V consecutive values of a row, V even; `wide`: the address is aligned for whole-vector loads.
template<bool BF16, int V> __device__ __forceinline__ void ld_acts(const void* p, size_t i, bool wide, float (&x)[V]) {
    if (wide) {
        if constexpr (BF16) {
            const uint32_t* w = (const uint32_t*) ((const uint16_t*) p + i);
            uint32_t r[V / 2];
            if constexpr (V % 8 == 0) {
#pragma unroll
                for (int j = 0; j < V / 8; ++j) *(uint4*) &r[4 * j] = ((const uint4*) w)[j];
            } else if constexpr (V == 4) *(uint2*) r = *(const uint2*) w;
            else {
#pragma unroll
                for (int j = 0; j < V / 2; ++j) r[j] = w[j];
            }
#pragma unroll
            for (int j = 0; j < V / 2; ++j) { x[2 * j] = __uint_as_float(r[j] << 16); x[2 * j + 1] = __uint_as_float(r[j] & 0xFFFF0000u); }
        } else {
            const float* w = (const float*) p + i;
            if constexpr (V % 4 == 0) {
#pragma unroll
                for (int j = 0; j < V / 4; ++j) *(float4*) &x[4 * j] = ((const float4*) w)[j];
            } else {
#pragma unroll
                for (int j = 0; j < V / 2; ++j) *(float2*) &x[2 * j] = ((const float2*) w)[j];
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) x[j] = ld_act<BF16>(p, i + j);
    }
}
// Whether whole-vector accesses of D / 32 values a lane are aligned for rows `ld` elements apart.
inline bool rows_wide(const void* p, int64_t ld, int elem) { return aligned16(p) && (ld * elem) % 16 == 0; }

}  // namespace maya
