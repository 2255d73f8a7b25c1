// kv_attn.cuh - attention over the paged 8-bit cache, what its kernels share: arguments, work tiles, partial results and their join.
//
// softmax(scale q.K) V over one tile of query rows in one pass over the cache: running maximum m (base 2), sum l and output O in f32.
//   s_j = (q . k_j) * scale * k_scale[block] * log2(e)          p_j = 2^(s_j - m)          O = sum p_j v_j,  l = sum p_j
// The codes of K and V become f16 exactly (|code| <= 127); a query row is multiplied by a power of two that brings its largest
// value to 2^11 .. 2^12 and rounded to f16, or for f32 activations split in two f16 terms (22 bits); P likewise, as 2^12 p
// (bf16: 2^4 p) with v_scale[block] in its exponent, so that m is a maximum of p v_scale and P in f16's range whatever the scales.  Products are summed in f32.
#pragma once

#include "maya_kv.cuh"
#include "maya_stream.cuh"

namespace maya {

constexpr float kRise = 8.0f;                    // how far a maximum may pass m (base 2) before m is raised to it
constexpr float kNone = -INFINITY;
// The power of two that brings a query row's largest value to 2^11 .. 2^12: -116 for the largest numbers there are, 126 at most (2^-126 is the smallest normal
// number), so that it and its reciprocal are normal numbers.
__device__ __forceinline__ int up_of_row(float amax) { return amax > 0.0f ? min(126, 138 - (int) (__float_as_uint(amax) >> 23)) : 0; }
// What multiplies the scores of a query row whose largest value is amax: NaN for a row with an infinity, whose products may be anything (0 times it among
// them).  A row with a NaN has NaN scores by itself.  Such rows are NaN wherever they see a token, so that what went wrong in front stays visible.
__device__ __forceinline__ float scale_of_row(float amax, float scale) { return amax < INFINITY ? scale : __uint_as_float(0x7fc00000u); }
// ln of a row's sum of exp(scores) from m and l, the sum of P (V's scale taken out again); -inf for a row that saw nothing.
__device__ __forceinline__ float lse_of(float m, float l, float bias) { return l == 0.0f ? kNone : (m + log2f(l) - bias) * 0.69314718055994531f; }

struct AttnView {
    const void* q;
    int64_t ld_q;
    void* out;
    float* lse;
    const int* sel;
    int n_sel, n_q, group, window, wide_q;
    float scale_log2;                            // scale * log2(e)
    int row_tiles;                               // tiles of a sequence (of a token, with sel)
    int tiles;                                   // of all sequences (tokens)
    bool direct;                                 // a thread block a (tile, head), in one piece
    unsigned* error;
    unsigned fixed;                              // > 0: every (tile, head) is cut into so many pieces (prompts)
    unsigned grid, pairs, parts_most;            // thread blocks; (tile, head)s; parts there is room for
    unsigned warm_q, warm_table;                 // lines of 128 bytes
    unsigned* taken;                             // pieces taken beyond each thread block's first; thread blocks that have left
    int* pre;                                    // pieces of a head in front of each tile: for the join
    float* part_o;                               // [piece][rows][D]
    float2* part_ml;                             // [piece][rows]
};

// The scratch: a 256-byte head (the error word, the counters), the prefix, the parts.
constexpr size_t kAttnHead = 256, kAttnPre = 2048;
constexpr int kCtasMost = 448;                   // thread blocks that share out the work: three an SM
constexpr int kPartRows = 2 * kCtasMost * 64;      // rows of parts
constexpr float kVsLeast = 1e-30f;               // bf16: a value scale of 0 is this in P's exponent, and so is one below it (off by 127e-30 at most): l stays in f32's range
constexpr uint32_t kVsExpLeast = 127 - 64;       // f32: 2^-64, the exponent alone; what is below it is in the factor, in full for scales down to 2^-79
// The join of the prompt kernel's pieces (kv_attn.cu), `rows` rows a tile.
int attn_join(const maya_kv_cache& c, const maya_attn_batch& b, const AttnView& A, int rows, cudaStream_t s);
constexpr int kNotTaken = 1;
// Attention of a prompt's rows on tcgen05 (kv_attn_prompt.cu); kNotTaken: not that kernel's call, nothing launched.
int attn_prompt(const maya_kv_cache& c, const maya_attn_batch& b, const AttnView& A, bool bf16, cudaStream_t s);

}  // namespace maya
