/*
 * maya_attn.h - C ABI of the attention half of a decode or prompt layer over a paged cache of 8-bit keys and values.
 *
 * The reference has such kernels in its engines (norm and rotation in front of the cache, kv_* cache rounding, attention of
 * glm_fast.cu's decode path) with layouts and formats of those engines' own; these entry points are this library's own
 * interface, under the conventions of maya_moe.h: device pointers of the current device, caller-owned memory, nothing
 * allocated, nothing synchronised, everything enqueued on `stream`, a status as the result (0 enqueued, < 0 refused with
 * nothing launched).  What is read from device memory (lengths, tables, lists) cannot be checked by the host: a block number
 * outside the cache, a block beyond the table or a list entry outside the sequence is passed over, never followed.
 *
 * Cache.  A block is MAYA_KV_BLOCK consecutive tokens of one sequence.  For every block and key/value head there are
 * 64 * head_dim codes (value / scale rounded to nearest, -127 .. 127, stored + 128 in one byte) and one f32 scale, for the
 * keys and for the values:
 *   k        [n_blocks][n_kv][head_dim / 64][64 tokens][64 values]   16-byte aligned
 *   v        [n_blocks][n_kv][head_dim][64 tokens]                   16-byte aligned
 *   k_scale, v_scale [n_blocks][n_kv]
 *   k_sum    [n_blocks][n_kv][head_dim]  the sum of the keys' codes (less 128) over the block's tokens, 16-byte aligned;
 *            NULL: not kept (maya_block_select needs it)
 *   table    [n_seq][table_ld] i32: tokens 64 b .. 64 b + 63 of sequence s are in block table[s][b]
 * head_dim is 64, 128, 192 or 256.  Nothing needs clearing: a block's scale and sum are written when its first token is.
 *
 * Batch.  The new tokens of a pass are packed: those of sequence s are rows start[s] .. start[s + 1] - 1 and the last of its
 * kv_len[s] tokens (kv_len counts them), so that row start[s] + i stands at position kv_len[s] - new + i.  A sequence may
 * have none.  n_tokens = start[n_seq]; max_new and max_len are upper bounds of the new tokens and of kv_len of any sequence.
 */
#ifndef MAYA_ATTN_H
#define MAYA_ATTN_H

#include "maya_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MAYA_KV_BLOCK 64
#define MAYA_MAX_SELECTED 512      /* list entries of maya_block_select / maya_attn_q8 */
#define MAYA_MAX_KV_BLOCKS 16384   /* blocks of one sequence maya_block_select takes (1M tokens; so many for groups of up to 248 heads) */

typedef struct maya_kv_cache {
    void* k;
    void* v;
    float* k_scale;
    float* v_scale;
    int16_t* k_sum;
    const int32_t* table;
    int table_ld, n_blocks, n_kv, head_dim;
} maya_kv_cache;

typedef struct maya_attn_batch {
    const int32_t* start;     /* [n_seq + 1] */
    const int32_t* kv_len;    /* [n_seq] */
    int n_seq, n_tokens, max_new, max_len;
} maya_attn_batch;

/* Norm, rotation, append ---------------------------------------------------------------------------- */
typedef struct maya_rope_args {
    const void* q;            /* [n_tokens][n_q][head_dim], rows ld_q elements apart */
    const void* k;            /* [n_tokens][n_kv][head_dim], ld_k; NULL (with v): queries only, the cache is left alone */
    const void* v;
    int64_t ld_q, ld_k, ld_v;
    int is_bf16;              /* type of q, k, v and q_out: bf16, else f32 */
    int n_q;
    const float* q_w;         /* [head_dim] weights of the RMS norm of every query head; NULL: queries are not normalised */
    const float* k_w;
    float eps;
    const float* cos;         /* [n_pos][rot_dim / 2] */
    const float* sin;
    const int32_t* pos;       /* [n_tokens] row of cos / sin; NULL: the token's position in its sequence */
    int n_pos;                /* rows of cos / sin; a position outside them takes the nearest row */
    int rot_dim;              /* the first rot_dim values of a head are rotated; even, 0: none (cos, sin NULL) */
    int pairs;                /* 1: value 2 i turns with 2 i + 1; 0: value i with i + rot_dim / 2 */
    void* q_out;              /* [n_tokens][n_q][head_dim]; may be q when ld_q = n_q * head_dim */
} maya_rope_args;

/* For each new token: q_out = rotate(rms(q) * q_w); rotate(rms(k) * k_w) and v into the cache.  rms(x) = x / sqrt(mean(x^2) + eps)
 * over a head's values; rotate: (a, b) -> (a cos - b sin, b cos + a sin).  In f32; q_out rounded once.
 * A block takes the pass's tokens together: its new scale is max(the old one if it holds tokens from before, amax of the new
 * tokens / 127, or 2^-126 where that is less and amax is not 0); a code is value / scale rounded to nearest, by the scale's reciprocal
 * (within 2^-15 of a step); when the scale grows, the codes it holds become round(code * old / new), so a code is rounded once more at each
 * growth; k_sum is made from the codes.  A pass may start at an earlier length than the last one ended (tokens taken back).  Not finite: a NaN is stored as 0, an infinity as 127 times a scale of 1e30.
 * No two sequences of a batch may append to the same block. */
MAYA_API int maya_qk_norm_rope_append(const maya_kv_cache* cache, const maya_attn_batch* batch, const maya_rope_args* a, void* stream);

/* Block blocks[i] as the values it stands for: k and v [n][64][n_kv][head_dim], mean [n][n_kv][head_dim] the mean key of its
 * first counts[i] tokens from k_sum (NULL each: not wanted), bf16 or f32 (out_is_bf16).  Tokens from counts[i] on are zeros (counts
 * NULL: all 64 are read).  A block number outside the cache reads as zeros. */
MAYA_API int maya_kv_read(const maya_kv_cache* cache, const int32_t* blocks, const int32_t* counts, int n, int out_is_bf16, void* k,
                          void* v, void* mean, void* stream);

/* Attention ------------------------------------------------------------------------------------------- */
typedef struct maya_attn_args {
    const void* q;            /* [n_tokens][n_q][head_dim], rows ld_q elements apart */
    int64_t ld_q;
    int is_bf16;              /* type of q and out: bf16, else f32 */
    int n_q;                  /* a multiple of n_kv: query heads h * (n_q / n_kv) .. read key/value head h */
    float scale;              /* of the scores, > 0 */
    int window;               /* > 0: a token sees the last `window` positions up to its own; 0: all of them */
    const int32_t* sel;       /* NULL, or [n_tokens][n_kv][n_sel]: the blocks (by place in the sequence) a token reads, each
                                 once, -1 where there are fewer */
    int n_sel;
    void* out;                /* [n_tokens][n_q][head_dim] */
    float* lse;               /* NULL, or [n_tokens][n_q]: ln of the sum of exp(scores), -inf for a row that sees nothing */
} maya_attn_args;

/* out = sum_j softmax(scale * q . k_j)_j v_j over the tokens j of the sequence that stand at or before the query's own position,
 * within `window` and within the selected blocks; a row that sees nothing is 0.  A query with a NaN or an infinity gives a row of NaN
 * (and NaN in lse) wherever it sees a token.  bf16: value scales below 1e-30 count as 1e-30.  The cache holds the new tokens' keys and values already.
 * One kernel serves a call's sequences: those of a few rows (new tokens times heads of a group) are cut along their contexts, from 128 rows
 * of any sequence on (bf16, heads of 64 and 128) all go through the prompt kernel, and beyond 256 sequences (fewer, of windows) none is cut.  So pass prompt chunks
 * and single tokens at long contexts as two calls (196 + 912 us where one call takes 3843: 4096 tokens, and 64 at up to 131k), and sequences
 * far longer than the rest in calls of at most 256.
 * scratch: maya_attn_scratch_bytes(...) bytes (the same for any max_tokens > 0: parts have room of their own), 256-byte aligned, zeroed before the first use and after a call that left its
 * error word set; one buffer serves one stream at a time. */
MAYA_API size_t maya_attn_scratch_bytes(const maya_kv_cache* cache, int n_q, int max_tokens);
MAYA_API int maya_attn_q8(const maya_kv_cache* cache, const maya_attn_batch* batch, const maya_attn_args* a, void* scratch,
                          size_t scratch_bytes, void* stream);
/* The sticky error word of a scratch: 0, or 1 after a launch in which a bounded wait ran out (its outputs are not valid).
 * Synchronises the stream. */
MAYA_API int maya_attn_error(const void* scratch, void* stream);

/* Block selection --------------------------------------------------------------------------------------- */
typedef struct maya_select_args {
    const void* q;            /* as for maya_attn_q8 */
    int64_t ld_q;
    int is_bf16;
    int n_q;
    int n_first, n_last;      /* always selected: the first n_first blocks and the last n_last (>= 1) up to the token's own */
    int n_sel;                /* entries of a list, >= n_first + n_last, <= MAYA_MAX_SELECTED */
    int32_t* sel;             /* [n_tokens][n_kv][n_sel], ascending, -1 behind the last */
} maya_select_args;

/* For each new token and key/value head the n_sel blocks it reads: the forced ones, and of those between them the ones with the
 * highest score, max over the group's query heads g of (f32(q8_g . k_sum_b) * s_g) * k_scale_b, where q8_g = round(q_g / s_g) and
 * s_g = amax(q_g) * f32(1 / 127).  The dot is of whole numbers and exact, so a list does not depend on the order of any sum; equal
 * scores go to the lower block.  A block that the table does not have stands behind all that it has. */
MAYA_API int maya_block_select(const maya_kv_cache* cache, const maya_attn_batch* batch, const maya_select_args* a, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* MAYA_ATTN_H */
