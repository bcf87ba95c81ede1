/*
 * bitserve.h -- C ABI of the operators that serve a batch of sequences together
 * (MI355X / gfx950): a Q8 KV cache in pages of a shared pool, its append, its
 * reading back, the attention of every sequence's new rows over it, and the
 * choice of next tokens from logits.
 *
 * They stand beside their one-sequence counterparts of bitllama.h
 * (btl_rope_kv_append, btl_attention, btl_greedy_next); the reference
 * (imonoonoko/Bit-TTT-Engine, crates/rust_engine) has the contiguous cache of one
 * sequence (src/layers/kv_cache.rs:14-128), its attention
 * (src/layers/attention.rs:149-239) and a pick at a temperature
 * (src/model/llama.rs:496-530); pages, batches and filters are this library's.
 *
 * Conventions are those of bitlinear.h: int status (BTL_OK / BTL_ERR_*),
 * btl_last_error(), device pointers, `stream` a hipStream_t as void*, nothing
 * allocated or freed on the caller's behalf except the library workspace when
 * ws == NULL (calls that use it must be ordered on one stream; a call that has
 * to grow it is refused under capture).  Every result is reproducible bit for
 * bit: no sum depends on the order in which workgroups run.  All calls can be
 * captured in a HIP graph; what they read on the device (lengths, pages,
 * filters, random numbers) may change between replays.
 */
#ifndef BITSERVE_H
#define BITSERVE_H

#include <stddef.h>
#include <stdint.h>

#include "bitlinear.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * One layer's Q8 cache in pages (device pointers).  Codes and scales are those
 * of btl_kv_q8_t: u8 = round(x / s) + 128, s = max|x| / 127 per (token, KV head).
 * k: [n_pages, n_kv_heads, page_size, head_dim] u8
 * v: [n_pages, n_kv_heads, page_size / 16, head_dim, 16] u8: blocks of 16 tokens,
 *    the tokens innermost (the order in which the attention's second product
 *    takes them: 16 tokens of one value are one load)
 * k_scale, v_scale: [n_pages, n_kv_heads, page_size] f32
 * page_size a multiple of 16 up to 65536, head_dim a multiple of 16 up to 128,
 * n_pages * n_kv_heads * page_size < 2^35; every array 16-byte aligned.
 */
typedef struct btl_kv_paged {
    uint8_t* k;
    uint8_t* v;
    float* k_scale;
    float* v_scale;
    int64_t n_pages;
    int64_t n_kv_heads;
    int64_t page_size;
    int64_t head_dim;
} btl_kv_paged_t;

/*
 * The sequences of one call.  row_start, pos and pages are device int32 arrays:
 * row_start [n_seqs + 1]: sequence s has the rows row_start[s] .. row_start[s+1]-1
 *   of q, k, v, out (none: it sits out).  Not decreasing.
 * pos [n_seqs]: the position of its first row: the tokens its pages hold already.
 * pages [n_seqs, max_pages]: the page of its positions j * page_size ...
 *   Two sequences may share pages that are only read; a slot that two rows of one
 *   append write holds either's bytes.
 * rows: rows of q, k, v and out; rows of no sequence are left as they were.
 * max_rows, max_len: the host's bounds on any sequence's rows and on its tokens
 *   with them (pos + rows); they choose launches and split the work.
 * What the device finds wrong is answered there: a sequence with pos < 0, more
 * than max_rows rows or more than min(max_len, max_pages * page_size, 2^23) tokens
 * has NaN in all its output rows and nothing is appended for it; a row that needs a
 * page outside [0, n_pages) has NaN (attention, read) or is not stored (append).
 */
typedef struct btl_paged_batch {
    const int32_t* row_start;
    const int32_t* pos;
    const int32_t* pages;
    int64_t n_seqs;
    int64_t max_pages;
    int64_t rows;
    int64_t max_rows;
    int64_t max_len;
} btl_paged_batch_t;

/*
 * btl_rope_kv_append for a batch: RoPE of q [rows, n_heads * head_dim] -> q_out
 * (may be q itself) and of k [rows, n_kv * head_dim], then the Q8 append of k and
 * v into the slots of the rows' positions; the codes and scales are bit for bit
 * those of btl_rope_kv_append.  q, k, v, q_out of dtype (BTL_F32 or BTL_BF16:
 * widened exactly, computed in f32, q_out rounded to nearest even; k is quantised
 * from its f32 rotation).  rope_cos / rope_sin: device [rope_len, head_dim / 2]
 * (btl_rope_table); a row at a position >= rope_len is not stored and its q_out
 * is NaN.  Every array is 16-byte aligned; q, k, v and q_out share no memory but
 * q_out == q.
 */
int btl_paged_rope_append(const void* q, const void* k, const void* v, int dtype, int64_t n_heads,
                          const btl_kv_paged_t* cache, const btl_paged_batch_t* batch, const float* rope_cos,
                          const float* rope_sin, int64_t rope_len, void* q_out, void* stream);

/*
 * The cache read back: for every row, its position's key and value (code - 128) *
 * scale into k_out and v_out [rows, n_kv * head_dim] of dtype (either may be
 * NULL), 16-byte aligned.  Whole contexts are rows at pos = 0.  Keys are as stored,
 * rotated.
 */
int btl_paged_read(const btl_kv_paged_t* cache, const btl_paged_batch_t* batch, void* k_out, void* v_out, int dtype,
                   void* stream);

/*
 * Attention of the rows (rotated queries [rows, n_heads * head_dim] of dtype) over
 * their sequences' pages, row i of a sequence seeing positions 0 .. pos + i (the
 * causal mask; the rows' own keys are in the cache, btl_paged_rope_append before
 * it): softmax(q . k_deq / sqrt(head_dim)) . v_deq -> out, of dtype.  GQA head h
 * reads KV head h / (n_heads / n_kv), n_heads / n_kv <= 16.
 * Arithmetic: the codes are exact in the matrix instructions' f16; queries and
 * softmax weights are taken in two f16 parts (22 bits) for BTL_F32; for BTL_BF16
 * queries in one (exact), weights in two for sequences of at most 16 rows times
 * heads of a group and in one (11 bits) for longer ones (for a single sequence
 * max_rows decides it); products are summed in f32, the softmax's maxima, sums and
 * outputs are f32.  Powers of two keep the parts in f16's range: one a row, by its
 * largest query, and one by the largest value scale that the row has seen.  Their
 * limits, with 2^e <= the row's largest query: a row of queries all below 2^-96 loses
 * bits from there on (e counts as -96); q . k of 2^(114 + e) and more is infinite (a
 * positive one makes the row NaN, a negative one is not seen); values of scales below
 * 2^-96, or below 2^-10 of the largest that the row sees, lose bits from there on, of a
 * weight less than 2^-33 of the likeliest key's at that largest scale.
 * What a row's mask hides has no effect on it, whatever it holds; a row that sees a
 * scale or holds a query that is not finite is NaN.
 * Chunks of keys, which are what few sequences spread over the chip by, are cut for
 * max_len, not for the lengths that the device finds: a bound far above them leaves
 * fewer and longer chunks.
 * ws: btl_paged_attention_workspace_bytes (or NULL: the library's).  q, out 16-byte
 * aligned; out overlaps nothing that is read.
 */
size_t btl_paged_attention_workspace_bytes(int64_t n_heads, const btl_kv_paged_t* cache,
                                           const btl_paged_batch_t* batch);
int btl_paged_attention(const void* q, int dtype, int64_t n_heads, const btl_kv_paged_t* cache,
                        const btl_paged_batch_t* batch, void* out, void* ws, size_t ws_bytes, void* stream);

/*
 * Next tokens from logits [rows, n] f32, `ld` apart (ld >= n), and given random
 * numbers u [rows] in [0, 1).  temperature, top_k, top_p, min_p: device arrays of
 * one value a row, or NULL (1, off, off, off).  Per row, with M the largest logit:
 *   w_i = rint(2^40 exp((l_i - M) / temperature)) in f64, a whole number: sums of
 *   it are exact, so neither their order nor their split changes a token;
 *   tokens are ordered by (logit descending, index ascending);
 *   min_p  (> 0): only those with w_i >= min_p * 2^40 stay (at least the first);
 *   top_k  (1 .. n-1): only the first top_k of them;
 *   top_p  (< 1): only the shortest prefix of what is left that holds at least
 *          top_p of its weight (at least the first token);
 *   W = the weight of what stays, id = the first in that order whose running
 *   weight exceeds floor(u * W).
 * ids [rows] int32; probs NULL or [rows] f32: w_id / W.  A temperature <= 0 (or
 * NaN) takes the first of the largest logits (probability 1).  A NaN logit counts
 * as -inf; with +inf among the logits only those share the weight; a row without a
 * finite or +inf logit has id -1 and probability 0.  A NaN filter is off; u below
 * 0 or NaN is taken as 0, from 1 on as the last token.
 * 1 <= n <= 2^22, at most 65535 rows.  ws: btl_sample_workspace_bytes (or NULL: the
 * library's).
 */
size_t btl_sample_workspace_bytes(int64_t rows, int64_t n);
int btl_sample(const float* logits, int64_t rows, int64_t n, int64_t ld, const float* temperature,
               const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* ids,
               float* probs, void* ws, size_t ws_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* BITSERVE_H */
