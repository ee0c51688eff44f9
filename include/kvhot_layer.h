/*
 * kvhot_layer.h -- C ABI of the rest of a layer's KV side, beside kvhot.h: a
 * step's block tables, the norms and rotation of queries and keys, and a KV
 * cache held in 4 bits with the attention over it.
 *
 * The conventions are kvhot.h's: stateless, ordered on the caller's stream, no
 * device memory allocated or freed, sizes and strides int64 (strides in
 * elements unless they say bytes), everything checked on the host before a
 * launch, the same return codes and kvhot_last_error().
 */
#ifndef KVHOT_LAYER_H
#define KVHOT_LAYER_H

#include "kvhot.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Block tables, starts, slots and positions of one engine step, built on the
 * device from the rows' lengths.  Row r has prior_lens[r] cached tokens, in the
 * first ceil(prior_lens[r] / block_size) blocks of block_table[r, :], and adds
 * q_lens[r] tokens (negative lengths count as 0).  The blocks it needs beyond
 * those it holds are the next ones of free_blocks, row by row in order:
 *   k_lens[r]   = prior_lens[r] + q_lens[r]
 *   q_starts[r] = sum of q_lens before r
 *   block_table[r, c] = the row's next free block, for its new blocks c; no
 *                       other entry is written
 *   slot_mapping, positions: as kvhot_build_slot_mapping, and -1 and 0 for the
 *                       tokens from the last row's end to total_query
 *   *blocks_taken = blocks that all rows need beyond those they hold
 * total_query is the length of slot_mapping and positions; nothing beyond it
 * is written.  Where *blocks_taken > num_free, the blocks that are not there
 * are entered as block 0 and their tokens' slots are -1 (so are those of tokens
 * beyond the table's bt_row_stride columns): the caller has to look at it.
 * max_q_len sizes the grid only.  Repeating a call repeats its results.
 * The reference allocates blocks and maps slots on the host, row by row
 * (serving_engine/block_manager.py:63-112, serving_engine/model_runner.py:142-170).
 */
int kvhot_build_block_tables(int32_t* block_table, int64_t bt_row_stride,
                             const int32_t* prior_lens, const int32_t* q_lens,
                             const int32_t* free_blocks, int64_t num_free,
                             int64_t num_rows, int64_t total_query,
                             int64_t max_q_len, int64_t block_size,
                             int32_t* q_starts, int32_t* k_lens,
                             int64_t* slot_mapping, int64_t* positions,
                             int32_t* blocks_taken, void* stream);

/*
 * Norms of queries and keys of each head and their rotation by position, in
 * one pass, between a layer's projections and its append.  For each token t
 * and head of q [T, num_q_heads, D] and k [T, num_kv_heads, D]:
 *   y = x * weight / sqrt(mean(x^2) + eps)      (y = x where the weight is NULL)
 *   (y[i], y[j]) -> (y[i] c - y[j] s, y[j] c + y[i] s) for the pairs of the first
 *   rotary_dim elements, (i, i + rotary_dim / 2) or, interleaved, (2 p, 2 p + 1)
 * with c = table[positions[t], p], s = table[positions[t], rotary_dim / 2 + p]
 * for pair p; table is fp32 [table_rows, rotary_dim], contiguous, 16-byte
 * aligned.  fp32 throughout, rounded once.  A position outside the table makes
 * the token's rows NaN.  head_dim (up to 512) and rotary_dim are multiples of
 * 8; tensors have a unit head_dim stride.  An output may be its input (the
 * same pointer and strides), but not overlap it otherwise.  Weights are
 * [head_dim], of weight_dtype: dtype or KVHOT_F32.  Positions are int64 or
 * int32.  The reference leaves this to the model.
 */
int kvhot_norm_rope(const void* q, const int64_t q_strides[3], const void* k,
                    const int64_t k_strides[3], void* q_out,
                    const int64_t q_out_strides[3], void* k_out,
                    const int64_t k_out_strides[3], const void* q_weight,
                    const void* k_weight, int weight_dtype, float eps,
                    const float* table, int64_t table_rows, int64_t rotary_dim,
                    int interleaved, const void* positions,
                    int positions_are_int64, int64_t num_tokens,
                    int64_t num_q_heads, int64_t num_kv_heads,
                    int64_t head_dim, int dtype, void* stream);

/*
 * A KV cache held in 4 bits.  One layer is [num_blocks, block_size / 16,
 * num_kv_heads, 17 * head_dim] bytes, contiguous but for the block stride
 * (bytes; a multiple of 16, as the base pointer is); block_size is a multiple
 * of 16, head_dim 64, 96, 128 or 256.  A record of 17 * head_dim bytes holds
 * the K and V of 16 tokens of a kv head:
 *   K codes  byte t * D/2 + b:       elements 2b (low half) and 2b + 1 of token t
 *   V codes  byte 8 D + 16 p + t:    elements 2p (low half) and 2p + 1 of token t
 *   K scales byte 16 D + 16 g + 4 (t % 4) + t / 4:  elements 32 g.. of token t
 *   V scales byte 16 D + D/2 + 16 g + t:            elements 32 g.. of token t
 * A code is a sign (8) and the index of 0, 0.5, 1, 1.5, 2, 3, 4, 6; a scale
 * byte x stands for 2^(x - 127), 255 for NaN.  The reference caches in the
 * model's dtype only (serving_engine/model_runner.py:101-110).
 *
 * kvhot_reshape_and_cache_4bit: kvhot_reshape_and_cache into such a cache.  The
 * scale of 32 elements is the smallest power of two s with max|x| <= 7 s, held
 * to [2^-125, 2^125] (fp16: [2^-23, 2^13]); codes are rounded to nearest even,
 * magnitudes above 6 s to 6 s.  A group with an infinity or a NaN becomes NaN,
 * all 32 elements.  Slots must be distinct.
 * kvhot_read_cache_4bit: key[i], value[i] (contiguous [num_slots,
 * num_kv_heads, head_dim], 16-byte aligned) = what the cache holds at slots[i], exact in
 * every dtype for values appended from it (zeros for a slot outside the pool).
 * as_blocks: into kv-interleaved blocks instead, for an attention over the copies:
 * key is [num_slots / 16, num_kv_heads, 2, 16, head_dim] (K, then V; value is not
 * used), num_slots a multiple of 16, and NaN reads as 0 (kvhot_spread_nan_4bit).
 */
int kvhot_reshape_and_cache_4bit(
    const void* key, const int64_t key_strides[3], const void* value,
    const int64_t value_strides[3], void* cache, int64_t block_stride_bytes,
    const void* slot_mapping, int slot_is_int64, int64_t num_tokens,
    int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
    int64_t num_blocks, int dtype, void* stream);
int kvhot_read_cache_4bit(const void* cache, int64_t block_stride_bytes,
                          const void* slots, int slot_is_int64,
                          int64_t num_slots, int64_t num_kv_heads,
                          int64_t head_dim, int64_t block_size,
                          int64_t num_blocks, void* key, void* value,
                          int as_blocks, int dtype, void* stream);

/*
 * kvhot_paged_attention over a cache held in 4 bits: the same rows, masking
 * and results (out in q's dtype, lse natural-log fp32, both for every query of
 * every row; a query with no visible key gets out = 0 and lse = -inf), with
 * the cache's values entering as what they stand for.  attn_flags: KVHOT_CAUSAL or
 * 0.  max_q_len / max_k_len must bound q_lens / k_lens, sum_q_lens their sum
 * (total_query does; a closer bound launches fewer empty work-groups).  The workspace holds
 * the partials of key ranges cut across work-groups and needs no clearing;
 * calls that share one must be ordered on one stream.
 * A NaN in the cache reaches the queries that see it and no other.  Repeated calls give the
 * same bits.
 */
int64_t kvhot_paged_attention_4bit_workspace_bytes(
    int64_t num_rows, int64_t sum_q_lens, int64_t max_q_len,
    int64_t max_k_len, int64_t num_q_heads, int64_t num_kv_heads,
    int64_t head_dim, int dtype);
int kvhot_paged_attention_4bit(
    const void* q, const int64_t q_strides[3], const void* cache,
    int64_t block_stride_bytes, void* out, const int64_t out_strides[3],
    float* lse, const int64_t lse_strides[2], const int32_t* block_table,
    int64_t bt_row_stride, const int32_t* q_lens, const int32_t* k_lens,
    const int32_t* q_starts, const int32_t* q_pos_offsets, int64_t num_rows,
    int64_t total_query, int64_t sum_q_lens, int64_t max_q_len,
    int64_t max_k_len, int64_t num_q_heads, int64_t num_kv_heads,
    int64_t head_dim, int64_t block_size, int64_t num_blocks, float scale,
    int attn_flags, int dtype, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * For prompts that are attended over dense copies of their keys
 * (kvhot_read_cache_4bit with as_blocks, then kvhot_paged_attention): writes NaN
 * into the outputs of the queries that see a NaN of the cache.  Row r of the
 * arrays is row rows[r] of block_table; for each of its queries, a NaN in a
 * visible K makes its heads' out and lse NaN, one in a visible V the 32
 * elements of out that share its scale.
 */
int kvhot_spread_nan_4bit(
    const void* cache, int64_t block_stride_bytes, void* out,
    const int64_t out_strides[3], float* lse, const int64_t lse_strides[2],
    const int32_t* block_table, int64_t bt_row_stride, const int32_t* rows,
    const int32_t* q_lens, const int32_t* k_lens, const int32_t* q_starts,
    const int32_t* q_pos_offsets, int64_t num_rows, int64_t total_query,
    int64_t max_q_len, int64_t max_k_len, int64_t num_q_heads,
    int64_t num_kv_heads, int64_t head_dim, int64_t block_size,
    int64_t num_blocks, int attn_flags, int dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* KVHOT_LAYER_H */
