/* rdl_attention.h -- the cache side of a step that serves several sequences on
 * one MI355X (librdlquant.so): page tables and slots, RoPE with the cache
 * write, and causal attention over a paged cache or over packed prompts.
 *
 * The rustml counterparts work on one sequence at a time:
 *   KVCache (append, views)               rustml/nn/main/src/core/kv_cache.rs:10-114
 *   RoPEFreqs::apply                      rustml/nn/main/src/core/rope.rs:134-200
 *   MultiHeadAttention::forward_with_cache rustml/nn/main/src/core/attention.rs:353-449
 * Here the rows of a step belong to n_seq sequences, packed one behind the
 * other: sequence b brings new_b >= 0 rows behind cached_b positions that the
 * cache holds already, its rows are row_start[b] .. row_start[b + 1] - 1, and
 * afterwards it has kv_len[b] = cached_b + new_b positions.  Positions live in
 * pages of page_positions; sequence b's page table row maps position p to
 * physical page table[b][p / page_positions].  The same rows serve a decode
 * step (every new_b = 1), prompt chunks, and any mix of both.
 *
 * Conventions are rdl_quant.h's device entry points': device pointers, a
 * hipStream_t of the current device passed as void* (another device's stream:
 * RDL_ERR_INVALID_DATA), stream-ordered, no synchronisation; lengths, tables
 * and slots are read on the device, so a captured graph follows their contents
 * at each replay.  Activations are f32, the cache f16 or f32.  Work memory
 * (the attention's partial results of split key ranges, at most 256 MB, and, for
 * long packed f32 prompts, 16-bit parts of their k and v, at most about 1 GB) is the
 * stream's, as rdl_linear_forward_dev describes (rdl_release_stream_work frees
 * it); under graph capture the graph owns it.  Steps of more than 2^24 - 1
 * workgroups (a sequence has one a KV head at least, or one a KV head for 128
 * pairs of row and query head of a group) are RDL_ERR_UNSUPPORTED.
 * What device-side arrays hold is never trusted with an address: page numbers,
 * slots and positions outside their array are skipped, row numbers and lengths
 * are cut to m and to the table's width.  Inference only: there is no backward
 * pass in this library. */
#ifndef RDL_ATTENTION_H
#define RDL_ATTENTION_H

#include <stddef.h>
#include <stdint.h>

#include "rdl_quant.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Cache element types: GGML type ids (rustml/gguf/main/src/api/types.rs:5-20), and
 * one of this library's own, RDL_KV_Q4: 4 bits and a share of a scale, 4.5 bits a
 * value.  32 consecutive values of a position and KV head are a block of a scale
 * d and codes 0 .. 15, value = d (code - 8).  d has the size of the block's largest
 * magnitude over 8, rounded to 8 significant bits, as f16, at most 8160, and the sign
 * that takes that value to code 0 (of a positive and a negative one as large, the
 * positive; zeros are positive); a code is value / d rounded to nearest, halves to even,
 * between -8 and 7, plus 8; where d rounds to 0 (magnitudes up to 2^-22) the codes are 8.  A
 * block that holds a value that is not finite reads as NaN (d is NaN, its codes unspecified).  With such a
 * scale every value is an f16 number; with one of more bits it is rounded to f16.
 * A page of a head is one run of bytes: page_positions * head_dim / 2 of codes,
 * then page_positions * head_dim / 32 f16 scales, positions in order.  In each
 * 4 bytes of codes, as a little-endian word, codes 0, 2, 4, 6 of 8 are the nibbles of the
 * low half and 1, 3, 5, 7 those of the high half, from the lowest bits up. */
enum {
    RDL_DTYPE_F32 = 0,
    RDL_DTYPE_F16 = 1,
    RDL_KV_Q4 = 0x104
};

/* A layer's paged K and V memory.  Element d of position o of page pg and KV
 * head h is at pg * page_stride + h * head_stride + o * position_stride + d of
 * k_dev and of v_dev (strides in elements; multiples of 16 bytes, as both
 * bases; position_stride below 2^24; the heads and positions of a page and the
 * pages must not overlap).
 * The decoder's own pools are [n_pages][n_kv_heads][page_positions][head_dim].
 * RDL_KV_Q4: strides in bytes (multiples of 16), position_stride = head_dim / 2,
 * head_dim a multiple of 32. */
typedef struct rdl_kv_pool {
    void* k_dev;
    void* v_dev;
    int32_t dtype;          /* RDL_DTYPE_F16, RDL_DTYPE_F32 or RDL_KV_Q4 */
    int32_t n_pages;
    int32_t page_positions; /* a power of two, 16 .. 1024 */
    int32_t n_kv_heads;
    int32_t head_dim;       /* a multiple of 8, 8 .. 256 */
    int64_t page_stride;
    int64_t head_stride;
    int64_t position_stride;
} rdl_kv_pool;

/* What rdl_kv_plan_dev found wrong (summary[2], 0: nothing). */
enum {
    RDL_PLAN_BAD_LENGTH = 1, /* a negative length (taken as 0), or one past 2^31 - 1 (cut) */
    RDL_PLAN_TABLE_FULL = 2, /* a sequence needs more pages than its table row has entries */
    RDL_PLAN_NO_PAGES = 4,   /* the free list is shorter than the pages needed */
    RDL_PLAN_NO_ROWS = 8     /* the step's rows are more than m */
};

/* Block tables, row starts, positions and slots of a step, from the lengths of
 * its sequences, in one launch.  Inputs (int32, device): cached [n_seq] and
 * new_rows [n_seq]; free_pages [n_free], physical pages no sequence holds;
 * tables [n_seq][table_stride], whose first ceil(cached_b / page_positions)
 * entries are filled.  Each sequence, in order, takes the pages it needs
 * beyond those from the front of the free list.  Outputs (int32, device):
 *   tables        the entries of the new pages (no others are written);
 *   row_start     [n_seq + 1];    kv_len  [n_seq];
 *   row_seq, positions, slots     [m]: the row's sequence, its position in it
 *                 and page * page_positions + offset of that position
 *                 (-1 past 2^31 - 1);
 *   summary       [4]: rows of the step, pages taken from the free list,
 *                 RDL_PLAN_* flags, the longest kv_len.
 * Rows row_start[n_seq] .. m - 1 of a padded batch get sequence -1, position 0
 * and slot -1.  Pages that are missing (TABLE_FULL, NO_PAGES) are -1 in the
 * table and in the slots of their rows, which the calls below then skip.
 * page_positions: a power of two, 16 .. 1024.  Outputs must not overlap. */
rdl_status rdl_kv_plan_dev(const int32_t* cached_dev, const int32_t* new_rows_dev, size_t n_seq,
                           const int32_t* free_pages_dev, size_t n_free, size_t page_positions, int32_t* tables_dev,
                           size_t table_stride, int32_t* row_start_dev, int32_t* kv_len_dev, size_t m,
                           int32_t* row_seq_dev, int32_t* positions_dev, int32_t* slots_dev, int32_t* summary_dev,
                           void* stream);

/* RoPE of a step's q and k rows (RoPEFreqs::apply, half-split pairs (i, i +
 * head_dim / 2)) and the write of its k and v rows into the pool (KVCache::
 * update), in one launch.  Row r of q (n_heads heads), k and v (the pool's KV
 * heads) starts r * stride floats behind its base, heads head_dim apart;
 * strides and bases are multiples of 16 bytes.  q_out rows may be the q rows
 * themselves (the same base and stride) and may not overlap them otherwise,
 * nor the k and v rows (RDL_ERR_INVALID_DATA) or the pool; n_heads = 0: no q.
 * positions (NULL without RoPE) select the rows of cos and sin
 * [n_positions][head_dim / 2] f32; cos and sin NULL: no RoPE, q is copied.
 * slots: page * page_positions + offset.  A row whose slot is negative or past
 * the pool, or whose position is outside the tables, is left out: nothing of it
 * is written.  The slots of two rows must differ. */
rdl_status rdl_kv_store_dev(const rdl_kv_pool* pool, size_t m, const float* q_dev, size_t q_stride, float* q_out_dev,
                            size_t q_out_stride, size_t n_heads, const float* k_dev, size_t k_stride,
                            const float* v_dev, size_t v_stride, const int32_t* positions_dev,
                            const int32_t* slots_dev, const float* cos_dev, const float* sin_dev, size_t n_positions,
                            void* stream);

/* The same with an RMS norm of every query and key head before its rotation
 * (MultiHeadAttention's q_norm and k_norm, rustml/nn/main/src/core/attention.rs):
 *   y = (x * r) * gamma,  r = 1 / sqrt(mean(x^2) + eps) over the head's values,
 * the mean square in 64 bits, r rounded to f32.  q_gamma and k_gamma: [head_dim] f32,
 * 16-byte aligned, the same for all heads; NULL: no norm of those rows.  eps is
 * finite and not negative.  Products and sums of the norm and of the rotation are
 * rounded one by one (rdl_kv_store_dev fuses a product with its sum, except over a 4-bit pool).  Otherwise as
 * rdl_kv_store_dev. */
rdl_status rdl_kv_store_norm_dev(const rdl_kv_pool* pool, size_t m, const float* q_dev, size_t q_stride,
                                 float* q_out_dev, size_t q_out_stride, size_t n_heads, const float* k_dev,
                                 size_t k_stride, const float* v_dev, size_t v_stride, const float* q_gamma_dev,
                                 const float* k_gamma_dev, float eps, const int32_t* positions_dev,
                                 const int32_t* slots_dev, const float* cos_dev, const float* sin_dev,
                                 size_t n_positions, void* stream);

/* What rdl_kv_fork_dev found wrong (summary[1], 0: nothing). */
enum {
    RDL_FORK_BAD_SEQUENCE = 1, /* a parent or child that is no sequence, or a parent that is its own child: the pair is left out */
    RDL_FORK_BAD_LENGTH = 2,   /* a parent's length that is negative (taken as 0) or past its table row (cut) */
    RDL_FORK_NO_PAGES = 4      /* the free list is shorter than the pages needed */
};

/* Forks sequences over shared pages: for each of n pairs (int32,
 * device) the sequence children[i] becomes a copy of parents[i].  Its table
 * row names the parent's pages, except that a last page that is not full is the
 * child's own: the next page of the free list, and -1 where that is used up.  src_pages
 * and dst_pages [n] receive the pages to copy, the parent's last and the child's
 * own (-1, -1: none), for rdl_kv_copy_pages_dev on every layer.
 *   tables [n_seq][table_stride], kv_len [n_seq]: the children's rows (as far as
 *                 the parent's length) and lengths are written;
 *   summary [2]:  pages taken from the free list, RDL_FORK_* flags.
 * Several children of one parent are its copies with a page of their own
 * each.  All pairs go by the parents' lengths from before the call.  A child may not be another
 * pair's parent or child: the row of a sequence that two pairs name so, and what is copied from it
 * (the row, length and src_pages entry of its own children), are unspecified; other pairs, all of
 * dst_pages and the summary are what those lengths make them.
 * Full pages are shared: the caller frees a page when no sequence names it.
 * page_positions: a power of two, 16 .. 1024.  Outputs must not overlap. */
rdl_status rdl_kv_fork_dev(int32_t* tables_dev, size_t table_stride, int32_t* kv_len_dev, size_t n_seq,
                           size_t page_positions, const int32_t* parents_dev, const int32_t* children_dev, size_t n,
                           const int32_t* free_pages_dev, size_t n_free, int32_t* src_pages_dev,
                           int32_t* dst_pages_dev, int32_t* summary_dev, void* stream);

/* Copies whole pages, K and V of every KV head, for n_pools (src, dst) pairs of pools
 * at once (a model's layers): page src_pages[i] of src[l] to page dst_pages[i] of
 * dst[l], i < n (int32, device).  A pair with a page outside its pool is left out.  src
 * and dst may be the same pools (a fork, compaction) or others of the same pages,
 * heads and head_dim in any types and strides: values of another type are rounded
 * to nearest (f16: past its range infinite; 4 bits as RDL_KV_Q4 says), those of the same type are
 * copied bit by bit.  All src pools agree in everything but their addresses, and so do
 * all dst pools (RDL_ERR_INVALID_DATA).  dst pages differ from one another, and
 * in the same pool none is also a pair's src, unless it is its own (its contents are
 * then unspecified); pools that are not the same must not overlap. */
rdl_status rdl_kv_copy_pages_dev(const rdl_kv_pool* src, const rdl_kv_pool* dst, size_t n_pools,
                                 const int32_t* src_pages_dev, const int32_t* dst_pages_dev, size_t n, void* stream);

/* Causal attention of a step's rows over the paged cache, which holds the
 * rows' own keys already: row i of sequence b's new_b = row_start[b + 1] -
 * row_start[b] rows sees the keys 0 .. kv_len[b] - new_b + i, and
 *   out = sum_j softmax_j(scale * q . k_j) v_j
 * per query head, head h reading KV head h / (n_heads / n_kv_heads); scale is
 * finite and positive (1 / sqrt(head_dim) in the reference).  A row that sees
 * no key gives zeros, and a key on a page that is not in the pool counts as
 * not seen.  Rows row_start[n_seq] .. m - 1 of out are left as they were.
 * q and out: f32 rows stride floats apart (n_heads * head_dim or more, a
 * multiple of 4; bases 16-byte aligned); out must not overlap q (RDL_ERR_INVALID_DATA),
 * the pool or the int arrays.
 * row_start ascends; where it does not, what the call's rows get is unspecified.
 * What a row does not see has no effect on it, NaN and infinities included.  Of
 * what it sees, a NaN in a key or in its query makes its outputs NaN, values that are
 * not finite make that element their sum whatever their weights (infinite, or NaN for
 * a NaN or both infinities), and infinite keys or queries, or scores past f32's range,
 * leave its outputs unspecified.
 * max_rows and max_kv tell the launch what to expect (the most rows of a
 * sequence, the longest kv_len; 0: unknown): results do not depend on them
 * beyond rounding, time does.  Products are formed on the matrix cores with
 * f32 sums from f16 pairs: with f16 keys and values, and 4-bit ones, which are exact in f16, they
 * carry 22 bits of q and of the weights; with f32 ones 23 bits of those and of
 * keys and values.  Sums, maxima and exponents are f32.
 * Errors are then about those of plain f32 sums and products.  What pairs cannot
 * hold: f32 elements far below the largest of their row end at 2^-38 of that in
 * queries and at 2^-33 in keys, and in values at 2^-28 of the largest of their
 * row or of the rows a query weighs with it.
 * n_heads must be a multiple of the pool's n_kv_heads. */
rdl_status rdl_attention_paged_dev(const rdl_kv_pool* pool, const float* q_dev, size_t q_stride, size_t n_heads,
                                   size_t m, const int32_t* row_start_dev, const int32_t* kv_len_dev, size_t n_seq,
                                   const int32_t* tables_dev, size_t table_stride, float scale, float* out_dev,
                                   size_t out_stride, size_t max_rows, size_t max_kv, void* stream);

/* Causal attention of whole prompts packed one behind the other, without a
 * cache (MultiHeadAttention::forward, attention.rs): sequence b's rows
 * row_start[b] .. row_start[b + 1] - 1 see one another up to their own place.
 * k and v rows are kv_dtype (f32 as a Linear leaves them, or f16), stride
 * elements apart (multiples of 16 bytes, as the bases), heads head_dim apart;
 * out must not overlap them either (RDL_ERR_INVALID_DATA).  Otherwise as
 * rdl_attention_paged_dev. */
rdl_status rdl_attention_packed_dev(const float* q_dev, size_t q_stride, size_t n_heads, const void* k_dev,
                                    size_t k_stride, const void* v_dev, size_t v_stride, int32_t kv_dtype,
                                    size_t n_kv_heads, size_t head_dim, size_t m, const int32_t* row_start_dev,
                                    size_t n_seq, float scale, float* out_dev, size_t out_stride, size_t max_rows,
                                    void* stream);

#ifdef __cplusplus
}
#endif

#endif
