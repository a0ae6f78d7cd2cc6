/*
 * lr_cache.h -- a key / value cache in pages: the pass that writes it, the attention that reads it, copies and moves of its
 * rows. Plain C ABI, gfx950; conventions as lr_attn.h (bf16 rows of 128, strides in elements, asynchronous on the caller's
 * stream, no allocation, no state, 0 or a hipError_t). The reference keeps keys and values of a prefix in rows only
 * (src/engines/qwen_image/dit.zig:352-370); nothing of it stands behind these calls.
 *
 * The pool. k_pages and v_pages hold n_pages pages of page_size rows (a power of two) of HK heads each: row r of page p of
 * head g at base + p * page_stride + r * row_stride + g * head_stride, in both the same strides (multiples of 8 elements, the
 * head's 128 elements contiguous). Rows of one page may lie token by token (head_stride 128) or head by head.
 * Calls over layers take base + l * layer_stride for layer l; pages have the same number in every layer. Keys and values, and
 * layers, may interleave in one buffer; those that share a row, or part of one, are rejected.
 *
 * A batch. Sequence b < B has the tokens starts[b] .. starts[b + 1] - 1 of the call's T (n_b of them; int32 [B + 1] on the
 * device, ascending) and lens[b] positions in all (int32 [B]), the call's tokens being its last ones: the first of them at
 * position c_b = lens[b] - n_b. Position j lies in row j % page_size of page page_table[b * table_stride + j / page_size]
 * (int32, table_pages entries a sequence). An entry outside [0, n_pages) holds no rows: nothing is written there, and its
 * positions are not seen. Tokens at and behind starts[B], if T is larger, are left out: their output rows stay as they were.
 * starts, lens and the tables are read by the kernels: a captured call follows what they hold at its replay.
 * Pages of 8 bits: lr_cache8.h.
 */
#ifndef LR_CACHE_H
#define LR_CACHE_H

#include "lr_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * New tokens into the cache in one pass: q [T][H][128], k and v [T][HK][128] rows (views of one packed projection qualify).
 * Queries and keys are normalised per head and rotated as lr_joint_q_prepare does (y = x / sqrt(mean(x^2) + eps) * w in fp32,
 * fp32 weights [128] or NULL for ones, table_kind LR_TABLE_*, pairs LR_PAIR_*, rot_dim; LR_PAIR_SPLIT_HALF: rot_dim % 16 ==
 * 0), rounded once to bf16; queries go to q_out rows, keys to the tokens' positions in the pages, values there as they are.
 * A token is rotated by table row positions[t] (int32 [T]), or without positions (NULL) by the row of its position in its
 * sequence; a token whose row is not one of the table's table_rows, or whose position the sequence's table or the pool does
 * not have, is left out whole. q NULL: keys and values only (q_out is not used). q_out may be q itself (same stride; k and v in
 * other columns of the same rows, if they are views of one projection); otherwise it must not overlap q, k or v. The pool must not
 * overlap q, k, v or q_out (all rejected).
 */
int lr_cache_append_bf16(const void* q, const void* k, const void* v, int64_t q_row_stride, int64_t k_row_stride,
                         int64_t v_row_stride, void* q_out, int64_t q_out_row_stride, void* k_pages, void* v_pages,
                         int64_t page_stride, int64_t row_stride, int64_t head_stride, int n_pages, int page_size,
                         const int* page_table, int64_t table_stride, int table_pages, const int* starts, const int* lens,
                         const int* positions, int B, int T, int H, int HK, const float* q_norm_w, const float* k_norm_w,
                         int table_kind, const void* table_a, const void* table_b, int64_t table_row_stride, int table_rows,
                         int pairing, int rot_dim, float eps, lr_stream_t stream);

/*
 * Attention of the batch's tokens over their sequences' pages (keys and values of the tokens themselves included: append
 * first). The token at position p sees j <= p: one token a sequence (a decode step), or a chunk.
 * tree != NULL: drafted tokens. tree [T][words] of 64 bits: a token sees every position below c_b, and the drafted position
 * c_b + x when bit x (word x / 64) of its words is set (its own bit too, if it is to see itself). Its position is c_b plus
 * the number of its bits less one.
 * window >= 1: of the positions below its own (under a tree: below c_b) a token at p sees those with p - j < window or
 * j < sinks. window 0: all.
 * A token that sees nothing gets zeros; a position that it does not see has no part in its result, whatever it holds.
 * max_rows: no sequence has more tokens in the call (those beyond are left out, under a tree as keys too); max_keys: no
 * sequence has more positions (those beyond are not seen). Both size the launch: a max_rows far above the tokens of any sequence
 * launches workgroups without rows for every sequence, and one that makes more of them than a grid holds (2^22) is rejected. At
 * most 2^30 positions; B at most 65,535.
 * workspace: lr_cache_attention_ws_bytes bytes for the same numbers (0: none, it may be NULL; fewer rows or positions may take
 * more; up to 273 MB, but where max_keys takes more entries of the table than a workgroup holds, 2,048, every row takes 520 bytes for
 * each part of as many), 256-byte aligned; it must not overlap q, out or the pool, nor out q or the pool (rejected). What it holds
 * before the call does not matter. Calls that overlap in time on one workspace race.
 */
size_t lr_cache_attention_ws_bytes(int B, int T, int max_rows, int max_keys, int H, int HK, int page_size, int window,
                                   int sinks);
int lr_cache_attention_bf16(const void* q, int64_t q_row_stride, void* out, int64_t out_row_stride, const void* k_pages,
                            const void* v_pages, int64_t page_stride, int64_t row_stride, int64_t head_stride, int n_pages,
                            int page_size, const int* page_table, int64_t table_stride, int table_pages, const int* starts,
                            const int* lens, int B, int T, int max_rows, int max_keys, int H, int HK, const uint64_t* tree,
                            int words, int window, int sinks, float scale, void* workspace, size_t workspace_bytes,
                            lr_stream_t stream);

/*
 * Pages copied inside the pool, in every layer: page src[i] to page dst[i] for i < n (int32 on the device). A pair with a page
 * outside the pool is left out. No page may be the target of one pair and in another pair at all, source or target (a page
 * may be the source of several): such pairs leave either page's old or new rows.
 */
int lr_cache_copy_pages(void* k_pages, void* v_pages, int layers, int64_t layer_stride, int64_t page_stride,
                        int64_t row_stride, int64_t head_stride, int n_pages, int page_size, int HK, const int* src,
                        const int* dst, int n, lr_stream_t stream);

/*
 * Rows moved inside their sequences, in every layer: for the moves starts[b] .. starts[b + 1] - 1 of sequence b (n in all, at
 * most max_rows <= 256 a sequence: those beyond are left out), position src[i] to position dst[i]. All of a sequence's rows
 * are read before any is written, so the moves of a sequence may chain or swap. No position may be the target of two moves of a
 * sequence: each of its heads' keys and values would be either one's, not all of them the same one's. Moves with a position that
 * the table or the pool does not have are left out. Sequences that share pages must not move rows of those.
 */
int lr_cache_move_rows(void* k_pages, void* v_pages, int layers, int64_t layer_stride, int64_t page_stride,
                       int64_t row_stride, int64_t head_stride, int n_pages, int page_size, int HK, const int* page_table,
                       int64_t table_stride, int table_pages, const int* starts, const int* src, const int* dst, int B, int n,
                       int max_rows, lr_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* LR_CACHE_H */
