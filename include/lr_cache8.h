/*
 * lr_cache8.h -- the key / value cache in pages of lr_cache.h, in 8 bits: the pass that writes it, the attention that reads it, page
 * copies. Conventions, pool and batch as there, but for what is said here. Nothing of the reference stands behind these calls.
 *
 * Pages in 8 bits. k_pages and v_pages are e4m3 (OCP, finite) bytes, strides in bytes (multiples of 16; row_stride below 2^23), page_size
 * 16 or more. 16 rows of a page (r / 16 the same) and a head share a scale 2^(x - 127), x the byte at
 * k_scales + p * scale_page_stride + (r / 16) * HK + g, in v_scales likewise; an element stands for its e4m3 value times that. Between layers the
 * scales are scale_layer_stride apart. The scales of keys and values, and of layers, may lie side by side in one buffer, in any order;
 * two that share a byte are rejected, and so is a span of scales that meets the pages' or that of rows which the call reads or writes.
 *
 * lr_cache_append_f8 is lr_cache_append_bf16 into such pages (B at most 65,535). Keys and values are rounded once, from fp32, to the scale of
 * their 16 rows: the least 2^e with max|y| <= 448 * 2^e over the call's rows among them, e in [-100, 119], and where positions before
 * the call's lie among them no less than what is there: then those are rounded again to the new scale (exactly, but for values below
 * its 2^-6): a scale that drafted tokens raised does not fall again where they are not accepted and written over behind others. An
 * infinity or NaN is held as NaN and has no part in the scale; finite values beyond 448 * 2^119 are held as that. Tokens that are left
 * out have no part in the scale either. Rows behind the sequence's last position stay as they were, whatever their scale does.
 * Scales that the call finds in its 16 rows must be such as it writes (bytes 27 .. 246).
 *
 * lr_cache_attention_f8 is lr_cache_attention_bf16 over such pages: queries, probabilities and the output are bf16, sums fp32; the
 * values that the bytes stand for take part as they are. A scale byte of 255 stands for NaN. Where other bytes than append's make values
 * that are no normal numbers of bf16, they are infinite from 2^128 on, and off by at most 2^-126 (0, for one) below 2^-126.
 * A workgroup holds 1,024 entries of the table (3,840 with more than 64 rows of a kv head): the workspace grows past them as there.
 *
 * lr_cache_copy_pages_f8 copies pages and their scales, in two launches.
 *
 * An accepted branch of a drafted tree is appended again from its tokens' keys and values, with `positions` as before: rows of 8 bits
 * cannot move to other rows' scales without rounding again.
 */
#ifndef LR_CACHE8_H
#define LR_CACHE8_H

#include "lr_cache.h"

#ifdef __cplusplus
extern "C" {
#endif

int lr_cache_append_f8(const void* q, const void* k, const void* v, int64_t q_row_stride, int64_t k_row_stride, int64_t v_row_stride,
                       void* q_out, int64_t q_out_row_stride, void* k_pages, void* v_pages, int64_t page_stride, int64_t row_stride,
                       int64_t head_stride, int n_pages, int page_size, void* k_scales, void* v_scales, int64_t scale_page_stride,
                       const int* page_table, int64_t table_stride, int table_pages, const int* starts, const int* lens,
                       const int* positions, int B, int T, int H, int HK, const float* q_norm_w, const float* k_norm_w, int table_kind,
                       const void* table_a, const void* table_b, int64_t table_row_stride, int table_rows, int pairing, int rot_dim,
                       float eps, lr_stream_t stream);
size_t lr_cache_attention_f8_ws_bytes(int B, int T, int max_rows, int max_keys, int H, int HK, int page_size, int window, int sinks);
int lr_cache_attention_f8(const void* q, int64_t q_row_stride, void* out, int64_t out_row_stride, const void* k_pages, const void* v_pages,
                          int64_t page_stride, int64_t row_stride, int64_t head_stride, int n_pages, int page_size, const void* k_scales,
                          const void* v_scales, int64_t scale_page_stride, const int* page_table, int64_t table_stride, int table_pages,
                          const int* starts, const int* lens, int B, int T, int max_rows, int max_keys, int H, int HK,
                          const uint64_t* tree, int words, int window, int sinks, float scale, void* workspace, size_t workspace_bytes,
                          lr_stream_t stream);
int lr_cache_copy_pages_f8(void* k_pages, void* v_pages, int layers, int64_t layer_stride, int64_t page_stride, int64_t row_stride,
                           int64_t head_stride, int n_pages, int page_size, int HK, void* k_scales, void* v_scales,
                           int64_t scale_layer_stride, int64_t scale_page_stride, const int* src, const int* dst, int n,
                           lr_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* LR_CACHE8_H */
