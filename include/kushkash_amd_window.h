/* kushkash_amd attention with a window (in kushkash_amd/libkushhip.so): the query at position p of a sequence sees, of
 * the keys 0 .. p, the last `window` (its own among them) and the first `sinks` -- what a sliding-window model computes,
 * and what keeps a full-attention model going past the context that its cache is to hold. The conventions of
 * kushkash_amd.h (device pointers, hipStream_t as void*, 0 on success, -1 unsupported head_dim, bits or dtype, -2 bad
 * arguments, -3 a HIP error, the message in kush_last_error()). window >= 1, sinks >= 0.
 */
#ifndef KUSHKASH_AMD_WINDOW_H
#define KUSHKASH_AMD_WINDOW_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* kush_decode_ex under a window: each sequence's query is its newest token (position seq_lens[s] - 1). With k and v (row
 * s the token at that position, rows 16-byte aligned, group <= 16) the token is appended first, as kush_append_decode
 * does; both null: the cache holds it already. Only the pages that are seen are read, and only their block_table
 * entries (with bt_cols > 0 the other entries of a row are loaded too, and not used): a page between the sinks and the
 * window may hold anything, or another sequence's tokens. n_splits counts over the pages that are seen. waves: 0, 2 or 4 (8 runs 4). */
int kush_window_decode(int head_dim, int bits, int group, int dtype, const void* q, void* out, void* cache,
                       int64_t block_stride, int64_t head_stride, void* tail_k, const int32_t* tail_idx,
                       const int32_t* block_table, const int32_t* seq_lens, int64_t bt_row_stride, int32_t hkv,
                       float scale, int32_t n_splits, float* part_ml, float* part_o, int32_t n_seqs, void* stream,
                       const void* k, const void* v, int64_t k_row_stride, int64_t v_row_stride, int32_t bt_cols,
                       int32_t* split_sync, int32_t waves, const int32_t* seq_order, int32_t rot, int32_t window,
                       int32_t sinks);

/* kush_attend (kushkash_amd_attend.h) of queries that are the last of their keys, under a window: query row t of a
 * sequence with T rows and N >= T keys is position N - T + t. Keys left out of the rows between the sinks and the first
 * query's window change nothing, as long as they are whole: positions count in the rows given. Splits: of the tiles that a
 * row tile sees. row_tiles, for ragged rows: the sum over the sequences of ceil(rows * group / (32 * waves)), which the
 * lengths on the host give -- as many workgroups per kv head are launched; 0: as many for every sequence as the longest needs. */
int kush_window_attend(int head_dim, int dtype, const void* q, const void* k, const void* v, void* out, float* lse,
                       const int64_t* strides, const int32_t* cu_q, const int32_t* cu_k, int32_t n_q, int32_t n_k,
                       int64_t total_q, int32_t n_seqs, int32_t hkv, int32_t group, float scale, int32_t out_f32,
                       int32_t waves, int32_t chunk, float* part_o, float* part_ml, void* stream, int32_t window,
                       int32_t sinks, int32_t row_tiles);

#ifdef __cplusplus
}
#endif

#endif
