/* kushkash_amd: what surrounds the attention of a serving step (in kushkash_amd/libkushhip.so, csrc/kush_step.hip) -- its
 * index arrays, built on the GPU from the requests' lengths, and the next tokens, drawn from the logits. The conventions
 * of kushkash_amd.h (device pointers, hipStream_t as void*, 0 on success, -1 unsupported dtype, -2 bad arguments, -3 a
 * HIP error, the message in kush_last_error()). No entry point allocates or synchronizes.
 */
#ifndef KUSHKASH_AMD_STEP_H
#define KUSHKASH_AMD_STEP_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* A decode step's block table from an engine's token map: table[r][p] = req_to_token[req[r]][32 p] / 32 for 32 p <
 * seq_lens[r], else 0 (p < pages). req_to_token is int32 [map_rows, map_cols]; pages past its columns, and requests
 * outside its rows, count as none. req and seq_lens are int32, or int64 where wide_req / wide_lens. lens_out and slots_out
 * (each may be null): seq_lens and req as int32. */
int kush_block_table(const int32_t* req_to_token, int64_t map_row_stride, int64_t map_rows, int64_t map_cols,
                     const void* req, int32_t wide_req, const void* seq_lens, int32_t wide_lens, int64_t n_reqs,
                     int64_t pages, int32_t* table, int64_t table_row_stride, int32_t* lens_out, int32_t* slots_out,
                     void* stream);

/* The index arrays of a prefill step whose request r adds new_tokens[r] tokens to history[r] cached ones (pages of 32):
 *   q_start, key_start [n + 1]  running sums of the new tokens, and of the keys (kept history + new tokens)
 *   seq_lens [n]                history + new tokens
 *   job_seq, job_page [jobs]    (request, logical page) of every page that new tokens touch
 *   page_blk, page_dst [pages]  block, and first key row, of every full page of kept history
 *   tail_blk [tails], tail_info [tails][3]  of every request whose history ends inside a page: block; key row, tokens, slot
 *   new_dst, slot_map [tokens]  of every new token: its key row; its block * 32 + its row in the page (int64)
 * in request order. window 0: all history is kept. Else the pages between the first `sinks` tokens and the window of the
 * request's first new token are left out of the keys. jobs, pages, tails and tokens are the arrays' sizes; entries past
 * them are not written, and entries that the lengths do not reach are left as they were. Pages past bt_cols read as
 * block 0. Negative lengths count as 0. */
int kush_step_maps(const int32_t* new_tokens, const int32_t* history, const int32_t* slots, const int32_t* block_table,
                   int64_t bt_row_stride, int64_t bt_cols, int64_t n_reqs, int32_t window, int32_t sinks, int64_t jobs,
                   int64_t pages, int64_t tails, int64_t tokens, int32_t* q_start, int32_t* key_start, int32_t* seq_lens,
                   int32_t* job_seq, int32_t* job_page, int32_t* page_blk, int32_t* page_dst, int32_t* tail_blk,
                   int32_t* tail_info, int32_t* new_dst, int64_t* slot_map, void* stream);

/* One token per row of logits [rows, vocab] (dtype 0 fp32, 1 fp16, 2 bf16; element row stride) and random number
 * uniforms[r] in [0, 1). With the row's tokens in the order of (logit descending, index ascending), max the largest logit
 * and w = exp((logit - max) / temperature):
 *   top_k > 0    the first top_k tokens are kept
 *   top_p < 1    of those, the tokens that have less than top_p of their mass before them
 *   min_p > 0    of those, the tokens with w >= min_p
 * the first token always. out[r] is the first index whose running sum of kept w, in the vocabulary's order, exceeds
 * uniforms[r] times the sum of all (1 and more: the last kept one; NaN and less than 0 count as 0). temperature 0: the first of the order. A row with a NaN, or with no logit above
 * -inf: -1. w is held in multiples of 2^-min(50, 63 - log2 vocab), one at least where it is above 0. The parameters are one value for all rows, or (pointer not null) one per row. scratch: kush_sample_scratch(rows,
 * vocab) bytes, 16-byte aligned, of any contents, this call's own until it has run. */
int64_t kush_sample_scratch(int64_t rows, int64_t vocab);
int kush_sample(int dtype, const void* logits, int64_t row_stride, int64_t rows, int64_t vocab, const float* uniforms,
                double temperature, const float* temperatures, int32_t top_k, const int32_t* top_ks, double top_p,
                const float* top_ps, double min_p, const float* min_ps, int64_t* out, void* scratch, int64_t scratch_bytes,
                void* stream);

#ifdef __cplusplus
}
#endif

#endif
