// C entry point of the prefill attention (kernels and design notes: kush_attend.h).
#include "kush_attend.h"

#include "kushkash_amd_attend.h"

extern "C" int kush_attend(int head_dim, int dtype, const void* q, const void* k, const void* v, void* out, float* lse,
                           const int64_t* strides, const int32_t* cu_q, const int32_t* cu_k, int32_t n_q, int32_t n_k,
                           int64_t total_q, int32_t n_seqs, int32_t hkv, int32_t group, float scale, int32_t causal,
                           int32_t out_f32, int32_t waves, int32_t chunk, float* part_o, float* part_ml, void* stream) {
    return kush::attend_impl<kush::AttendArgs>("kush_attend", head_dim, dtype, q, k, v, out, lse, strides, cu_q, cu_k, n_q, n_k, total_q, n_seqs,
                       hkv, group, scale, causal, out_f32, waves, chunk, part_o, part_ml, stream);
}
