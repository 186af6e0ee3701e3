// C entry point of the prefill attention under a window (kernels and design notes: kush_attend.h).
#include "kush_attend.h"

#include "kushkash_amd_window.h"

extern "C" int kush_window_attend(int head_dim, int dtype, const void* q, const void* k, const void* v, void* out, float* lse,
                                  const int64_t* strides, const int32_t* cu_q, const int32_t* cu_k, int32_t n_q, int32_t n_k,
                                  int64_t total_q, int32_t n_seqs, int32_t hkv, int32_t group, float scale, int32_t out_f32,
                                  int32_t waves, int32_t chunk, float* part_o, float* part_ml, void* stream, int32_t window,
                                  int32_t sinks, int32_t row_tiles) {
    if (window <= 0 || sinks < 0 || row_tiles < 0 || (row_tiles > 0 && cu_q == nullptr) || (int64_t)row_tiles * hkv > 0x7fffffff)
        return kush_fail(-2, "kush_window_attend: bad window %d / sinks %d / row_tiles %d", window, sinks, row_tiles);
    return kush::attend_impl<kush::WindowArgs>("kush_window_attend", head_dim, dtype, q, k, v, out, lse, strides, cu_q, cu_k, n_q, n_k,
                       total_q, n_seqs, hkv, group, scale, 1, out_f32, waves, chunk, part_o, part_ml, stream, window, sinks,
                                               n_seqs, row_tiles);
}
