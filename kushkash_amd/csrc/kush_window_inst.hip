// Instantiations of the decode kernel with a window for one input dtype and one rot flag, chosen by the build
// (-DKUSH_INST_IN=float | _Float16 | kush::bf16_t, -DKUSH_INST_ROT=0 | 1): 2 and 4 waves, one or two page streams.
//
// o = sum of p_j v_j, p the softmax of scale q.k_j over the j < n with j >= n - window or j < sinks: the plain decode over the
// list of pages that hold such a j, hidden tokens of those pages masked. It reads what is seen and is bound as the plain
// decode is, by HBM, or by one launch's chain where there is little: 64 sequences of 20,000 - 32,768 tokens, 4,096 + 4 seen, int4,
// D 128, 28 q over 4 kv heads: the kernel 32 us, 4.9 TB/s of 157 MB (37 us a launch among others, a plain decode of as many
// tokens 34); 97 of up to 5,000, 1,111 seen, int8, D 64, 12 kv heads: 37 us; one sequence, 512 + 4 seen: 10.6 us.
#include "kush_decode.h"

#if !defined(KUSH_INST_IN) || !defined(KUSH_INST_ROT)
#error "build with -DKUSH_INST_IN=<dtype> -DKUSH_INST_ROT=<0|1>"
#endif

namespace kush {

template <int D, int BITS, typename IN, int NW, bool ROT>
int launch_window(dim3 grid, hipStream_t stream, const void* q, void* out, const void* cache, int64_t bs, int64_t hs,
                  const void* tail_k, const int32_t* tail_idx, const int32_t* block_table, const int32_t* seq_lens,
                  int64_t bt_stride, int bt_cols, int hkv, int group, float p2, float rs, int n_splits, float* part_ml,
                  float* part_o, int32_t* sync, const int32_t* seq_order, const void* app_k, const void* app_v,
                  int64_t app_ks, int64_t app_vs, int window, int sinks) {
    auto kern = group <= 8 ? decode_kernel<D, BITS, IN, NW, 2, ROT, false, 2, int, int>
                           : decode_kernel<D, BITS, IN, NW, 1, ROT, false, 2, int, int>;
    kern<<<grid, dim3(NW * WAVE), 0, stream>>>((const IN*)q, (IN*)out, (uint8_t*)cache, bs, hs, (IN*)tail_k, tail_idx,
                                               block_table, seq_lens, bt_stride, bt_cols, hkv, group, p2, rs, n_splits,
                                               part_ml, part_o, sync, seq_order, (const IN*)app_k, (const IN*)app_v,
                                               app_ks, app_vs, 1, window, sinks);
    return kush_check_launch("kush_window_decode");
}

namespace {

template <int D, int BITS, int NW>
void* launcher() {
    if constexpr (decode_fits<D, BITS, NW>())
        return reinterpret_cast<void*>(&launch_window<D, BITS, KUSH_INST_IN, NW, (KUSH_INST_ROT != 0)>);
    else
        return nullptr;
}

// taking their addresses instantiates the launchers (and their kernels) in this object
__attribute__((used)) void* const launchers[] = {
    launcher<64, 4, 2>(),  launcher<64, 4, 4>(),  launcher<64, 8, 2>(),  launcher<64, 8, 4>(),
    launcher<128, 4, 2>(), launcher<128, 4, 4>(), launcher<128, 8, 2>(), launcher<128, 8, 4>(),
    launcher<256, 4, 2>(), launcher<256, 4, 4>(), launcher<256, 8, 2>(), launcher<256, 8, 4>()};

}  // namespace
}  // namespace kush
