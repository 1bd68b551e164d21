// mirec_sample with replacement: see sample_kernel.h.
#include "sample_kernel.h"

namespace mirec {

int sample_with_replacement(const void* scores, int dtype, int64_t n, int64_t m, int64_t stride, const int32_t* ids, int64_t ids_stride,
                             const int64_t* mask_indptr, const int32_t* mask_indices, const float* uniforms, int draws,
                             const SampleParams& par, int bits, int32_t* out_ids, float* out_logprob, hipStream_t stream) {
    return launch_sample<true>(scores, dtype, n, m, stride, ids, ids_stride, mask_indptr, mask_indices, uniforms, draws, par, bits, out_ids,
                               out_logprob, stream);
}

}  // namespace mirec
