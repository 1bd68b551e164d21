// mirec_sample: checks, and what the kernels take as parameters (sample_kernel.h).
#include <cmath>

#include "sample_kernel.h"

namespace mirec {

// Fraction bits of a weight: the sum of m of them stays below 2^62.
static int sample_bits(int64_t m) {
    int b = 0;
    while (((int64_t)1 << b) < m) ++b;
    return 62 - b < 51 ? 62 - b : 51;
}

// The least sum of weights that is drawn from: m roundings of half a unit are 2^-24 of it at most (up to 2^19 items; beyond,
// half the largest weight, which the best item has).
static uint64_t sample_renew_below(int64_t m, int bits) {
    int b = 0;
    while (((int64_t)1 << b) < m) ++b;
    return 1ull << (b + 23 < bits - 1 ? b + 23 : bits - 1);
}

}  // namespace mirec

extern "C" int mirec_sample(const void* scores, int dtype, int64_t n, int64_t m, int64_t row_stride, const int32_t* ids,
                            int64_t ids_stride, const int64_t* mask_indptr, const int32_t* mask_indices,
                            const float* uniforms, int draws, int replacement, double temperature,
                            const float* row_temperature, int32_t top_k, const int32_t* row_top_k, double top_p,
                            const float* row_top_p, double min_p, const float* row_min_p, int32_t* out_ids,
                            float* out_logprob, mirec_stream_t stream_) {
    using namespace mirec;
    hipStream_t stream = (hipStream_t)stream_;
    MIREC_REQUIRE(n >= 0 && m >= 0 && draws >= 0, MIREC_E_INVALID, "mirec_sample: negative size");
    MIREC_REQUIRE(dtype == MIREC_F32 || dtype == MIREC_F16 || dtype == MIREC_BF16, MIREC_E_INVALID,
                  "mirec_sample: unknown score type %d", dtype);
    MIREC_REQUIRE(draws <= SM_MAX_DRAWS, MIREC_E_UNSUPPORTED, "mirec_sample: %d draws a row; at most %d are supported",
                  draws, SM_MAX_DRAWS);
    MIREC_REQUIRE(m <= ((int64_t)1 << 30), MIREC_E_UNSUPPORTED, "mirec_sample: more than 2^30 items");
    MIREC_REQUIRE(row_temperature || (temperature >= 0.0 && temperature < INFINITY), MIREC_E_INVALID,
                  "mirec_sample: temperature must be finite and not negative (got %g)", temperature);
    MIREC_REQUIRE(row_top_p || (top_p >= 0.0 && top_p <= 1.0), MIREC_E_INVALID,
                  "mirec_sample: top_p must lie in [0, 1] (got %g)", top_p);
    MIREC_REQUIRE(row_min_p || (min_p >= 0.0 && min_p <= 1.0), MIREC_E_INVALID,
                  "mirec_sample: min_p must lie in [0, 1] (got %g)", min_p);
    MIREC_REQUIRE(row_top_k || top_k >= 0, MIREC_E_INVALID, "mirec_sample: top_k must not be negative (got %d)", top_k);
    if (n == 0 || draws == 0) return MIREC_OK;
    MIREC_REQUIRE((scores || m == 0) && uniforms && out_ids && out_logprob, MIREC_E_INVALID, "mirec_sample: null argument");
    MIREC_REQUIRE(row_stride >= 0 && ids_stride >= 0, MIREC_E_INVALID, "mirec_sample: negative row stride");
    MIREC_REQUIRE(((uintptr_t)scores & (dtype == MIREC_F32 ? 3 : 1)) == 0, MIREC_E_INVALID,
                  "mirec_sample: scores are not aligned to their type");
    MIREC_REQUIRE(!(ids && mask_indptr), MIREC_E_INVALID, "mirec_sample: a filter names items by position: not with ids");
    MIREC_REQUIRE(!mask_indptr || m <= SM_MAX_MASKED_ITEMS, MIREC_E_UNSUPPORTED,
                  "mirec_sample: a filter over %lld items; at most %lld are supported", (long long)m,
                  (long long)SM_MAX_MASKED_ITEMS);
    SampleParams par = {};
    par.greedy = !(temperature >= SM_MIN_TEMPERATURE);
    par.step = par.greedy ? 0.0 : 1.4426950408889634 / temperature;
    par.top_p = top_p;
    par.top_k = top_k;
    par.row_temperature = row_temperature;
    par.row_top_k = row_top_k;
    par.row_top_p = row_top_p;
    par.row_min_p = row_min_p;
    const int bits = sample_bits(m);
    par.floor_w = (uint64_t)std::ceil(min_p * (double)(1ull << bits));
    par.renew_below = sample_renew_below(m, bits);
    return (replacement ? sample_with_replacement : sample_without_replacement)(
        scores, dtype, n, m, row_stride, ids, ids_stride, mask_indptr, mask_indices, uniforms, draws, par, bits, out_ids, out_logprob, stream);
}
