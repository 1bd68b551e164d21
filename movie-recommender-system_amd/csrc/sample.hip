// Drawing items from rows of scores: softmax at a temperature, cut to the k best, to the shortest best-first prefix
// that holds a share top_p of the mass and to the items at least min_p times as likely as the best, then one inverse
// look-up in the running sum per given random number.  The stochastic counterpart of the top-K pass that
// recommenders/als_recommender.py:181-186 serves: it takes that pass's ranked lists or dense rows of scores.
//
// The order of a row is (score descending, index ascending), as in the top-K kernels; all three cuts keep a prefix of
// it, so what is kept is described by one threshold key and by how many of the items that tie with it stay.  Weights
// are 64-bit fixed-point numbers, w_i = rint(2^S exp((s_i - max s) / T)): integer sums do not depend on the order they
// are formed in, so a histogram by atomics, a split row and a scan give the same bits on every run, and a running sum
// of 27 000 weights is exact where fp32 would move its borders by more than the width of an unlikely item.
#include <float.h>
#include <hip/hip_fp16.h>

#include "common.h"

namespace mirec {

constexpr int SM_THREADS = 256;
constexpr int SM_MAX_DRAWS = MIREC_SAMPLE_MAX_DRAWS;
constexpr int64_t SM_MAX_MASKED_ITEMS = MIREC_SAMPLE_MAX_MASKED_ITEMS;   // the filter of a row is a bitmap in LDS
constexpr double SM_MIN_TEMPERATURE = 1e-37;      // below: greedy

struct SampleParams {
    double temperature, top_p, min_p;
    int32_t top_k;
    const float* row_temperature;
    const int32_t* row_top_k;
    const float* row_top_p;
    const float* row_min_p;
};

// Monotone integer image of a score: larger is better, 0 = excluded (filtered, not above its type's lowest finite
// value, or NaN); -0 counts as +0.
__device__ __forceinline__ uint32_t sm_order(float s) {
    s = (s == 0.f) ? 0.f : s;
    const uint32_t b = __float_as_uint(s);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

__device__ __forceinline__ float sm_unorder(uint32_t o) {
    return __uint_as_float((o & 0x80000000u) ? (o & 0x7fffffffu) : ~o);
}

template <int DT>
struct ScoreType;
template <>
struct ScoreType<MIREC_F32> {
    typedef float raw;
    static constexpr float lowest = -FLT_MAX;
    __device__ static __forceinline__ float widen(raw v) { return v; }
};
template <>
struct ScoreType<MIREC_F16> {
    typedef _Float16 raw;
    static constexpr float lowest = -65504.f;
    __device__ static __forceinline__ float widen(raw v) { return (float)v; }
};
template <>
struct ScoreType<MIREC_BF16> {
    typedef uint16_t raw;
    static constexpr float lowest = -3.38953139e38f;
    __device__ static __forceinline__ float widen(raw v) { return __uint_as_float((uint32_t)v << 16); }
};

// 2^t for t <= 0 as a fixed-point number with `bits` fraction bits (bits <= 51): t = k + f with |f| <= 1/2, 2^f by its
// power series to the tenth term (the eleventh is below 2.2e-13 of the value), scaled and rounded to an integer by
// adding 2^52.
__device__ __forceinline__ uint64_t sm_weight(double t, int bits) {
    t = fmax(t, -2000.0);   // also what an infinite difference times a zero step gives
    const double k = rint(t);
    const double f = t - k;
    double p = 7.054911620801121e-09;                 // ln2^10 / 10!
    p = __builtin_fma(p, f, 1.0178086009239696e-07);   // ln2^9 / 9!
    p = __builtin_fma(p, f, 1.3215486790144305e-06);
    p = __builtin_fma(p, f, 1.5252733804059838e-05);
    p = __builtin_fma(p, f, 1.5403530393381606e-04);
    p = __builtin_fma(p, f, 1.3333558146428441e-03);
    p = __builtin_fma(p, f, 9.618129107628477e-03);
    p = __builtin_fma(p, f, 5.5504108664821576e-02);
    p = __builtin_fma(p, f, 2.402265069591007e-01);
    p = __builtin_fma(p, f, 6.931471805599453e-01);
    p = __builtin_fma(p, f, 1.0);
    const double v = ldexp(p, (int)k + bits) + 4503599627370496.0;
    return (uint64_t)__double_as_longlong(v) & 0xfffffffffffffull;
}

__device__ __forceinline__ uint64_t sm_shfl_xor(uint64_t v, int m) {
    return ((uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), m, 64) << 32) | (uint32_t)__shfl_xor((int)v, m, 64);
}

__device__ __forceinline__ uint64_t sm_shfl_up(uint64_t v, int d) {
    return ((uint64_t)(uint32_t)__shfl_up((int)(v >> 32), d, 64) << 32) | (uint32_t)__shfl_up((int)v, d, 64);
}

__device__ __forceinline__ uint64_t sm_wave_sum(uint64_t v) {
#pragma unroll
    for (int m = 32; m > 0; m >>= 1) v += sm_shfl_xor(v, m);
    return v;
}

__device__ __forceinline__ uint64_t sm_wave_scan(uint64_t v) {   // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint64_t o = sm_shfl_up(v, d);
        v += lane >= d ? o : 0ull;
    }
    return v;
}

// One workgroup per row; the row is read again for every step (max, one histogram per byte of the key and per cut, the
// kept mass, the draws).
template <int DT>
__global__ __launch_bounds__(SM_THREADS) void sample_rows_kernel(
    const typename ScoreType<DT>::raw* __restrict__ scores, int64_t n, int64_t m, int64_t stride,
    const int32_t* __restrict__ ids, int64_t ids_stride, const int64_t* __restrict__ mask_indptr,
    const int32_t* __restrict__ mask_indices, const float* __restrict__ uniforms, int draws, int replacement,
    SampleParams par, int bits, int32_t* __restrict__ out_ids, float* __restrict__ out_logprob) {
    extern __shared__ uint32_t liked[];   // one bit per item, when there is a filter
    __shared__ uint64_t hist[256];
    __shared__ uint64_t part[SM_THREADS / 64];
    __shared__ uint32_t part32[SM_THREADS / 64];
    __shared__ uint64_t bcast[2];
    __shared__ int64_t drawn[SM_MAX_DRAWS];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;

    for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
        const typename ScoreType<DT>::raw* s = scores + row * stride;
        const int32_t* id = ids ? ids + row * ids_stride : nullptr;
        __syncthreads();
        if (mask_indptr) {
            for (int64_t w = tid; w < (m + 31) / 32; w += SM_THREADS) liked[w] = 0;
            __syncthreads();
            for (int64_t e = mask_indptr[row] + tid; e < mask_indptr[row + 1]; e += SM_THREADS) {
                const int64_t it = mask_indices[e];
                if (it >= 0 && it < m) atomicOr(&liked[it >> 5], 1u << (it & 31));
            }
            __syncthreads();
        }
        auto key_of = [&](int64_t i) -> uint32_t {
            const float v = ScoreType<DT>::widen(s[i]);
            bool ok = v > ScoreType<DT>::lowest;
            if (mask_indptr) ok = ok && !((liked[i >> 5] >> (i & 31)) & 1u);
            if (id) ok = ok && id[i] >= 0;
            return ok ? sm_order(v) : 0u;
        };
        auto block_sum = [&](uint64_t v) -> uint64_t {
            v = sm_wave_sum(v);
            __syncthreads();
            if (lane == 0) part[wave] = v;
            __syncthreads();
            uint64_t t = 0;
            for (int w = 0; w < SM_THREADS / 64; ++w) t += part[w];
            return t;
        };

        // the best score
        uint32_t top = 0;
        for (int64_t i = tid; i < m; i += SM_THREADS) {
            const uint32_t k = key_of(i);
            top = k > top ? k : top;
        }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            const uint32_t o = (uint32_t)__shfl_xor((int)top, d, 64);
            top = o > top ? o : top;
        }
        __syncthreads();
        if (lane == 0) part32[wave] = top;
        __syncthreads();
        for (int w = 0; w < SM_THREADS / 64; ++w) top = part32[w] > top ? part32[w] : top;
        if (top == 0) {
            for (int d = tid; d < draws; d += SM_THREADS) {
                out_ids[row * draws + d] = -1;
                out_logprob[row * draws + d] = -INFINITY;
            }
            continue;
        }

        const double T = par.row_temperature ? (double)par.row_temperature[row] : par.temperature;
        const double top_p = par.row_top_p ? (double)par.row_top_p[row] : par.top_p;
        const double min_p = par.row_min_p ? (double)par.row_min_p[row] : par.min_p;
        int64_t top_k = par.row_top_k ? par.row_top_k[row] : par.top_k;
        const bool greedy = !(T >= SM_MIN_TEMPERATURE);
        if (top_k <= 0 || top_k > m) top_k = m;
        if (greedy) top_k = 1;
        const double step = greedy ? 0.0 : 1.4426950408889634 / T;
        const double best = (double)sm_unorder(top);
        auto exponent = [&](uint32_t k) -> double { return k == top ? 0.0 : ((double)sm_unorder(k) - best) * step; };
        auto weight = [&](uint32_t k) -> uint64_t { return sm_weight(exponent(k), bits); };

        // `cut` is the last key kept, `ties` how many of the items that have it
        uint32_t cut = 1;
        int64_t ties = m;
        if (top_k < m) {
            uint32_t prefix = 0, known = 0;
            uint64_t above = 0;   // items in buckets above the current one
            bool all = false;
            for (int shift = 24; shift >= 0 && !all; shift -= 8) {
                hist[tid] = 0;
                __syncthreads();
                for (int64_t i = tid; i < m; i += SM_THREADS) {
                    const uint32_t k = key_of(i);
                    if (k && (k & known) == prefix) atomicAdd((unsigned long long*)&hist[(k >> shift) & 255], 1ull);
                }
                __syncthreads();
                if (tid == 0) {
                    uint64_t a = above;
                    int b = 255;
                    while (b >= 0 && a + hist[b] < (uint64_t)top_k) a += hist[b--];
                    bcast[0] = a;
                    bcast[1] = (uint64_t)(int64_t)b;
                }
                __syncthreads();
                const int b = (int)(int64_t)bcast[1];
                above = bcast[0];
                all = b < 0;   // fewer than top_k items in the row
                if (!all) {
                    prefix |= (uint32_t)b << shift;
                    known |= 255u << shift;
                }
                __syncthreads();
            }
            if (!all) {
                cut = prefix;
                ties = top_k - (int64_t)above;
            }
        }
        if (top_p < 1.0) {
            // the mass of what top_k left
            uint64_t v = 0;
            for (int64_t i = tid; i < m; i += SM_THREADS) {
                const uint32_t k = key_of(i);
                if (k > cut) v += weight(k);
            }
            const uint64_t total = block_sum(v) + (cut > 1 ? (uint64_t)ties * weight(cut) : 0ull);
            const double bound = top_p * (double)total;
            uint32_t prefix = 0, known = 0;
            uint64_t above = 0;
            bool all = false;
            for (int shift = 24; shift >= 0 && !all; shift -= 8) {
                hist[tid] = 0;
                __syncthreads();
                for (int64_t i = tid; i < m; i += SM_THREADS) {
                    const uint32_t k = key_of(i);
                    if (k > cut && (k & known) == prefix)
                        atomicAdd((unsigned long long*)&hist[(k >> shift) & 255], (unsigned long long)weight(k));
                }
                __syncthreads();
                if (tid == 0) {
                    uint64_t* hc = hist;
                    if (cut > 1 && (cut & known) == prefix) hc[(cut >> shift) & 255] += (uint64_t)ties * weight(cut);
                    // the last bucket with mass that starts before the bound
                    uint64_t a = above;
                    int b = 255, last = -1;
                    uint64_t at = above;
                    for (; b >= 0; --b) {
                        if (hc[b] == 0) continue;
                        if (last >= 0 && !((double)a < bound)) break;
                        last = b;
                        at = a;
                        a += hc[b];
                    }
                    bcast[0] = at;
                    bcast[1] = (uint64_t)(int64_t)last;
                }
                __syncthreads();
                const int b = (int)(int64_t)bcast[1];
                above = bcast[0];
                all = b < 0;
                if (!all) {
                    prefix |= (uint32_t)b << shift;
                    known |= 255u << shift;
                }
                __syncthreads();
            }
            if (!all) {
                // of the items with this key the first r with above + (r - 1) w < bound
                const double w = (double)weight(prefix);
                double r = ceil((bound - (double)above) / w);
                r = r < 1.0 ? 1.0 : r;
                int64_t have = prefix == cut ? ties : m;
                ties = r < (double)have ? (int64_t)r : have;
                cut = prefix;
            }
        }
        const double floor_w = min_p > 0.0 ? fmin(min_p, 1.0) * (double)(1ull << bits) : 0.0;

        // kept weights in index order; `drawn_count` positions have been taken out
        int drawn_count = 0;
        auto kept = [&](int64_t i, int64_t& seen) -> uint64_t {   // called by the whole workgroup, i ascending over it
            const uint32_t k = i < m ? key_of(i) : 0u;
            const bool tie = k == cut && k != 0;
            const uint64_t votes = __ballot(tie);
            __syncthreads();
            if (lane == 0) part32[wave] = (uint32_t)__popcll(votes);
            __syncthreads();
            int64_t before = seen + __popcll(votes & ((1ull << lane) - 1));
            for (int w = 0; w < SM_THREADS / 64; ++w) {
                before += w < wave ? part32[w] : 0;
                seen += part32[w];
            }
            uint64_t wgt = 0;
            if (k > cut || (tie && before < ties)) {
                wgt = weight(k);
                if ((double)wgt < floor_w) wgt = 0;
            }
            for (int j = 0; j < drawn_count; ++j) wgt = drawn[j] == i ? 0ull : wgt;
            return wgt;
        };
        uint64_t total = 0;
        for (int d = 0; d < draws; ++d) {
            if (d == 0 || !replacement) {
                uint64_t v = 0;
                int64_t seen = 0;
                for (int64_t i0 = 0; i0 < m; i0 += SM_THREADS) v += kept(i0 + tid, seen);
                total = block_sum(v);
            }
            int32_t got = -1;
            if (total > 0) {
                const float u = uniforms[row * draws + d];
                const double uc = u > 0.f ? fmin((double)u, 1.0 - 0x1p-53) : 0.0;
                const uint64_t t = __umul64hi(total, (uint64_t)(uc * 0x1p53) << 11);
                uint64_t run = 0;
                int64_t seen = 0;
                if (tid == 0) bcast[0] = ~0ull;
                for (int64_t i0 = 0; i0 < m && run <= t; i0 += SM_THREADS) {
                    const int64_t i = i0 + tid;
                    const uint64_t w = kept(i, seen);
                    const uint64_t inc = sm_wave_scan(w);
                    __syncthreads();
                    if (lane == 63) part[wave] = inc;
                    __syncthreads();
                    uint64_t base = run;
                    for (int v = 0; v < SM_THREADS / 64; ++v) {
                        base += v < wave ? part[v] : 0ull;
                        run += part[v];
                    }
                    if (w && base + inc > t && base + inc - w <= t) bcast[0] = (uint64_t)i;
                    __syncthreads();
                }
                __syncthreads();
                const int64_t i = (int64_t)bcast[0];
                got = 0;
                if (tid == 0) {
                    out_ids[row * draws + d] = id ? id[i] : (int32_t)i;
                    out_logprob[row * draws + d] =
                        (float)(exponent(key_of(i)) * 0.69314718055994531 - log(ldexp((double)total, -bits)));
                    drawn[drawn_count] = i;
                }
                if (!replacement) ++drawn_count;
                __syncthreads();
            }
            if (got < 0 && tid == 0) {
                out_ids[row * draws + d] = -1;
                out_logprob[row * draws + d] = -INFINITY;
            }
        }
    }
}

// Fraction bits of a weight: the sum of m of them stays below 2^62.
static int sample_bits(int64_t m) {
    int b = 0;
    while (((int64_t)1 << b) < m) ++b;
    return 62 - b < 51 ? 62 - b : 51;
}

}  // namespace mirec

extern "C" size_t mirec_sample_workspace_bytes(int64_t n, int64_t m, int dtype, int draws) {
    (void)n, (void)m, (void)dtype, (void)draws;
    return 0;
}

extern "C" int mirec_sample(const void* scores, int dtype, int64_t n, int64_t m, int64_t row_stride, const int32_t* ids,
                            int64_t ids_stride, const int64_t* mask_indptr, const int32_t* mask_indices,
                            const float* uniforms, int draws, int replacement, double temperature,
                            const float* row_temperature, int32_t top_k, const int32_t* row_top_k, double top_p,
                            const float* row_top_p, double min_p, const float* row_min_p, int32_t* out_ids,
                            float* out_logprob, void* ws, size_t ws_bytes, mirec_stream_t stream_) {
    using namespace mirec;
    hipStream_t stream = (hipStream_t)stream_;
    (void)ws, (void)ws_bytes;
    MIREC_REQUIRE(n >= 0 && m >= 0 && draws >= 0, MIREC_E_INVALID, "mirec_sample: negative size");
    MIREC_REQUIRE(dtype == MIREC_F32 || dtype == MIREC_F16 || dtype == MIREC_BF16, MIREC_E_INVALID,
                  "mirec_sample: unknown score type %d", dtype);
    MIREC_REQUIRE(draws <= SM_MAX_DRAWS, MIREC_E_UNSUPPORTED, "mirec_sample: %d draws a row; at most %d are supported",
                  draws, SM_MAX_DRAWS);
    MIREC_REQUIRE(m < ((int64_t)1 << 31), MIREC_E_UNSUPPORTED, "mirec_sample: more than 2^31 items");
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
    const SampleParams par = {temperature, top_p, min_p, top_k, row_temperature, row_top_k, row_top_p, row_min_p};
    const int bits = sample_bits(m);
    const unsigned blocks = (unsigned)(n < 262144 ? n : 262144);
    const size_t lds = mask_indptr ? (size_t)((m + 31) / 32) * 4 : 0;
    // the filter's bitmap of a long row (up to 64 KiB) takes more dynamic LDS than a kernel gets unasked
#define MIREC_SAMPLE(DT)                                                                                             \
    do {                                                                                                             \
        static OncePerDevice once;                                                                                   \
        bool* done = once.slot();                                                                                    \
        MIREC_REQUIRE(done, MIREC_E_HIP, "mirec_sample: cannot read the current device");                            \
        if (!*done) {                                                                                                \
            MIREC_HIP(hipFuncSetAttribute((const void*)sample_rows_kernel<DT>,                                       \
                                          hipFuncAttributeMaxDynamicSharedMemorySize,                                \
                                          (int)(SM_MAX_MASKED_ITEMS / 8)));                                          \
            *done = true;                                                                                            \
        }                                                                                                            \
        hipLaunchKernelGGL((sample_rows_kernel<DT>), dim3(blocks), dim3(SM_THREADS), lds, stream,                    \
                           (const ScoreType<DT>::raw*)scores, n, m, row_stride, ids, ids_stride, mask_indptr,        \
                           mask_indices, uniforms, draws, replacement, par, bits, out_ids, out_logprob);             \
    } while (0)
    if (dtype == MIREC_F32) MIREC_SAMPLE(MIREC_F32);
    else if (dtype == MIREC_F16) MIREC_SAMPLE(MIREC_F16);
    else MIREC_SAMPLE(MIREC_BF16);
#undef MIREC_SAMPLE
    MIREC_LAUNCH_CHECK();
    return MIREC_OK;
}
