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
//
// Draws without replacement take weights out of that sum.  Once it is so low that the roundings of its terms count (or
// nothing but them is left), the weights of the items that were kept and are still there are formed anew, relative to the
// best of these (`renew_below`).
#pragma once

#include <float.h>

#include <type_traits>

#include "common.h"

namespace mirec {

constexpr int SM_MAX_DRAWS = MIREC_SAMPLE_MAX_DRAWS;
constexpr int64_t SM_MAX_MASKED_ITEMS = MIREC_SAMPLE_MAX_MASKED_ITEMS;   // the filter of a row is a bitmap in LDS
constexpr double SM_MIN_TEMPERATURE = 1e-37;      // below: greedy
constexpr int SM_SHORT = 256;                     // rows up to this length: in the registers of a wavefront
constexpr int64_t SM_FEW_ROWS = 256;              // no more rows than compute units: larger workgroups
constexpr int64_t SM_SOME_ROWS = 768;             // no more rows than three workgroups to a compute unit
constexpr int SM_AHEAD = 2;                       // loads in flight ahead of the work
constexpr int SM_BINS = 1024;                     // of a histogram over a row
constexpr int SM_FEW = 256;                        // entries that are compared with each other for every sum
constexpr int SM_LIST = 512;                     // entries that are ranked against each other in LDS

struct SampleParams {
    double step, top_p;   // step: log2 e / temperature
    uint64_t floor_w;     // least weight that min_p keeps
    uint64_t renew_below; // without replacement: the least sum of weights that is drawn from
    int32_t top_k;
    bool greedy;
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

// a b + c with c in scalar registers.  (Left alone, the compiler copies each constant into the accumulator of a
// two-address multiply-add first: nine copies for nine steps below.)
__device__ __forceinline__ double sm_fma(double a, double b, double c) {
    double r;
    asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
    return r;
}

// 2^f for |f| <= 1/2 to 1.6e-14 of it: 1 + f q(f), q of degree 8 fitted to the least largest relative error (a Lawson
// iteration on (2^f - 1) / f); exact at f = 0.
__device__ __forceinline__ double sm_exp2_fraction(double f) {
    double p = 1.0148328577088516e-07;
    p = sm_fma(p, f, 1.3258336037497191e-06);
    p = sm_fma(p, f, 1.5252989797007882e-05);
    p = sm_fma(p, f, 1.5403440872165233e-04);
    p = sm_fma(p, f, 1.3333557626651542e-03);
    p = sm_fma(p, f, 9.618129181194148e-03);
    p = sm_fma(p, f, 5.550410866839772e-02);
    p = sm_fma(p, f, 2.4022650695722697e-01);
    p = sm_fma(p, f, 6.931471805598861e-01);
    return __builtin_fma(p, f, 1.0);
}

constexpr double SM_ROUND = 6755399441055744.0;   // 1.5 2^52: the sum's low bits are the nearest integer

// The weight of a score: 2^((s - best) step) with `bits` (at most 51) fraction bits, the nearest such number; 0 for minus
// infinity.  Vector float64 instructions run at the rate of float32 ones here, and about twenty of them are all there is:
// adding 2^(52 - bits) rounds and leaves the integer in the mantissa.
__device__ __forceinline__ uint64_t sm_weight(float score, double best, double step, double rounder) {
    const double t = fmax(((double)score - best) * step, -80.0);   // (a NaN, infinity times zero, becomes -80 too)
    const double k = t + SM_ROUND;
    const double p = sm_exp2_fraction(t - (k - SM_ROUND));
    const double v = __hiloint2double(__double2hiint(p) + (__double2loint(k) << 20), __double2loint(p)) + rounder;   // p 2^k
    return (uint64_t)__double_as_longlong(v) & 0xfffffffffffffull;
}

__device__ __forceinline__ double sm_rounder(int bits) { return __hiloint2double((1023 + 52 - bits) << 20, 0); }   // 2^(52 - bits)

// log2 x of a positive normal number to 1e-13 or so: the fp32 logarithm, then one Newton step with the power above.
__device__ __forceinline__ double sm_log2(double x) {
    const double l = (double)__builtin_amdgcn_logf((float)x);
    const double k = l + SM_ROUND;
    const double back = sm_exp2_fraction((k - SM_ROUND) - l);   // 2^(k - l)
    const double r = ldexp(x, -(int)(uint32_t)__double_as_longlong(k)) * back - 1.0;   // x / 2^l - 1
    return __builtin_fma(r * (1.0 - 0.5 * r), 1.4426950408889634, l);
}

// ---- sums and maxima over a wavefront, by data-parallel moves between lanes (no LDS)

// One step: v of another lane is added where the move reaches from a lane that is there (elsewhere the instruction does
// nothing).  Written out because the compiler moves and adds separately: seven instructions a step instead of two, a third
// of what a piece of a long row costs.  A data-parallel read of a register needs two wait states behind its write, and so
// does reading vcc as a carry behind the vector instruction that wrote it (the compiler puts an s_nop 1 there, too): the
// wait between the two instructions of a step is enough for both.
#define SM_ADD_STEP(MOVE)                                       \
    "v_add_co_u32_dpp %0, vcc, %0, %0 " MOVE " bank_mask:0xf\n"  \
    "s_nop 1\n"                                                 \
    "v_addc_co_u32_dpp %1, vcc, %1, %1, vcc " MOVE " bank_mask:0xf\n"

__device__ __forceinline__ uint64_t sm_half_scan(uint64_t v) {   // inclusive, over lanes 0 .. 31 and 32 .. 63
    uint32_t lo = (uint32_t)v, hi = (uint32_t)(v >> 32);
    asm("s_nop 1\n"                                              // shifted by 1, 2, 4, 8 within rows of 16 lanes,
        SM_ADD_STEP("row_shr:1 row_mask:0xf") SM_ADD_STEP("row_shr:2 row_mask:0xf") SM_ADD_STEP("row_shr:4 row_mask:0xf")
        SM_ADD_STEP("row_shr:8 row_mask:0xf") SM_ADD_STEP("row_bcast:15 row_mask:0xa")   // lane 15 of a row to rows 1 and 3
        "s_nop 1" : "+v"(lo), "+v"(hi) : : "vcc");
    return ((uint64_t)hi << 32) | lo;
}

__device__ __forceinline__ uint64_t sm_wave_scan(uint64_t v) {
    v = sm_half_scan(v);
    uint32_t lo = (uint32_t)v, hi = (uint32_t)(v >> 32);
    asm("s_nop 1\n" SM_ADD_STEP("row_bcast:31 row_mask:0xc") "s_nop 1" : "+v"(lo), "+v"(hi) : : "vcc");   // lane 31 to rows 2 and 3
    return ((uint64_t)hi << 32) | lo;
}

__device__ __forceinline__ uint64_t sm_lane(uint64_t v, int lane) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32) |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}

__device__ __forceinline__ uint64_t sm_wave_sum(uint64_t v) { return sm_lane(sm_wave_scan(v), 63); }

#define SM_MAX_STEP(MOVE) "s_nop 1\nv_max_f32_dpp %0, %0, %0 " MOVE " bank_mask:0xf\n"

__device__ __forceinline__ float sm_half_max(float v) {   // in lanes 31 and 63
    asm(SM_MAX_STEP("row_shr:1 row_mask:0xf") SM_MAX_STEP("row_shr:2 row_mask:0xf") SM_MAX_STEP("row_shr:4 row_mask:0xf")
        SM_MAX_STEP("row_shr:8 row_mask:0xf") SM_MAX_STEP("row_bcast:15 row_mask:0xa") "s_nop 1" : "+v"(v));
    return v;
}

__device__ __forceinline__ float sm_wave_max(float v) {
    v = sm_half_max(v);
    asm(SM_MAX_STEP("row_bcast:31 row_mask:0xc") "s_nop 1" : "+v"(v));
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

// Where a number of [0, 1) falls in a total: floor(u * total), exactly (u is a 24-bit integer over a power of two); 0 for
// NaN and below the range, total - 1 above it.
__device__ __forceinline__ uint64_t sm_target(float u, uint64_t total) {
    const uint32_t b = __float_as_uint(fmaxf(u, 0.f)) & 0x7fffffffu, e = b >> 23;
    const uint32_t M = (b & 0x7fffffu) | (e > 0 ? 0x800000u : 0u), q = 150 - (e > 0 ? e : 1);   // u = M 2^-q
    const uint64_t lo = (uint64_t)M * (uint32_t)total, hi = (uint64_t)M * (uint32_t)(total >> 32) + (lo >> 32);
    const uint64_t near = (hi << ((32 - q) & 63)) | ((uint32_t)lo >> (q & 31));   // 24 <= q < 32
    const uint64_t far = hi >> (q - 32 < 63 ? q - 32 : 63);
    return u >= 1.f ? total - 1 : q < 32 ? near : far;
}

// The least integer mass that is not below a share of a total.
__device__ __forceinline__ uint64_t sm_bound(double share, uint64_t total) { return (uint64_t)ceil(fmax(share, 0.0) * (double)total); }

// What the cuts and the temperature of one row come to.
struct RowCuts {
    int64_t top_k;
    double top_p, step;   // step: log2 e / temperature
    uint64_t floor_w;     // least weight that min_p keeps
};

__device__ __forceinline__ RowCuts sm_cuts(const SampleParams& par, int64_t row, int64_t m, int bits) {
    RowCuts c;
    c.step = par.step;
    bool greedy = par.greedy;
    if (par.row_temperature) {
        const double T = (double)par.row_temperature[row];
        greedy = !(T >= SM_MIN_TEMPERATURE);
        c.step = greedy ? 0.0 : 1.4426950408889634 / T;
    }
    c.top_p = par.row_top_p ? (double)par.row_top_p[row] : par.top_p;
    c.floor_w = par.floor_w;
    if (par.row_min_p) {
        const double min_p = (double)par.row_min_p[row];
        c.floor_w = min_p > 0.0 ? sm_bound(fmin(min_p, 1.0), 1ull << bits) : 0ull;
    }
    c.top_k = par.row_top_k ? par.row_top_k[row] : par.top_k;
    if (c.top_k <= 0 || c.top_k > m) c.top_k = m;
    if (greedy) c.top_k = 1;
    return c;
}

__device__ __forceinline__ float sm_logprob(float score, double best, double step, uint64_t total, int bits) {
    const double t = fmax(((double)score - best) * step, -80.0);
    // (not above zero: the sum's terms are rounded)
    return fminf((float)((t - sm_log2(ldexp((double)total, -bits))) * 0.69314718055994531), 0.f);
}

// ------------------------------------------------------------------------------------------------------ short rows

// One wavefront per R rows of at most 64 E / R items, all of it in registers: items E l .. E l + E - 1 in lane l of the row's
// lanes, so that one scan over the lanes gives every running sum.  A ranked list is in order already (one comparison of
// neighbours says so), and then the running sum in index order is the running sum in rank order too: the scan serves the
// cuts and the draws.  Otherwise every item is compared with every other.  The lanes of a row take `rows_each` rows, one after
// the other, and keep their draws, one each, until all lanes have one: logarithms and stores are then one for all.
// AGAIN: drawn items come back.
// What bounds it is the number of vector instructions per row; most of them are for the row, not for its items, so that two
// rows of up to 128 items share them.  Measured: 262144 lists of 100 under top_p and min_p 104 us (2 TB/s of scores and ids;
// the bytes alone 53 us), of 50 76 us, one list 3.4 us; ten draws without replacement under top_p 412 us.
template <int DT, int E, int R, bool AGAIN>
__global__ __launch_bounds__(256) void sample_short_kernel(
    const typename ScoreType<DT>::raw* __restrict__ scores, int64_t n, int m, int64_t stride, const int32_t* __restrict__ ids,
    int64_t ids_stride, const int64_t* __restrict__ mask_indptr, const int32_t* __restrict__ mask_indices,
    const float* __restrict__ uniforms, int draws, int rows_each, SampleParams par, int bits,
    int32_t* __restrict__ out_ids, float* __restrict__ out_logprob) {
    constexpr int LANES = 64 / R;
    const int lane = threadIdx.x & 63, half = R == 1 ? 0 : lane / LANES, sub = lane % LANES, first = E * sub;
    const double rounder = sm_rounder(bits);
    // Within a row's lanes: the value of a lane that is the same for both rows (`at`), or not (`pick`); of the last lane.
    auto at32 = [&](uint32_t v, int l) -> uint32_t {
        const uint32_t x = (uint32_t)__builtin_amdgcn_readlane((int)v, l);
        if (R == 1) return x;
        const uint32_t y = (uint32_t)__builtin_amdgcn_readlane((int)v, LANES + l);
        return half ? y : x;
    };
    auto at64 = [&](uint64_t v, int l) -> uint64_t { return ((uint64_t)at32((uint32_t)(v >> 32), l) << 32) | at32((uint32_t)v, l); };
    auto pick32 = [&](uint32_t v, int l) -> uint32_t {
        if (R == 1) return (uint32_t)__builtin_amdgcn_readlane((int)v, l);
        return (uint32_t)__builtin_amdgcn_ds_bpermute(4 * (half * LANES + l), (int)v);
    };
    auto pick64 = [&](uint64_t v, int l) -> uint64_t { return ((uint64_t)pick32((uint32_t)(v >> 32), l) << 32) | pick32((uint32_t)v, l); };
    auto votes_of = [&](bool yes) -> uint64_t {
        const uint64_t votes = __ballot(yes);
        return R == 1 ? votes : half ? votes >> 32 : votes & 0xffffffffull;
    };
    auto first_vote = [&](uint64_t votes) -> int { return R == 1 ? __builtin_ctzll(votes) : __builtin_ctz((uint32_t)votes | 0x80000000u); };
    auto scan64 = [&](uint64_t v) -> uint64_t { return R == 1 ? sm_wave_scan(v) : sm_half_scan(v); };

    // the rows of these lanes, and one that is there for lanes without
    const int64_t row0 = (((int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * R + half) * rows_each;
    const int64_t row1 = row0 + rows_each < n ? row0 + rows_each : n;
    int64_t row = row0 < n ? row0 : n - 1;
    const typename ScoreType<DT>::raw* s = scores + row * stride;
    const int32_t* list = ids ? ids + row * ids_stride : nullptr;
    const float* uniform = uniforms + row * draws;
    // draws that are not written yet, in lanes 0 .. waiting - 1: number out0 + lane
    int waiting = 0;
    int64_t out0 = row0 * draws;
    const int64_t out1 = row1 * draws;
    int32_t got = -1;
    float got_f = 0.f, got_best = 0.f;
    double got_step = 0.0;
    uint64_t got_total = 1;
    auto flush = [&]() {
        if (sub < waiting && out0 + sub < out1) {
            out_ids[out0 + sub] = got;
            out_logprob[out0 + sub] = got >= 0 ? sm_logprob(got_f, (double)got_best, got_step, got_total, bits) : -INFINITY;
        }
        out0 += waiting;
        waiting = 0;
    };

    // A row is read while the one before it is worked on.
    typename ScoreType<DT>::raw next_s[E] = {};
    int32_t next_id[E] = {};
    float next_u = 0.f;
    auto fetch = [&]() {
#pragma unroll
        for (int j = 0; j < E; ++j)
            if (first + j < m) {
                next_s[j] = s[first + j];
                if (ids) next_id[j] = list[first + j];
            }
        if (sub < draws) next_u = uniform[sub];
    };
    fetch();
    for (int i = 0; i < rows_each && __any(row0 + i < row1); ++i) {
        float f[E];   // minus infinity where excluded; infinity counts as the largest finite score
        int32_t id[E];
#pragma unroll
        for (int j = 0; j < E; ++j) {
            const float v = ScoreType<DT>::widen(next_s[j]);
            id[j] = ids ? next_id[j] : first + j;
            f[j] = first + j < m && v > ScoreType<DT>::lowest && id[j] >= 0 ? fminf(v, FLT_MAX) : -INFINITY;
        }
        const float u0 = next_u;
        const float* row_u = uniform;
        const int64_t this_row = row;
        if (row + 1 < row1) {   // (lanes without a further row stay where they are; what they draw is not written)
            ++row;
            s += stride;
            if (ids) list += ids_stride;
            uniform += draws;
        }
        if (i + 1 < rows_each) fetch();
        if (mask_indptr) {   // each lane looks for its items in the row's filter
            for (int64_t e = mask_indptr[this_row]; e < mask_indptr[this_row + 1]; ++e) {
                const int32_t it = mask_indices[e];
#pragma unroll
                for (int j = 0; j < E; ++j) f[j] = it == first + j ? -INFINITY : f[j];
            }
        }
        float top = f[0];
#pragma unroll
        for (int j = 1; j < E; ++j) top = fmaxf(top, f[j]);
        top = R == 1 ? sm_wave_max(top) : __uint_as_float(at32(__float_as_uint(sm_half_max(top)), LANES - 1));
        const RowCuts cut = sm_cuts(par, this_row, m, bits);
        const int k = (int)cut.top_k;   // (at most m)
        float best32 = top > -INFINITY ? top : 0.f;
        const double best = (double)best32;
        uint32_t left = 0;   // without replacement: this lane's items that are kept and not drawn yet
        uint64_t w[E];
#pragma unroll
        for (int j = 0; j < E; ++j) w[j] = sm_weight(f[j], best, cut.step, rounder);

        // in order if no item is better than the one before it (the next lane's first: minus infinity after the last lane)
        float before_f = __int_as_float(__builtin_amdgcn_update_dpp((int)0xff800000, __float_as_int(f[0]), 0x130, 0xf, 0xf, false));
        if (R > 1) before_f = sub == LANES - 1 ? -INFINITY : before_f;
        bool ordered = true;
#pragma unroll
        for (int j = E - 1; j >= 0; --j) {
            ordered = ordered && f[j] >= before_f;
            before_f = f[j];
        }
        uint64_t run[E];   // sum of the kept weights up to and with the item
        auto scan = [&]() -> uint64_t {
            uint64_t sum = w[0];
#pragma unroll
            for (int j = 1; j < E; ++j) sum += w[j];
            const uint64_t inc = scan64(sum);
            run[E - 1] = inc;
#pragma unroll
            for (int j = E - 1; j > 0; --j) run[j - 1] = run[j] - w[j];
            return at64(inc, LANES - 1);
        };
        uint64_t total;
        if (__all(ordered)) {
            if (__any(k < m)) {
#pragma unroll
                for (int j = 0; j < E; ++j) w[j] = first + j < k ? w[j] : 0ull;
            }
            total = scan();
            const uint64_t bound = cut.top_p < 1.0 ? sm_bound(cut.top_p, total) : ~0ull;
            if (!AGAIN) {
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    const uint64_t before = j > 0 ? run[j - 1] : run[0] - w[0];
                    const bool stays = first + j < k && f[j] > -INFINITY && (first + j == 0 || before < bound) && w[j] >= cut.floor_w;
                    left |= stays ? 1u << j : 0u;
                }
            }
            if (__any(cut.top_p < 1.0 || cut.floor_w > 0)) {
                // A prefix stays: the running sum at its end.  (What a draw looks for is the first running sum above a number
                // below that: the items behind it may keep their weights.)
                uint64_t last = 0;
                const uint64_t least = cut.floor_w > 1 ? cut.floor_w : 1;
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    const uint64_t before = j > 0 ? run[j - 1] : run[0] - w[0];
                    const bool stays = (first + j == 0 || before < bound) && w[j] >= least;
                    last = stays ? run[j] : last;
                }
                const uint64_t votes = votes_of(last != 0);
                const int l = R == 1 ? 63 - __builtin_clzll(votes | 1) : 31 - __builtin_clz((uint32_t)votes | 1);
                const uint64_t mass = pick64(last, l);
                total = votes ? mass : 0ull;
            }
        } else {
            uint32_t rank[E];
            uint64_t before[E];
#pragma unroll
            for (int j = 0; j < E; ++j) {
                rank[j] = 0;
                before[j] = 0;
            }
            if (__any(k < m || cut.top_p < 1.0)) {
                for (int l = 0; E * l < m; ++l)
#pragma unroll
                    for (int q = 0; q < E; ++q) {
                        const float g = __uint_as_float(at32(__float_as_uint(f[q]), l));
                        const uint64_t gw = at64(w[q], l);
#pragma unroll
                        for (int j = 0; j < E; ++j) {
                            const bool ahead = (g > f[j]) | ((g == f[j]) & (E * l + q < first + j));
                            rank[j] += ahead ? 1u : 0u;
                            before[j] += ahead ? gw : 0ull;
                        }
                    }
            }
            uint64_t mass = 0;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                if (rank[j] >= (uint32_t)k) w[j] = 0;
                mass += w[j];
            }
            mass = at64(scan64(mass), LANES - 1);
            const uint64_t bound = cut.top_p < 1.0 ? sm_bound(cut.top_p, mass) : ~0ull;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                const bool stays = rank[j] < (uint32_t)k && (rank[j] == 0 || before[j] < bound) && w[j] >= cut.floor_w;
                left |= stays && f[j] > -INFINITY ? 1u << j : 0u;
                if (!stays) w[j] = 0;
            }
            total = scan();
        }

        for (int d0 = 0; d0 < draws; d0 += LANES) {
            const int cnt = draws - d0 < LANES ? draws - d0 : LANES;
            const float u = d0 == 0 ? u0 : sub < cnt ? row_u[d0 + sub] : 0.f;
            if (waiting + cnt > LANES) flush();
            const uint64_t targets = sm_target(u, total);
            for (int d = 0; d < cnt; ++d, ++waiting) {
                if (!__any(total != 0)) {
                    if (sub == waiting) got = -1;
                    continue;
                }
                const uint64_t t = AGAIN ? at64(targets, d) : sm_target(__uint_as_float(at32(__float_as_uint(u), d)), total);
                // the first lane whose last running sum is above the number, and its first item for which that holds
                const int l = first_vote(votes_of(run[E - 1] > t));
                int j_of = E - 1;
                int32_t my_id = id[E - 1];
                float my_f = f[E - 1];
#pragma unroll
                for (int j = E - 2; j >= 0; --j) {
                    const bool above = run[j] > t;
                    j_of = above ? j : j_of;
                    my_id = above ? id[j] : my_id;
                    my_f = above ? f[j] : my_f;
                }
                const int32_t item = (int32_t)pick32((uint32_t)my_id, l);
                const float score = __uint_as_float(pick32(__float_as_uint(my_f), l));
                if (sub == waiting) {
                    got = total != 0 ? item : -1;
                    got_f = score;
                    got_best = best32;
                    got_step = cut.step;
                    got_total = total;
                }
                if (!AGAIN) {   // the item leaves: every running sum from it on is lower by its weight
                    const int at = E * l + (int)pick32((uint32_t)j_of, l);
                    uint64_t mine = 0;
#pragma unroll
                    for (int j = 0; j < E; ++j) mine = first + j == at ? w[j] : mine;
                    const bool drawn = total != 0;
                    const uint64_t leaves = pick64(mine, l), gone = drawn ? leaves : 0ull;
                    total -= gone;
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        w[j] = first + j == at ? 0ull : w[j];
                        run[j] -= first + j >= at ? gone : 0ull;
                        left &= first + j == at && drawn ? ~(1u << j) : ~0u;
                    }
                    const bool low = total < par.renew_below;
                    if (__any(low && left != 0)) {
                        float most = -INFINITY;
#pragma unroll
                        for (int j = 0; j < E; ++j) most = fmaxf(most, (left >> j) & 1u ? f[j] : -INFINITY);
                        most = R == 1 ? sm_wave_max(most) : __uint_as_float(at32(__float_as_uint(sm_half_max(most)), LANES - 1));
                        const bool renew = low && most > -INFINITY;   // (the other row of the wavefront may have no need)
                        best32 = renew ? most : best32;
#pragma unroll
                        for (int j = 0; j < E; ++j) {
                            const uint64_t anew = (left >> j) & 1u ? sm_weight(f[j], (double)best32, cut.step, rounder) : 0ull;
                            w[j] = renew ? anew : w[j];
                        }
                        const uint64_t sum = scan();
                        total = renew ? sum : total;
                    }
                }
            }
        }
    }
    flush();
}

// ------------------------------------------------------------------------------------------------------- long rows

// Scores of 16 bytes, from any address that is aligned to their type.
typedef uint32_t sm_words __attribute__((ext_vector_type(4), aligned(2)));

typedef uint16_t sm_u16x2 __attribute__((ext_vector_type(2)));
template <int DT>
struct Chunk {
    static constexpr int V = DT == MIREC_F32 ? 4 : 8;   // scores of a thread's 16 bytes
    uint32_t word[4];
    __device__ __forceinline__ float raw(int v) const {
        if constexpr (DT == MIREC_F32)
            return __uint_as_float(word[v]);
        else if constexpr (DT == MIREC_BF16)
            return __uint_as_float(v & 1 ? word[v >> 1] & 0xffff0000u : word[v >> 1] << 16);
        else
            return (float)__builtin_bit_cast(_Float16, (uint16_t)(word[v >> 1] >> (16 * (v & 1))));
    }
    // minus infinity where excluded (once settle() has run); infinity counts as the largest finite score
    __device__ __forceinline__ float score(int v) const { return DT == MIREC_F32 ? raw(v) : fminf(raw(v), FLT_MAX); }
    __device__ __forceinline__ void exclude(int v) {
        if constexpr (DT == MIREC_F32) word[v] = 0xff800000u;
        else {
            const uint32_t inf = DT == MIREC_BF16 ? 0xff80u : 0xfc00u;
            word[v >> 1] = v & 1 ? (word[v >> 1] & 0xffffu) | (inf << 16) : (word[v >> 1] & 0xffff0000u) | inf;
        }
    }
    // Whether a score is not below the largest finite magnitude: it may be one that is excluded, or infinite.
    __device__ __forceinline__ bool unsettled() const {
        if constexpr (DT == MIREC_F32) {
            // (a sum of magnitudes is not below any of them, and a NaN where one is; that it can be too large costs time only)
            return !((fabsf(raw(0)) + fabsf(raw(1))) + (fabsf(raw(2)) + fabsf(raw(3))) < FLT_MAX);
        } else {
            sm_u16x2 most = __builtin_bit_cast(sm_u16x2, word[0] & 0x7fff7fffu);
#pragma unroll
            for (int i = 1; i < 4; ++i) most = __builtin_elementwise_max(most, __builtin_bit_cast(sm_u16x2, word[i] & 0x7fff7fffu));
            const uint16_t limit = DT == MIREC_BF16 ? 0x7f7f : 0x7bff;
            return most[0] >= limit || most[1] >= limit;
        }
    }
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float f = raw(v);
            if constexpr (DT == MIREC_F32)
                word[v] = __float_as_uint(f > ScoreType<DT>::lowest ? fminf(f, FLT_MAX) : -INFINITY);
            else if (!(f > ScoreType<DT>::lowest))
                exclude(v);
        }
    }
};

// One workgroup of NT threads per row.  The row is cut into pieces of S chunks, a chunk is 16 bytes per lane; piece g NW + w
// belongs to wavefront w, so pieces, chunks and lanes are in index order; S makes at most SM_BINS pieces of a row.  Each
// pass reads the row again (from L2, mostly): rows held in registers spilled.
//
// A cut is the last item that stays (score and index).  It is found by a histogram whose bins are ordered like the items
// -- first by the score's distance from the best, in 1/32 octaves of the weight, then, should a bin hold more than
// SM_LIST items, by equal ranges of K = (monotone image of the score, complemented index), which is larger for a better
// item -- and by ranking the items of the bin that the border falls into against each other.
//
// What bounds it: where the rows in flight exceed L2 each pass reads them at the rate of memory (two passes over 4096 x 27000
// in 186 us, 4.75 TB/s), and a weight is 21 instructions (nine of them its polynomial); under top_p both take about 280 of
// the 340 us of those rows.  Hence as few passes as possible, and four rows of 256 threads side by side on a compute unit, or
// fewer of more threads where there are fewer rows.  Measured: 1024 x 27000 under top_p 105 us, 512 x 200000 bf16 uncut,
// 8 draws, 144 us, one row of 27000 under top_k 17 us.
// Registers: few rows, of 1024 threads, run one or two workgroups to a compute unit and are faster with more registers
// (one row of 27000: 22.3 -> 17.7 us with 4 wavefronts per SIMD in place of 6).  512 threads ask for 6; of 256 threads LDS
// admits four rows, and a fifth (histogram, list and draws in one place) gains under top_p what it loses under top_k.  Without
// AGAIN (drawn items come back) those of 256 have to be asked for the four: weights formed anew take more registers
// (1024 x 27000 uncut, 5 draws: 78 us with three rows, 63 with four).  Each time that weights are formed anew reads the row twice:
// at a temperature of 0.02 of the scores' deviation, 10 draws of 1024 x 27000 take 392 us, at 0.5 of it 83.
template <int DT, int NT, bool LISTS, bool AGAIN>
__global__ __launch_bounds__(NT, NT == 1024 || (NT == 256 && !AGAIN) ? 4 : 6) void sample_long_kernel(
    const typename ScoreType<DT>::raw* __restrict__ scores, int64_t n, int64_t m, int64_t stride,
    const int32_t* __restrict__ ids, int64_t ids_stride, const int64_t* __restrict__ mask_indptr,
    const int32_t* __restrict__ mask_indices, const float* __restrict__ uniforms, int draws,
    SampleParams par, int bits, int32_t* __restrict__ out_ids, float* __restrict__ out_logprob) {
    typedef Chunk<DT> C;
    constexpr int V = C::V, NW = NT / 64, WAVE_CHUNK = 64 * V;
    constexpr int BINS_PER = SM_BINS / NT;
    extern __shared__ uint32_t liked[];   // one bit per item, when there is a filter
    __shared__ __attribute__((aligned(16))) ulonglong2 list[SM_LIST];   // K and weight
    __shared__ uint64_t mass_bins[SM_BINS], piece_mass[SM_BINS];
    __shared__ uint32_t count_bins[SM_BINS];
    __shared__ uint64_t before_of[SM_LIST];
    __shared__ uint64_t part[2][NW];
    __shared__ uint64_t shared_key[2];
    __shared__ uint32_t shared_int[2];
    __shared__ int32_t gone[SM_MAX_DRAWS];   // items drawn so far, when they do not come back
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const double rounder = sm_rounder(bits);
    const int64_t row_chunks = (m + WAVE_CHUNK - 1) / WAVE_CHUNK;
    const int S = (int)((row_chunks + SM_BINS - 1) / SM_BINS);
    const int pieces = (int)((row_chunks + S - 1) / S);   // at most SM_BINS
    const int items = (int)m, last_whole = items - WAVE_CHUNK;   // (items <= 2^30; where the last whole chunk may begin)

    for (int64_t row = blockIdx.x; row < n; row += gridDim.x) {
        const typename ScoreType<DT>::raw* s = scores + row * stride;
        const int32_t* id = LISTS ? ids + row * ids_stride : nullptr;
        __syncthreads();   // the row before is done with the shared arrays
        if (mask_indptr) {
            for (int w = tid; w < pieces * S * (WAVE_CHUNK / 32); w += NT) liked[w] = 0;
            __syncthreads();
            for (int64_t e = mask_indptr[row] + tid; e < mask_indptr[row + 1]; e += NT) {
                const int64_t it = mask_indices[e];
                if (it >= 0 && it < m) atomicOr(&liked[it >> 5], 1u << (it & 31));
            }
            __syncthreads();
        }
        // a lane's first item of chunk `sub` of piece p
        auto first_item = [&](int p, int sub) -> int32_t { return (p * S + sub) * WAVE_CHUNK + lane * V; };
        // its 16 bytes (minus infinity behind the row's end); whether a chunk ends inside the row is asked once for all lanes
        auto load = [&](int p, int sub) -> C {
            const int begin = (p * S + sub) * WAVE_CHUNK;
            C q;
            if (begin <= last_whole) {
                const sm_words x = *reinterpret_cast<const sm_words*>(s + begin + lane * V);
#pragma unroll
                for (int v = 0; v < 4; ++v) q.word[v] = x[v];
                return q;
            }
            const int i = begin + lane * V;
#pragma unroll
            for (int v = 0; v < 4; ++v) q.word[v] = DT == MIREC_F32 ? 0xff800000u : DT == MIREC_BF16 ? 0xff80ff80u : 0xfc00fc00u;
#pragma unroll
            for (int v = 0; v < V; ++v)
                if (i + v < items) {
                    if constexpr (DT == MIREC_F32) q.word[v] = __float_as_uint(s[i + v]);
                    else {
                        const uint32_t raw = __builtin_bit_cast(uint16_t, s[i + v]);
                        q.word[v >> 1] = v & 1 ? (q.word[v >> 1] & 0xffffu) | (raw << 16) : (q.word[v >> 1] & 0xffff0000u) | raw;
                    }
                }
            return q;
        };
        // what is excluded set to minus infinity
        auto filter = [&](C& q, int32_t i) {
            if (__any(q.unsettled())) q.settle();
            if (mask_indptr) {
                const uint32_t out = (liked[i >> 5] >> (i & 31)) & ((1u << V) - 1);
                if (__any(out != 0)) {
#pragma unroll
                    for (int v = 0; v < V; ++v)
                        if ((out >> v) & 1u) q.exclude(v);
                }
            }
            if constexpr (LISTS) {
#pragma unroll
                for (int v = 0; v < V; ++v)
                    if (i + v < items && id[i + v] < 0) q.exclude(v);
            }
        };
        // f(chunk, the lane's first item, its piece, number within the piece) for every chunk of this wavefront, in order,
        // SM_AHEAD loads ahead of the work
        auto each = [&](auto&& f) {
            const int mine = wave < pieces ? ((pieces - wave - 1) / NW + 1) * S : 0;
            C ahead[SM_AHEAD];
            int lp = wave, lsub = 0;   // the chunk to load next
            auto fetch = [&](C& q) {
                if (lp < pieces) q = load(lp, lsub);
                if (++lsub == S) {
                    lsub = 0;
                    lp += NW;
                }
            };
#pragma unroll
            for (int u = 0; u < SM_AHEAD; ++u) fetch(ahead[u]);
            int p = wave, sub = 0;
            for (int c = 0; c < mine; c += SM_AHEAD)
#pragma unroll
                for (int u = 0; u < SM_AHEAD; ++u)
                    if (c + u < mine) {
                        C q = ahead[u];
                        fetch(ahead[u]);
                        const int32_t first = first_item(p, sub);
                        filter(q, first);
                        f(q, first, p, sub);
                        if (++sub == S) {
                            sub = 0;
                            p += NW;
                        }
                    }
        };
        auto order_of = [&](float f, int32_t item) -> uint64_t {
            return ((uint64_t)sm_order(f) << 32) | (0xffffffffu - (uint32_t)item);
        };

        // the best score
        float own_top = -INFINITY;
        each([&](const C& q, int32_t, int, int) {
#pragma unroll
            for (int v = 0; v < V; ++v) own_top = fmaxf(own_top, q.score(v));
        });
        float top = sm_wave_max(own_top);
        if (lane == 0) part[0][wave] = __float_as_uint(top);
        __syncthreads();
#pragma unroll
        for (int w = 0; w < NW; ++w) top = fmaxf(top, __uint_as_float((uint32_t)part[0][w]));
        __syncthreads();
        if (!(top > -INFINITY)) {
            for (int d = tid; d < draws; d += NT) {
                out_ids[row * draws + d] = -1;
                out_logprob[row * draws + d] = -INFINITY;
            }
            continue;
        }
        const RowCuts cuts = sm_cuts(par, row, m, bits);
        const float step32 = cuts.step > 0.0 ? (float)(cuts.step * 32.0) : 32.f;   // (any scale finds the best item)
        const double best = (double)top;
        auto weight = [&](float f) -> uint64_t { return sm_weight(f, best, cuts.step, rounder); };
        // a bin of the first histogram: in 1/32 octaves below the best, everything from 32 octaves on in the last
        auto first_bin = [&](float f) -> uint32_t {
            const uint32_t b = (uint32_t)((top - f) * step32);
            return b < SM_BINS - 1 ? b : SM_BINS - 1;
        };

        // The bin in which a running sum over the bins, from `base` on, satisfies here(sum before it, its own); -1 if none
        // does.  Leaves the sum before the bin in shared_key[1]; `all`: the sum over all bins.
        auto find_bin = [&](auto bins, uint64_t base, auto&& here, uint64_t& all) -> int {
            uint64_t sum = 0, mine[BINS_PER];
#pragma unroll
            for (int i = 0; i < BINS_PER; ++i) {
                mine[i] = (uint64_t)bins[tid * BINS_PER + i];
                sum += mine[i];
            }
            const uint64_t inc = sm_wave_scan(sum);
            if (lane == 63) part[0][wave] = inc;
            if (tid == 0) {
                shared_int[0] = 0;
                shared_key[1] = 0;
            }
            __syncthreads();
            uint64_t at = base + inc - sum;
            all = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                at += w < wave ? part[0][w] : 0ull;
                all += part[0][w];
            }
            int found = -1;
            uint64_t found_at = 0;
#pragma unroll
            for (int i = 0; i < BINS_PER; ++i) {
                if (here(at, mine[i], all)) {
                    found = tid * BINS_PER + i;
                    found_at = at;
                }
                at += mine[i];
            }
            if (found >= 0) atomicMax(&shared_int[0], (uint32_t)found + 1);
            __syncthreads();
            const int b = (int)shared_int[0] - 1;
            if (found == b && b >= 0) shared_key[1] = found_at;
            __syncthreads();
            return b;
        };

        // A handful of items are to stay.  The top_k-th best of the threads' own best scores is not above the row's
        // top_k-th best score, and few scores are above it: those go to a list, where every sum is formed by comparing each
        // with each.
        if (cuts.top_k <= SM_FEW / 2) {
            for (int b = tid; b < SM_BINS; b += NT) count_bins[b] = 0;
            if (tid == 0) shared_int[1] = 0;
            __syncthreads();
            if (own_top > -INFINITY) atomicAdd(&count_bins[first_bin(own_top)], 1u);
            __syncthreads();
            uint64_t all;
            const uint64_t target = (uint64_t)cuts.top_k;
            const int found = find_bin(count_bins, 0, [&](uint64_t at, uint64_t mine, uint64_t) { return at < target && at + mine >= target; },
                                       all);
            const uint32_t last_bin = found >= 0 ? (uint32_t)found : SM_BINS - 1;   // (fewer threads with scores: all of them)
            each([&](const C& q, int32_t first, int, int) {
                float most = q.score(0);
#pragma unroll
                for (int v = 1; v < V; ++v) most = fmaxf(most, q.score(v));
                if (!__any(most > -INFINITY && first_bin(most) <= last_bin)) return;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float f = q.score(v);
                    if (f > -INFINITY && first_bin(f) <= last_bin) {
                        const uint32_t e = atomicAdd(&shared_int[1], 1u);
                        if (e < SM_FEW) list[e].x = order_of(f, first + v);
                    }
                }
            });
            __syncthreads();
            const uint32_t have = shared_int[1];
            if (have <= SM_FEW) {
                // Entry e of the list to NT / SM_FEW threads, which share the entries it is compared with.
                constexpr uint32_t SLICES = NT / SM_FEW;
                const uint32_t e = tid % SM_FEW, slice = tid / SM_FEW;
                uint64_t* sums = mass_bins;                 // by entry: the mass before it in rank order, then its running sum
                uint64_t* runs = mass_bins + SM_FEW;
                uint64_t K = 0, w = 0;
                if (slice == 0) {
                    sums[e] = runs[e] = 0;
                    count_bins[e] = 0;
                    if (e < have) {
                        K = list[e].x;
                        w = weight(sm_unorder((uint32_t)(K >> 32)));
                        list[e].y = w;
                    }
                    if (e == 0) shared_key[0] = shared_key[1] = 0;
                }
                __syncthreads();
                if (e < have) {
                    K = list[e].x;
                    uint32_t rank = 0;
                    uint64_t before = 0;
#pragma unroll 4
                    for (uint32_t j = slice; j < have; j += SLICES) {
                        const ulonglong2 x = list[j];
                        rank += x.x > K ? 1u : 0u;
                        before += x.x > K ? x.y : 0ull;
                    }
                    if (SLICES > 1) {
                        atomicAdd(&count_bins[e], rank);
                        atomicAdd((unsigned long long*)&sums[e], (unsigned long long)before);
                    } else {
                        count_bins[e] = rank;
                        sums[e] = before;
                    }
                }
                __syncthreads();
                uint32_t rank = 0;
                uint64_t before = 0;
                if (slice == 0 && e < have) {
                    rank = count_bins[e];
                    before = sums[e];
                    // the last entry that top_k leaves has all their mass up to and with it
                    if (rank + 1 == (cuts.top_k < (int64_t)have ? (uint32_t)cuts.top_k : have)) shared_key[0] = before + w;
                }
                __syncthreads();
                if (slice == 0 && e < have) {
                    const uint64_t bound = cuts.top_p < 1.0 ? sm_bound(cuts.top_p, shared_key[0]) : ~0ull;
                    const bool stays = rank < cuts.top_k && (rank == 0 || before < bound) && w >= cuts.floor_w;
                    w = stays ? w : 0ull;
                    list[e].y = w;
                    count_bins[e] = stays ? 1u : 0u;
                }
                __syncthreads();
                if (e < have) {   // in index order: a larger complement is a smaller index
                    uint64_t run = 0;
#pragma unroll 4
                    for (uint32_t j = slice; j < have; j += SLICES) {
                        const ulonglong2 x = list[j];
                        run += (uint32_t)x.x >= (uint32_t)K ? x.y : 0ull;
                    }
                    if (SLICES > 1) atomicAdd((unsigned long long*)&runs[e], (unsigned long long)run);
                    else runs[e] = run;
                    atomicAdd((unsigned long long*)&shared_key[1], slice == 0 ? (unsigned long long)w : 0ull);
                }
                __syncthreads();
                if (wave != 0) continue;
                constexpr int SLOTS = SM_FEW / 64;
                uint64_t total = shared_key[1], item_K[SLOTS], item_w[SLOTS], run[SLOTS];
                uint32_t left = 0;   // slots that are kept and not drawn yet
                double best_left = best;
#pragma unroll
                for (int i = 0; i < SLOTS; ++i) {
                    const bool real = lane + 64 * i < (int)have;
                    left |= real && count_bins[lane + 64 * i] != 0 ? 1u << i : 0u;
                    item_K[i] = real ? list[lane + 64 * i].x : 0ull;
                    item_w[i] = real ? list[lane + 64 * i].y : 0ull;
                    run[i] = real ? runs[lane + 64 * i] : 0ull;
                }
                for (int d = 0; d < draws; ++d) {
                    if (total == 0) {
                        if (lane == 0) {
                            out_ids[row * draws + d] = -1;
                            out_logprob[row * draws + d] = -INFINITY;
                        }
                        continue;
                    }
                    const uint64_t t = sm_target(uniforms[row * draws + d], total);
                    uint64_t out_K = 0, out_w = 0;
#pragma unroll
                    for (int i = 0; i < SLOTS; ++i) {
                        const bool here = item_w[i] != 0 && run[i] > t && run[i] - item_w[i] <= t;
                        out_K = here ? item_K[i] : out_K;
                        out_w = here ? item_w[i] : out_w;
                    }
                    if (out_w != 0) {
                        const int32_t item = (int32_t)(0xffffffffu - (uint32_t)out_K);
                        out_ids[row * draws + d] = LISTS ? id[item] : item;
                        out_logprob[row * draws + d] = sm_logprob(sm_unorder((uint32_t)(out_K >> 32)), best_left, cuts.step, total, bits);
                    }
                    if (!AGAIN) {
                        const int l = __builtin_ctzll(__ballot(out_w != 0));
                        const uint64_t gone_K = sm_lane(out_K, l), less = sm_lane(out_w, l);
                        total -= less;
#pragma unroll
                        for (int i = 0; i < SLOTS; ++i) {
                            run[i] -= (uint32_t)gone_K >= (uint32_t)item_K[i] ? less : 0ull;
                            item_w[i] = item_K[i] == gone_K ? 0ull : item_w[i];
                            left &= item_K[i] == gone_K ? ~(1u << i) : ~0u;
                        }
                        if (total < par.renew_below && __any(left != 0)) {
                            float most = -INFINITY;
#pragma unroll
                            for (int i = 0; i < SLOTS; ++i) most = fmaxf(most, (left >> i) & 1u ? sm_unorder((uint32_t)(item_K[i] >> 32)) : -INFINITY);
                            best_left = (double)sm_wave_max(most);
                            uint64_t sum = 0;
#pragma unroll
                            for (int i = 0; i < SLOTS; ++i) {
                                const float f = sm_unorder((uint32_t)(item_K[i] >> 32));
                                item_w[i] = (left >> i) & 1u ? sm_weight(f, best_left, cuts.step, rounder) : 0ull;
                                run[i] = 0;
                                sum += item_w[i];
                                if (lane + 64 * i < (int)have) list[lane + 64 * i].y = item_w[i];
                            }
                            total = sm_wave_sum(sum);
                            asm volatile("" ::: "memory");   // written by other lanes of this wavefront, in order
                            for (int j = 0; j < (int)have; ++j) {
                                const ulonglong2 x = list[j];
#pragma unroll
                                for (int i = 0; i < SLOTS; ++i) run[i] += (uint32_t)x.x >= (uint32_t)item_K[i] ? x.y : 0ull;
                            }
                            asm volatile("" ::: "memory");
                        }
                    }
                }
                continue;
            }
            __syncthreads();   // the list overflowed: the cuts below
        }

        // the last item that stays; at first every item that is not excluded does
        float cut_f = -INFINITY;
        int32_t cut_i = -1;
        auto kept = [&](float f, int32_t item) -> bool { return (f > cut_f) | ((f == cut_f) & (item <= cut_i)); };
        // whether a wavefront's chunk holds an item that may stay
        auto any_kept = [&](const C& q) -> bool {
            float most = q.score(0);
#pragma unroll
            for (int v = 1; v < V; ++v) most = fmaxf(most, q.score(v));
            return __any(most >= cut_f && most > -INFINITY);
        };
        bool summed = false;   // piece_mass holds the kept mass of every piece
        // Moves `cut` to the item at the border: the target-th in order (by count), or the last item whose
        // predecessors hold less than the share top_p of what stayed so far.  Where the row has no border it stays.
        auto find_cut = [&](auto by_mass, uint64_t target, double top_p) {
            constexpr bool BY_MASS = decltype(by_mass)::value;
            uint64_t base = 0;      // count or mass of the items above the current range
            uint64_t lo = 0, hi = 0, bound = 0;
            int shift = -1;         // -1: the first histogram
            for (;;) {
                for (int b = tid; b < SM_BINS; b += NT) {
                    if (BY_MASS) mass_bins[b] = 0;
                    else count_bins[b] = 0;
                }
                if (tid == 0) {
                    shared_int[1] = 0;   // entries in the list
                    shared_key[0] = ~0ull;
                }
                __syncthreads();
                auto count = [&](uint32_t b, float f) {
                    if (BY_MASS) atomicAdd((unsigned long long*)&mass_bins[b], (unsigned long long)weight(f));
                    else atomicAdd(&count_bins[b], 1u);
                };
                if (shift < 0) {
                    each([&](const C& q, int32_t first, int, int) {
                        if (!any_kept(q)) return;
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            const float f = q.score(v);
                            if (kept(f, first + v)) count(first_bin(f), f);
                        }
                    });
                } else {
                    each([&](const C& q, int32_t first, int, int) {
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            const float f = q.score(v);
                            const uint64_t K = order_of(f, first + v);
                            if (K >= lo && K <= hi) count((uint32_t)((hi - K) >> shift), f);
                        }
                    });
                }
                __syncthreads();
                // The border's bin.  By count: the one that takes the running count to the target.  By mass: the last
                // with mass that starts below the bound, or the first with mass.
                uint64_t all;
                int b;
                if constexpr (BY_MASS)
                    b = find_bin(mass_bins, base, [&](uint64_t at, uint64_t mine, uint64_t sum) {
                        if (shift < 0) bound = sm_bound(top_p, sum);
                        return mine > 0 && (at < bound || at == base);
                    }, all);
                else
                    b = find_bin(count_bins, base, [&](uint64_t at, uint64_t mine, uint64_t) { return at < target && at + mine >= target; },
                                 all);
                if (b < 0) return;   // by count: fewer items than the target
                base = shared_key[1];
                auto member = [&](float f, int32_t item) -> bool {
                    if (shift < 0) return first_bin(f) == (uint32_t)b && kept(f, item);
                    const uint64_t K = order_of(f, item);
                    return K >= lo && K <= hi && (int)((hi - K) >> shift) == b;
                };
                if (BY_MASS && shift < 0) {
                    // the members to the list, the mass of what is above the bin to its pieces: one pass for both
                    uint64_t w = 0;
                    each([&](const C& q, int32_t first, int p, int sub) {
                        if (any_kept(q)) {
#pragma unroll
                            for (int v = 0; v < V; ++v) {
                                const float f = q.score(v);
                                const uint32_t in = first_bin(f);
                                const bool on = (in <= (uint32_t)b) & kept(f, first + v);
                                if (__any(on)) {
                                    const uint64_t wf = weight(f);
                                    w += on & (in < (uint32_t)b) & (wf >= cuts.floor_w) ? wf : 0ull;
                                }
                                if (on && in == (uint32_t)b) {
                                    const uint32_t e = atomicAdd(&shared_int[1], 1u);
                                    if (e < SM_LIST) list[e].x = order_of(f, first + v);
                                }
                            }
                        }
                        if (sub == S - 1) {
                            w = sm_wave_sum(w);
                            if (lane == 0) piece_mass[p] = w;
                            w = 0;
                        }
                    });
                } else {
                    each([&](const C& q, int32_t first, int, int) {
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            const float f = q.score(v);
                            if (member(f, first + v)) {
                                const uint32_t e = atomicAdd(&shared_int[1], 1u);
                                if (e < SM_LIST) list[e].x = order_of(f, first + v);
                            }
                        }
                    });
                }
                __syncthreads();
                const uint32_t members = shared_int[1];
                if (members <= SM_LIST) {
                    // every entry to `slices` threads, which share the entries it is compared with
                    int span = 64;
                    while (span < (int)members) span *= 2;
                    const int slices = NT / span > 0 ? NT / span : 1;
                    for (uint32_t e = tid; e < members; e += NT) {
                        list[e].y = BY_MASS ? weight(sm_unorder((uint32_t)(list[e].x >> 32))) : 1ull;
                        before_of[e] = base;
                    }
                    __syncthreads();
                    for (uint32_t e0 = 0; e0 < members; e0 += NT) {
                        const uint32_t e = e0 + (tid & (span - 1));
                        if (e < members && (int)(tid / span) < slices) {
                            const uint64_t K = list[e].x;
                            uint64_t before = 0;
#pragma unroll 4
                            for (uint32_t j = tid / span; j < members; j += slices) before += list[j].x > K ? list[j].y : 0ull;
                            atomicAdd((unsigned long long*)&before_of[e], (unsigned long long)before);
                        }
                    }
                    __syncthreads();
                    for (uint32_t e = tid; e < members; e += NT) {
                        const ulonglong2 x = list[e];
                        const uint64_t before = before_of[e];
                        const bool stays = BY_MASS ? x.y > 0 && (before < bound || before == base) : before < target;
                        if (stays) {
                            atomicMin((unsigned long long*)&shared_key[0], (unsigned long long)x.x);
                            // (by mass in the first histogram: what lies above the bin is in the pieces already)
                            if (BY_MASS && shift < 0 && x.y >= cuts.floor_w)
                                atomicAdd((unsigned long long*)&piece_mass[(int32_t)(0xffffffffu - (uint32_t)x.x) / (WAVE_CHUNK * S)],
                                          (unsigned long long)x.y);
                        }
                    }
                    if (BY_MASS && shift < 0) summed = true;
                    __syncthreads();
                    cut_f = sm_unorder((uint32_t)(shared_key[0] >> 32));
                    cut_i = (int32_t)(0xffffffffu - (uint32_t)shared_key[0]);
                    __syncthreads();
                    return;
                }
                // too many for the list: the bin's range of K, in equal parts
                if (shift < 0) {
                    uint64_t most = 0, least = ~0ull;
                    each([&](const C& q, int32_t first, int, int) {
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            const float f = q.score(v);
                            if (member(f, first + v)) {
                                const uint64_t K = order_of(f, first + v);
                                most = K > most ? K : most;
                                least = K < least ? K : least;
                            }
                        }
                    });
                    __syncthreads();
                    if (tid == 0) shared_key[1] = 0;
                    __syncthreads();
                    atomicMax((unsigned long long*)&shared_key[1], (unsigned long long)most);
                    atomicMin((unsigned long long*)&shared_key[0], (unsigned long long)least);
                    __syncthreads();
                    hi = shared_key[1];
                    lo = shared_key[0];
                } else {
                    hi -= (uint64_t)b << shift;
                    const uint64_t down = hi - ((1ull << shift) - 1);
                    lo = down > lo ? down : lo;
                }
                shift = 64 - __builtin_clzll((hi - lo) | 1ull) - 10;
                shift = shift > 0 ? shift : 0;
                __syncthreads();
            }
        };

        for (int p = tid; p < SM_BINS; p += NT) piece_mass[p] = 0;
        if (cuts.top_k < m) find_cut(std::false_type{}, (uint64_t)cuts.top_k, 0.0);
        if (cuts.top_p < 1.0) find_cut(std::true_type{}, 0ull, cuts.top_p);

        // The kept mass of every piece, then its running sum in index order.
        auto kept_weight = [&](float f, int32_t item) -> uint64_t {
            const uint64_t w = weight(f);
            return kept(f, item) & (w >= cuts.floor_w) ? w : 0ull;
        };
        const bool uncut = cut_f == -INFINITY && cuts.floor_w == 0;   // an excluded item has no weight
        __syncthreads();
        if (!summed) {
            uint64_t w = 0;
            each([&](const C& q, int32_t first, int p, int sub) {
                if (uncut) {
#pragma unroll
                    for (int v = 0; v < V; ++v) w += weight(q.score(v));
                } else if (any_kept(q)) {
#pragma unroll
                    for (int v = 0; v < V; ++v) w += kept_weight(q.score(v), first + v);
                }
                if (sub == S - 1) {
                    w = sm_wave_sum(w);
                    if (lane == 0) piece_mass[p] = w;
                    w = 0;
                }
            });
        }
        __syncthreads();
        auto scan_pieces = [&]() -> uint64_t {
            uint64_t sum = 0, mine[BINS_PER];
#pragma unroll
            for (int i = 0; i < BINS_PER; ++i) {
                mine[i] = piece_mass[tid * BINS_PER + i];
                sum += mine[i];
            }
            const uint64_t inc = sm_wave_scan(sum);
            if (lane == 63) part[0][wave] = inc;
            __syncthreads();
            uint64_t at = inc - sum, all = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                at += w < wave ? part[0][w] : 0ull;
                all += part[0][w];
            }
#pragma unroll
            for (int i = 0; i < BINS_PER; ++i) {
                at += mine[i];
                piece_mass[tid * BINS_PER + i] = at;
            }
            __syncthreads();
            return all;
        };
        uint64_t total = scan_pieces();

        // A draw: the piece its number falls into, by two looks at the running sums, then the item, from the piece's
        // scores once more.  `weigh` gives a kept item's weight (0 where it has none, or is drawn already); returns the item's
        // weight and leaves its number in `item`.
        auto draw = [&](int d, double best_left, auto&& weigh, int32_t& item) -> uint64_t {
            const uint64_t t = sm_target(uniforms[row * draws + d], total);
            const int p16 = __builtin_ctzll(__ballot(piece_mass[lane * (SM_BINS / 64) + SM_BINS / 64 - 1] > t));
            const uint64_t upto16 = piece_mass[p16 * (SM_BINS / 64) + (lane & (SM_BINS / 64 - 1))];
            const int p = p16 * (SM_BINS / 64) + __builtin_ctzll(__ballot(lane >= SM_BINS / 64 || upto16 > t));
            uint64_t run = p > 0 ? piece_mass[p - 1] : 0ull;
            for (int sub = 0; sub < S; ++sub) {
                C q = load(p, sub);
                const int32_t first = first_item(p, sub);
                filter(q, first);
                uint64_t w[V], mine_w = 0;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    w[v] = weigh(q.score(v), first + v);
                    mine_w += w[v];
                }
                const uint64_t upto = run + sm_wave_scan(mine_w);
                const uint64_t votes = __ballot(upto > t);
                if (votes == 0) {
                    run = sm_lane(upto, 63);
                    continue;
                }
                const int l = __builtin_ctzll(votes);
                uint64_t before = upto - mine_w, drawn = 0;
                int at_v = 0;
                bool found = false;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    if (!found && w[v] && before + w[v] > t) {
                        found = true;
                        at_v = v;
                        drawn = w[v];
                    }
                    before += w[v];
                }
                if (lane == l) {
                    const int32_t mine = first + at_v;
                    float f = 0.f;
#pragma unroll
                    for (int v = 0; v < V; ++v) f = at_v == v ? q.score(v) : f;
                    out_ids[row * draws + d] = LISTS ? id[mine] : mine;
                    out_logprob[row * draws + d] = sm_logprob(f, best_left, cuts.step, total, bits);
                }
                item = __builtin_amdgcn_readlane(first + at_v, l);
                const uint64_t less = sm_lane(drawn, l);
                for (int j = p + lane; !AGAIN && j < SM_BINS; j += 64) piece_mass[j] -= less;
                asm volatile("" ::: "memory");
                return less;
            }
            return 0;   // (not reached: the piece holds the number)
        };
        if (AGAIN) {   // shared out over the wavefronts
            int32_t item;
            for (int d = wave; d < draws; d += NW) draw(d, best, kept_weight, item);
            continue;
        }
        // Drawn items that stay away: one wavefront draws and takes an item's weight out of every running sum behind it.  Where
        // the sum has become too low, all wavefronts form the weights of what is left anew.
        double best_left = best;
        auto is_gone = [&](int32_t item, int taken) -> bool {
            bool out = false;
            for (int j = 0; j < taken; ++j) out |= gone[j] == item;
            return out;
        };
        for (int d = 0;;) {
            if (wave == 0) {
                for (; d < draws && total >= par.renew_below; ++d) {
                    int32_t item = 0;
                    total -= draw(d, best_left, [&](float f, int32_t i) -> uint64_t {
                        // (what has left may have been better than the best of the rest: its weight is none)
                        const bool in = kept(f, i) && (cuts.floor_w == 0 || weight(f) >= cuts.floor_w) && !is_gone(i, d);
                        return in ? sm_weight(f, best_left, cuts.step, rounder) : 0ull;
                    }, item);
                    if (lane == 0) gone[d] = item;
                    asm volatile("" ::: "memory");
                }
                if (lane == 0) shared_int[0] = (uint32_t)d;
            }
            __syncthreads();
            d = (int)shared_int[0];
            if (d == draws) break;
            // the drawn items in a table (open addressing, at most half full)
            int32_t* table = reinterpret_cast<int32_t*>(mass_bins);
            constexpr uint32_t SLOTS = 2 * SM_MAX_DRAWS;
            static_assert(sizeof(mass_bins) >= SLOTS * 4, "two places for every draw");
            auto slot_of = [&](int32_t item) -> uint32_t { return ((uint32_t)item * 2654435769u >> 16) & (SLOTS - 1); };
            for (uint32_t i = tid; i < SLOTS; i += NT) table[i] = -1;
            for (int p = tid; p < SM_BINS; p += NT) piece_mass[p] = 0;
            __syncthreads();
            for (int j = tid; j < d; j += NT) {
                uint32_t at = slot_of(gone[j]);
                while (atomicCAS(&table[at], -1, gone[j]) != -1) at = (at + 1) & (SLOTS - 1);
            }
            __syncthreads();
            auto stays = [&](float f, int32_t item) -> bool {
                if (!kept(f, item) || (cuts.floor_w > 0 && weight(f) < cuts.floor_w)) return false;
                uint32_t at = slot_of(item);
                while (table[at] != -1 && table[at] != item) at = (at + 1) & (SLOTS - 1);
                return table[at] == -1;
            };
            float most = -INFINITY;
            each([&](const C& q, int32_t first, int, int) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float f = q.score(v);
                    if (f > most && stays(f, first + v)) most = f;
                }
            });
            most = sm_wave_max(most);
            if (lane == 0) part[0][wave] = __float_as_uint(most);
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; ++w) most = fmaxf(most, __uint_as_float((uint32_t)part[0][w]));
            if (!(most > -INFINITY)) {   // nothing is left
                for (int j = d + tid; j < draws; j += NT) {
                    out_ids[row * draws + j] = -1;
                    out_logprob[row * draws + j] = -INFINITY;
                }
                break;
            }
            best_left = (double)most;
            uint64_t w = 0;
            each([&](const C& q, int32_t first, int p, int sub) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float f = q.score(v);
                    if (f <= most && stays(f, first + v)) w += sm_weight(f, best_left, cuts.step, rounder);
                }
                if (sub == S - 1) {
                    w = sm_wave_sum(w);
                    if (lane == 0) piece_mass[p] = w;
                    w = 0;
                }
            });
            __syncthreads();
            total = scan_pieces();
        }
    }
}

template <int DT, int E, int R, bool AGAIN>
static int launch_short(const typename ScoreType<DT>::raw* scores, int64_t n, int m, int64_t stride, const int32_t* ids,
                        int64_t ids_stride, const int64_t* mask_indptr, const int32_t* mask_indices, const float* uniforms,
                        int draws, const SampleParams& par, int bits, int32_t* out_ids, float* out_logprob,
                        hipStream_t stream) {
    // each row its lanes until the chip is full (256 compute units of 28 wavefronts), then runs of up to 64 rows
    int64_t rows_each = n / (256 * 28 * R);
    rows_each = rows_each < 1 ? 1 : rows_each > 64 ? 64 : rows_each;
    const int64_t blocks = (n + 4 * R * rows_each - 1) / (4 * R * rows_each);
    MIREC_REQUIRE(blocks < ((int64_t)1 << 24), MIREC_E_UNSUPPORTED, "mirec_sample: more than 2^32 rows");
    hipLaunchKernelGGL((sample_short_kernel<DT, E, R, AGAIN>), dim3((unsigned)blocks), dim3(256), 0, stream, scores, n, m, stride, ids,
                       ids_stride, mask_indptr, mask_indices, uniforms, draws, (int)rows_each, par, bits, out_ids,
                       out_logprob);
    MIREC_LAUNCH_CHECK();
    return MIREC_OK;
}

template <int DT, int NT, bool LISTS, bool AGAIN>
static int launch_long(const typename ScoreType<DT>::raw* scores, int64_t n, int64_t m, int64_t stride, const int32_t* ids,
                       int64_t ids_stride, const int64_t* mask_indptr, const int32_t* mask_indices, const float* uniforms,
                       int draws, const SampleParams& par, int bits, int32_t* out_ids, float* out_logprob,
                       hipStream_t stream) {
    // the filter's bitmap of a long row (up to 64 KiB) takes more dynamic LDS than a kernel gets unasked
    static OncePerDevice once;   // idempotent; a race only repeats the call
    bool* done = once.slot();
    MIREC_REQUIRE(done, MIREC_E_HIP, "mirec_sample: cannot read the current device");
    if (!*done) {
        MIREC_HIP(hipFuncSetAttribute((const void*)sample_long_kernel<DT, NT, LISTS, AGAIN>, hipFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)(SM_MAX_MASKED_ITEMS / 8)));
        *done = true;
    }
    // (a bit for every item of whole pieces; at SM_MAX_MASKED_ITEMS these end with the row)
    constexpr int64_t CHUNK_ITEMS = 64 * Chunk<DT>::V;
    const int64_t chunks = (m + CHUNK_ITEMS - 1) / CHUNK_ITEMS, per = (chunks + SM_BINS - 1) / SM_BINS;
    const size_t lds = mask_indptr ? (size_t)((chunks + per - 1) / per * per * (CHUNK_ITEMS / 8)) : 0;
    hipLaunchKernelGGL((sample_long_kernel<DT, NT, LISTS, AGAIN>), dim3((unsigned)(n < 262144 ? n : 262144)), dim3(NT), lds, stream, scores,
                       n, m, stride, ids, ids_stride, mask_indptr, mask_indices, uniforms, draws, par, bits, out_ids, out_logprob);
    MIREC_LAUNCH_CHECK();
    return MIREC_OK;
}

template <int DT, bool AGAIN>
static int launch_rows(const void* scores_, int64_t n, int64_t m, int64_t stride, const int32_t* ids, int64_t ids_stride,
                         const int64_t* mask_indptr, const int32_t* mask_indices, const float* uniforms, int draws,
                         const SampleParams& par, int bits, int32_t* out_ids, float* out_logprob, hipStream_t stream) {
    const typename ScoreType<DT>::raw* scores = (const typename ScoreType<DT>::raw*)scores_;
#define MIREC_SAMPLE_ARGS \
    stride, ids, ids_stride, mask_indptr, mask_indices, uniforms, draws, par, bits, out_ids, out_logprob, stream
    // Two rows to a wavefront where a row has at most two items a lane then (262144 lists of 50: 107 -> 76 us).  Up to 128
    // items ranked lists, which are in order, still gain (of 100: 139 -> 107 us); dense rows cost their comparisons and are
    // sooner done with a wavefront each (one of 100: 17 us shared, 11 us alone; 262144: 1.28 ms either way).
    if (m <= 64) return launch_short<DT, 2, 2, AGAIN>(scores, n, (int)m, MIREC_SAMPLE_ARGS);
    if (ids && m <= 128) return launch_short<DT, 4, 2, AGAIN>(scores, n, (int)m, MIREC_SAMPLE_ARGS);
    if (m <= 128) return launch_short<DT, 2, 1, AGAIN>(scores, n, (int)m, MIREC_SAMPLE_ARGS);
    if (m <= SM_SHORT) return launch_short<DT, 4, 1, AGAIN>(scores, n, (int)m, MIREC_SAMPLE_ARGS);
    // Threads to a row: as few as fill the chip, since a row's barriers cost by the thread (256 / 512 threads, uncut: 1024 x 27000
    // 47 / 53 us, 4096 x 12000 74 / 92 us; under top_k 50: 41 / 60 and 86 / 132 us); few long rows need more (512 x 200000 under
    // top_p 831 / 612 us; with 1024 threads 256 x 27000 under top_p 36 us, with 512 47).
    if (ids && n <= SM_SOME_ROWS && m > 16384) return launch_long<DT, 512, true, AGAIN>(scores, n, m, MIREC_SAMPLE_ARGS);
    if (ids) return launch_long<DT, 256, true, AGAIN>(scores, n, m, MIREC_SAMPLE_ARGS);
    if (n <= SM_FEW_ROWS && m > 8192) return launch_long<DT, 1024, false, AGAIN>(scores, n, m, MIREC_SAMPLE_ARGS);
    if (n <= SM_SOME_ROWS && m > 16384) return launch_long<DT, 512, false, AGAIN>(scores, n, m, MIREC_SAMPLE_ARGS);
    return launch_long<DT, 256, false, AGAIN>(scores, n, m, MIREC_SAMPLE_ARGS);
#undef MIREC_SAMPLE_ARGS
}

// All of one mode (instantiated in a source file of its own each: a minute of the compiler's time).
template <bool AGAIN>
static int launch_sample(const void* scores, int dtype, int64_t n, int64_t m, int64_t stride, const int32_t* ids, int64_t ids_stride,
                         const int64_t* mask_indptr, const int32_t* mask_indices, const float* uniforms, int draws,
                         const SampleParams& par, int bits, int32_t* out_ids, float* out_logprob, hipStream_t stream) {
    auto* launch = dtype == MIREC_F32   ? launch_rows<MIREC_F32, AGAIN>
                   : dtype == MIREC_F16 ? launch_rows<MIREC_F16, AGAIN>
                                        : launch_rows<MIREC_BF16, AGAIN>;
    return launch(scores, n, m, stride, ids, ids_stride, mask_indptr, mask_indices, uniforms, draws, par, bits, out_ids, out_logprob,
                  stream);
}

typedef int SampleLaunch(const void* scores, int dtype, int64_t n, int64_t m, int64_t stride, const int32_t* ids, int64_t ids_stride,
                         const int64_t* mask_indptr, const int32_t* mask_indices, const float* uniforms, int draws,
                         const SampleParams& par, int bits, int32_t* out_ids, float* out_logprob, hipStream_t stream);
SampleLaunch sample_with_replacement, sample_without_replacement;

}  // namespace mirec
