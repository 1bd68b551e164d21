// Distilling a factor model from a teacher's ranked lists: per row the Kullback-Leibler divergence of the student's
// softmax over the whole catalogue from the teacher's distribution on its list, and its gradients, from the factor
// matrices -- as in the top-K pass the matrix of scores is never written.  The teacher's side is what the reference
// serves for a user (recommenders/als_recommender.py:181-186): ids and scores, best first.
//
//   z_bj = x_b . y_j / T,  q_b = softmax(z_b) over all m items,  p_b = softmax(t_b / T) over the list (or
//   exp(t / T - lse) with the teacher's log-sum-exp given: what the list leaves, p_r = 1 - sum p, is one class more,
//   which the student gives q_r = 1 - sum over the list of q)
//   loss_b = T^2 [ sum_list p (log p - log q) + p_r (log p_r - log q_r) ]
//   d loss_b / d (x_b . y_j) = T (q_j - p_j) on the list, T (1 - p_r / q_r) q_j elsewhere (T q_j without the class)
//
// Without the class, with mean_b = sum_j q_bj y_j over all items
//   dX_b = grad_b T [ mean_b - sum_list p_k y_k ],   dY_j = sum_b grad_b T g_bj x_b,
//   g_bj = q_bj, or q_k - p_k where j is on row b's list.
// With it nothing is formed as a difference of near values (a student that is nearly certain of its list leaves a q_r of
// 1e-6, less than the fp32 error of one): the pass over the items leaves the listed ones out, so that its mass and mean
// are those of the rest, S_b = sum e_bj and mean_b = sum e_bj y_j / S_b over j off the list, e the exponentials; the
// list's own logits complete the log-sum-exp, q_r = S_b / (S_b + sum_list e), and
//   dX_b = grad_b T [ (q_r - p_r) mean_b + sum_list (q_k - p_k) y_k ],   g_bj = (q_r - p_r) e_bj / S_b off the list.
//
// The two passes over the n x m logits have one form: a wavefront owns 32 rows of one side (in registers), the other
// side streams through LDS in tiles of 32 rows, a tile's 32 x 32 logits come off the matrix cores with the owned rows
// as columns, so that a lane holds 16 logits of ONE owned row, become probabilities in registers and go straight back
// into the matrix cores as the operand that weights the streamed rows: the streamed side's image is laid out for that
// (below) and no logit passes through LDS or memory.
//   distill_forward_kernel   owns rows of X, streams Y: running maximum, mass and mean of the items (dX's dense part); with
//                            the class the listed items' logits become minus infinity, found by the lists' entries
//                            grouped by (row tile, item tile) before the pass (4096 x 27000 at 128, lists of 100: a step
//                            takes 414 us with all this, 391 without)
//   distill_backward_kernel  owns rows of Y, streams X: dY; the logits are formed a second time (three of twelve
//                            matrix products) because keeping them would write and read n m of them
// What bounds them: the matrix cores from 128 columns on (2048 x 200000 at 128: 0.51 and 0.57 ms, from run to run 1.08 to 1.16
// PFLOP/s of plane products; a large fp16 product of the library reaches 1.15 here; 4096 x 27000 with the class: 0.17 and
// 0.20 ms); below, the exponentials and conversions of a logit beside few products (1024 x 27000 at 64: 27 and 42 us, 0.6
// PFLOP/s).
//
// fp32 on the fp16 matrix cores: an operand is two fp16 planes, hi = fp16(v), mid = fp16(v - hi), of the value scaled
// by a power of two that puts its matrix's largest entry just below 2^15, and a product is hi hi + hi mid + mid hi in
// fp32 (mid mid is below 2^-24 of it).  Entries within 2^-18 of the largest keep 22 bits or more, smaller ones an
// absolute error of 2^-40 of the largest, which is what a sum with the large ones leaves of them anyway.
#include <float.h>

#include "common.h"

namespace mirec {

constexpr int DI_LIST = MIREC_DISTILL_MAX_LIST;   // longest list
constexpr int64_t DI_MANY_ROWS = 1024;            // beyond: a wavefront per row in distill_list_kernel
constexpr int DI_THREADS = 256;
constexpr int DI_NW = 8;                          // wavefronts of a workgroup of the two passes
constexpr int DI_OWN = 32 * DI_NW;                // rows it owns
constexpr int DI_PARTS = 256;                     // partial maxima of a matrix
constexpr int DI_MAX_THREADS = 1024;              // of the workgroups that find them and group lists
constexpr int DI_RANGES = 256;                    // most ranges that the items are cut into in the forward pass
constexpr int DI_PREPARE_THREADS = DI_MAX_THREADS;
constexpr int DI_WEIGH_BLOCKS = 64;
constexpr int DI_BINS = 4096;                     // item tiles that di_group counts at a time
constexpr int DI_CUS = 256;                       // workgroups that run at once
constexpr int DI_JOIN_STEPS = 4;                  // of the backward pass: what joining cut blocks takes
constexpr float DI_HEADROOM = 7.f;                // log2 of a probability's scale when its row's reference is current

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// Image of 32 factor rows (a tile), 256 F bytes, in 16-byte chunks of eight fp16 values:
//   products over the columns:  hi, then mid: chunk (s, h, r) = row r, columns 16 s + 8 h ...    (F / 16 values of s)
//   products over the rows:     hi, then mid: chunk (t, s, h, c) = column 32 t + c, rows 16 s + {4 h .. 4 h + 3, 8 + 4 h ..}
// A wavefront's operand is 64 chunks in a row, whichever product; the rows of the second kind come in the order in
// which a lane holds the logits of the first.
template <int F>
struct DistillTile {
    static constexpr int KS = F / 16;          // steps of a product over the columns
    static constexpr int NT = F / 32;          // tiles of columns
    static constexpr int PLANE = 64 * F;       // bytes of one plane, either kind
    static constexpr int BYTES = 256 * F;
    // tiles in LDS at once: a narrow tile's work (0.6 us at F = 64) is shorter than the way of the next one from L2
    static constexpr int STAGES_FORWARD = F <= 96 ? 4 : 3, STAGES_BACKWARD = F <= 96 ? 4 : F <= 128 ? 3 : 2;
};

// Workspace of a call pair (host side): what mirec_distill_loss leaves for mirec_distill_grad, and scratch.
struct DistillWorkspace {
    size_t max_off, ref_off, mass_off, a_off, count_off, id_off, val_off, start_off, place_off, gval_off, row_off, base_off;
    size_t ximg_off, yimg_off, pref_off, pmass_off, part_off, bytes;
    int64_t xtiles, ytiles;
    int splits_x;      // ranges that Y is cut into in the forward pass
    int64_t runs;      // workgroups of the backward pass
};

// Into how many ranges to cut the streamed tiles: the fewest rounds of workgroups, each paying for its start (four
// tiles' time) and for the partial results (written and read once more: 0.025 of a tile's time per owned block).
static int distill_splits(int64_t blocks, int64_t tiles, int64_t places) {
    int best = 1;
    double cost = 1e300;
    for (int64_t s = 1; s <= DI_RANGES && s <= tiles; ++s) {
        const double rounds = (double)((blocks * s + places - 1) / places);
        const double c = rounds * ((double)((tiles + s - 1) / s) + 4.0) + (s > 1 ? 0.025 * (double)(blocks * s) : 0.0);
        if (c < cost) {
            cost = c;
            best = (int)s;
        }
    }
    return best;
}

static DistillWorkspace distill_layout(int64_t n, int64_t m, int f, int k) {
    DistillWorkspace w;
    size_t at = 0;
    auto take = [&](size_t b) {
        const size_t o = at;
        at += align_up(b, 256);
        return o;
    };
    w.xtiles = (n + 31) / 32;
    w.ytiles = (m + 31) / 32;
    const int64_t xblocks = (n + DI_OWN - 1) / DI_OWN, yblocks = (m + DI_OWN - 1) / DI_OWN;
    // workgroups of the two passes that run at once (2000 x 20000 at 32 columns: backward 43 us with one on a compute unit, 35 with
    // two; at 64 columns two gain nothing)
    const int64_t places = f <= 32 ? 2 * DI_CUS : DI_CUS;
    w.splits_x = distill_splits(xblocks, w.ytiles, places);
    // Cut the blocks of items where that saves more steps than the join of their parts costs.  (256 rows of 7207 items at 96
    // columns, 8 row tiles and 29 blocks: 56 us cut, 64 whole; 128 of 27000 at 128 columns, 4 and 106: 84 and 71; 512 of 60000, 16
    // and 235: 170 and 154.)
    const int64_t steps = yblocks * w.xtiles, whole = (yblocks + places - 1) / places * w.xtiles;
    w.runs = whole <= (steps + places - 1) / places + DI_JOIN_STEPS ? yblocks : steps < places ? steps : places;
    w.max_off = take(3 * DI_PARTS * 4);       // partial maxima of |X|, |Y|, |grad|
    w.ref_off = take((size_t)n * 4);          // M_b: log2 reference of a row's mass
    w.mass_off = take((size_t)n * 4);         // sum_j 2^(z_bj log2 e - M_b), over all items or those off the list
    w.a_off = take((size_t)n * 4);            // what the mean counts for: 1, or q_r - p_r
    w.count_off = take((size_t)n * 4);        // entries of the merged list
    w.id_off = take((size_t)n * k * 4);       // merged list
    w.val_off = take((size_t)n * k * 4);      // q - p of those
    // the same by (row tile, item tile): where a group begins, the entries' places in their 32 x 32 block, q - p (before that,
    // with teacher_lse: the lists' entries for the forward pass, in place of q - p)
    w.start_off = take((size_t)w.xtiles * (w.ytiles + 1) * 2);
    w.place_off = take((size_t)n * k * 2);
    w.gval_off = take((size_t)n * k * 4);
    w.row_off = take((size_t)w.xtiles * 32 * 16);   // what a row brings to the backward pass
    w.base_off = take((size_t)n * f * 4);     // dX_b / (grad_b T)
    w.ximg_off = take((size_t)w.xtiles * 256 * f);
    w.yimg_off = take((size_t)w.ytiles * 256 * f);
    w.pref_off = take((size_t)w.splits_x * n * 4);
    w.pmass_off = take((size_t)w.splits_x * n * 4);
    const size_t px = (size_t)w.splits_x * n * f * 4, py = w.runs == yblocks ? 0 : (size_t)w.runs * 2 * DI_OWN * f * 4;
    w.part_off = take(px > py ? px : py);     // partial means, later parts of dY
    w.bytes = at;
    return w;
}

// ------------------------------------------------------------------------------------------------ operand images

// Largest magnitude of two arrays, as DI_PARTS partial maxima of bit patterns each (a NaN's is above every number's).
__device__ __forceinline__ void di_absmax(int block, const float* __restrict__ a, int64_t na, const float* __restrict__ b, int64_t nb,
                                          uint32_t* __restrict__ parts) {
    __shared__ uint32_t part[DI_MAX_THREADS / 64];
    const float* v = block >= DI_PARTS ? b : a;
    const int64_t cnt = block >= DI_PARTS ? nb : na;
    uint32_t top = 0;
    constexpr int64_t step = (int64_t)DI_PARTS * DI_MAX_THREADS * 4;
    // (the widths are multiples of 32: no tail; a thread past the end reads its first value again)
    for (int64_t e = ((int64_t)(block % DI_PARTS) * DI_MAX_THREADS + threadIdx.x) * 4; e < cnt; e += 4 * step) {
        f32x4 q[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) q[u] = *reinterpret_cast<const f32x4*>(v + (e + u * step < cnt ? e + u * step : e));
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t b = __float_as_uint(q[u][i]) & 0x7fffffffu;
                top = b > top ? b : top;
            }
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)top, d, 64);
        top = o > top ? o : top;
    }
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < DI_MAX_THREADS / 64; ++w) top = part[w] > top ? part[w] : top;
        parts[block] = top;
    }
}

// Exponent of the power of two that puts the largest magnitude (a bit pattern) into [2^14, 2^15), within 2^+-100 (2^0
// where there is none, or it is not finite).
__device__ __forceinline__ int di_exponent_of(uint32_t top) {
    const int e = (int)(top >> 23);   // |v| in [2^(e - 127), 2^(e - 126))
    if (top == 0 || e == 255) return 0;
    const int s = 14 + 127 - e;
    return s > 100 ? 100 : (s < -100 ? -100 : s);
}

// The same from partial maxima, by a whole wavefront.
__device__ __forceinline__ int di_scale_exponent(const uint32_t* __restrict__ parts) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < DI_PARTS / 64; ++i) {
        const uint32_t u = parts[(threadIdx.x & 63) + 64 * i];
        top = u > top ? u : top;
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)top, d, 64);
        top = o > top ? o : top;
    }
    return di_exponent_of(top);
}

// What takes a product of the scaled factors to the logit it stands for, in octaves.  It does not vanish, so that minus infinity
// stays what it is: 2^-126 times the largest scaled logit (192 2^30) is nothing beside one, as the logit itself would be.
__device__ __forceinline__ float di_logit_factor(float step, int exponent) { return fmaxf(ldexpf(step, -exponent), FLT_MIN); }

// What an entry of a list must be to count.
__device__ __forceinline__ bool di_counts(int32_t id, float score, int64_t m) { return id >= 0 && id < m && score > -FLT_MAX; }

__device__ __forceinline__ uint32_t di_pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
}

// (a, b) -> packed pairs hi, mid; both roundings to nearest, the remainder is exact (one instruction for the widening of hi
// and the difference).
__device__ __forceinline__ void di_split(float a, float b, uint32_t& hi, uint32_t& mid) {
    hi = di_pack(a, b);
    float ra, rb;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[0,0,0] op_sel_hi:[1,0,0]" : "=v"(ra) : "v"(hi), "v"(a));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(rb) : "v"(hi), "v"(b));
    mid = di_pack(ra, rb);
}

// One workgroup per tile of 32 rows: their lists' entries grouped by item tile, and where every item tile's group begins.
// A group's order does not matter: its entries are places of one 32 x 32 block.  Item tiles are counted in LDS, DI_BINS at a
// time.  MERGED: lists as distill_list_kernel leaves them, `count` entries a row, written as place (row in the tile, column in the
// item tile) and value (q - p); else the caller's lists, written to `word` for distill_forward_kernel.
static_assert(((int64_t)1 << 26) / 32 < (1 << 22) - 1, "an item tile fits 22 bits, below the mark of no entry");
template <bool MERGED>
__device__ __forceinline__ void di_group(int64_t tile, const int32_t* __restrict__ count, const int32_t* __restrict__ list_id,
                                         const float* __restrict__ list_val, int64_t n, int64_t m, int k, int64_t ytiles,
                                         uint16_t* __restrict__ start, uint16_t* __restrict__ place, float* __restrict__ val,
                                         uint32_t* __restrict__ word) {
    __shared__ int32_t bins[DI_BINS];
    __shared__ int32_t part[DI_PREPARE_THREADS / 64];
    constexpr int PER = DI_BINS / DI_PREPARE_THREADS;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row0 = tile * 32;
    const int rows = (int)(n - row0 < 32 ? n - row0 : 32);
    uint16_t* tile_start = start + tile * (ytiles + 1);
    // this thread's entries: item tile (-1: not an entry), place in the 32 x 32 block, value
    constexpr int HELD = 32 * DI_LIST / DI_PREPARE_THREADS;
    int32_t in[HELD], spot[HELD];
    float v[HELD];
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int e = tid + i * DI_PREPARE_THREADS;
        in[i] = -1;
        if (e < rows * k) {
            const int r = e / k;
            const int32_t id = list_id[row0 * k + e];
            v[i] = list_val[row0 * k + e];
            spot[i] = r * 32 + (id & 31);
            const bool entry = MERGED ? e - r * k < count[row0 + r] : di_counts(id, v[i], m);
            in[i] = entry ? id >> 5 : -1;
        }
    }
    int base = 0;
    for (int64_t t0 = 0; t0 < ytiles; t0 += DI_BINS) {
        for (int i = tid; i < DI_BINS; i += DI_PREPARE_THREADS) bins[i] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int64_t t = in[i] - t0;
            if (in[i] >= 0 && t >= 0 && t < DI_BINS) atomicAdd(&bins[t], 1);
        }
        __syncthreads();
        int sum = 0;
        for (int i = 0; i < PER; ++i) sum += bins[tid * PER + i];
        int inc = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(inc, d, 64);
            inc += lane >= d ? o : 0;
        }
        if (lane == 63) part[wave] = inc;
        __syncthreads();
        int at = base + inc - sum;
        for (int w = 0; w < DI_PREPARE_THREADS / 64; ++w) {
            at += w < wave ? part[w] : 0;
            base += part[w];
        }
        for (int i = 0; i < PER; ++i) {
            const int c = bins[tid * PER + i];
            bins[tid * PER + i] = at;
            if (t0 + tid * PER + i < ytiles) tile_start[t0 + tid * PER + i] = (uint16_t)at;
            at += c;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < HELD; ++i) {
            const int64_t t = in[i] - t0;
            if (in[i] >= 0 && t >= 0 && t < DI_BINS) {
                const int64_t to = row0 * k + atomicAdd(&bins[t], 1);
                if (MERGED) {
                    place[to] = (uint16_t)spot[i];
                    val[to] = v[i];
                } else {
                    word[to] = (uint32_t)in[i] << 10 | (uint32_t)spot[i];
                }
            }
        }
        __syncthreads();
    }
    if (tid == 0) tile_start[ytiles] = (uint16_t)base;
}

// What the images and the forward pass wait for: workgroups 0 .. 2 DI_PARTS - 1 find the largest magnitudes, the others (only
// with teacher_lse) group the lists.
__global__ __launch_bounds__(DI_MAX_THREADS) void distill_scan_kernel(
    const float* __restrict__ X, const float* __restrict__ Y, int f, uint32_t* __restrict__ parts, const int32_t* __restrict__ ids,
    const float* __restrict__ scores, int64_t n, int64_t m, int k, int64_t ytiles, uint16_t* __restrict__ start,
    uint32_t* __restrict__ word) {
    if (blockIdx.x < 2 * DI_PARTS)
        di_absmax((int)blockIdx.x, X, n * f, Y, m * f, parts);
    else
        di_group<false>((int64_t)blockIdx.x - 2 * DI_PARTS, nullptr, ids, scores, n, m, k, ytiles, start, nullptr, nullptr, word);
}

// One workgroup per tile: tiles of X first, then tiles of Y.  Rows behind the last are zero.
template <int F>
__global__ __launch_bounds__(DI_THREADS) void distill_image_kernel(const float* __restrict__ X, int64_t n, int64_t xtiles,
                                                                   char* __restrict__ ximg, const float* __restrict__ Y,
                                                                   int64_t m, char* __restrict__ yimg,
                                                                   const uint32_t* __restrict__ parts) {
    typedef DistillTile<F> D;
    constexpr int LD = F + 4;
    __shared__ __attribute__((aligned(16))) float v[32 * LD];
    const bool is_y = (int64_t)blockIdx.x >= xtiles;
    const int64_t tile = is_y ? blockIdx.x - xtiles : blockIdx.x;
    const float* src = is_y ? Y : X;
    const int64_t rows = is_y ? m : n;
    char* dst = (is_y ? yimg : ximg) + tile * D::BYTES;
    const float scale = ldexpf(1.f, di_scale_exponent(parts + (is_y ? DI_PARTS : 0)));
    for (int e = threadIdx.x; e < 32 * F / 4; e += DI_THREADS) {
        const int r = e / (F / 4), c = e % (F / 4) * 4;
        const int64_t row = tile * 32 + r;
        f32x4 q = {0.f, 0.f, 0.f, 0.f};
        if (row < rows) q = *reinterpret_cast<const f32x4*>(src + row * F + c);
        *reinterpret_cast<f32x4*>(v + r * LD + c) = q * scale;
    }
    __syncthreads();
    for (int e = threadIdx.x; e < 4 * F; e += DI_THREADS) {   // chunks of a plane, over the columns
        const int r = e & 31, h = (e >> 5) & 1, s = e >> 6;
        const float* p = v + r * LD + 16 * s + 8 * h;
        u32x4 hi, mid;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t a, b;
            di_split(p[2 * i], p[2 * i + 1], a, b);
            hi[i] = a;
            mid[i] = b;
        }
        reinterpret_cast<u32x4*>(dst)[e] = hi;
        reinterpret_cast<u32x4*>(dst + D::PLANE)[e] = mid;
    }
    for (int e = threadIdx.x; e < 4 * F; e += DI_THREADS) {   // over the rows
        const int c = e & 31, h = (e >> 5) & 1, s = (e >> 6) & 1, t = e >> 7;
        const float* p = v + (16 * s + 4 * h) * LD + 32 * t + c;
        u32x4 hi, mid;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 2 * i < 4 ? 2 * i : 2 * i + 4;
            uint32_t a, b;
            di_split(p[r * LD], p[(r + 1) * LD], a, b);
            hi[i] = a;
            mid[i] = b;
        }
        reinterpret_cast<u32x4*>(dst + 2 * D::PLANE)[e] = hi;
        reinterpret_cast<u32x4*>(dst + 3 * D::PLANE)[e] = mid;
    }
}

// ------------------------------------------------------------------------------------------------------ the passes

// Queue the copy of BYTES (a multiple of 4 KiB) of a tile's image into LDS: 1 KiB per wavefront and instruction.
template <int BYTES>
__device__ __forceinline__ void di_fetch(const char* __restrict__ src, char* lds) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < (BYTES / 1024 + DI_NW - 1) / DI_NW; ++i) {
        const int o = (i * DI_NW + wave) * 1024;
        if ((i + 1) * DI_NW * 1024 <= BYTES || o < BYTES)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + o + lane * 16),
                                             (__attribute__((address_space(3))) void*)(lds + o), 16, 0, 0);
    }
}

// Wait for a tile whose copy was queued TILES copies (of at least PER instructions a wavefront) before the newest; copies
// return in order, and whatever else was asked for in between only makes the wait stricter.
template <int TILES, int PER>
__device__ __forceinline__ void di_wait(bool more) {
    if (more) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(TILES * PER) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

__device__ __forceinline__ f32x16 di_mma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The owned rows' operand: 32 rows of an image, both planes.
template <int F>
__device__ __forceinline__ void di_load_own(const char* __restrict__ img, u32x4 (&own)[2][F / 16]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int s = 0; s < F / 16; ++s)
            own[p][s] = reinterpret_cast<const u32x4*>(img + p * DistillTile<F>::PLANE)[s * 64 + lane];
}

// 32 x 32 scaled logits: streamed rows x owned rows.
template <int F>
__device__ __forceinline__ f32x16 di_logits(const char* tile, const u32x4 (&own)[2][F / 16]) {
    const int lane = threadIdx.x & 63;
    f32x16 z = {};
#pragma unroll
    for (int s = 0; s < F / 16; ++s) {
        const u32x4 hi = reinterpret_cast<const u32x4*>(tile)[s * 64 + lane];
        const u32x4 mid = reinterpret_cast<const u32x4*>(tile + DistillTile<F>::PLANE)[s * 64 + lane];
        z = di_mma(mid, own[0][s], z);
        z = di_mma(hi, own[1][s], z);
        z = di_mma(hi, own[0][s], z);
    }
    return z;
}

// acc[t] += columns 32 t .. of the streamed rows, weighted by w (32 streamed rows x 32 owned rows, in the accumulator
// order of di_logits).
template <int F>
__device__ __forceinline__ void di_accumulate(const char* tile, const f32x16& w, f32x16 (&acc)[F / 32]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        u32x4 whi, wmid;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t a, b;
            di_split(w[8 * s + 2 * i], w[8 * s + 2 * i + 1], a, b);
            whi[i] = a;
            wmid[i] = b;
        }
#pragma unroll
        for (int t = 0; t < F / 32; ++t) {
            const u32x4 hi = reinterpret_cast<const u32x4*>(tile + 2 * DistillTile<F>::PLANE)[(2 * t + s) * 64 + lane];
            const u32x4 mid = reinterpret_cast<const u32x4*>(tile + 3 * DistillTile<F>::PLANE)[(2 * t + s) * 64 + lane];
            acc[t] = di_mma(mid, whi, acc[t]);
            acc[t] = di_mma(hi, wmid, acc[t]);
            acc[t] = di_mma(hi, whi, acc[t]);
        }
    }
}

// Workgroup index -> (owned block, range of the streamed side): the workgroups of an XCD (every eighth index) take
// neighbouring work, range by range, so that what streams through an XCD's L2 is shared by its compute units.
__device__ __forceinline__ uint32_t di_work_index() {
    const uint32_t total = gridDim.x, per = total / 8, i = blockIdx.x;
    return i < per * 8 ? (i % 8) * per + i / 8 : i;
}

// Rows [32 w, 32 w + 32) of the block per wavefront against a range of item tiles: reference, mass and (GRAD) the
// weighted sum of the items, per row and range.  REST: of the items that are not on the row's list (a reference of minus
// infinity where that leaves none).  `listed` holds a row tile's entries by ascending item tile, (item tile, row, column)
// in 22, 5 and 5 bits; a wavefront holds 64 of them at a time, one per lane, and sets a bit for each that falls into the
// current tile in the word of the lane that holds its logit.
template <int F, bool GRAD, bool REST>
__global__ __launch_bounds__(64 * DI_NW) void distill_forward_kernel(
    const char* __restrict__ ximg, int64_t n, int64_t blocks, const char* __restrict__ yimg, int64_t m, int64_t ytiles,
    int64_t tiles_per_range, float step, const uint32_t* __restrict__ parts, int k, const uint16_t* __restrict__ start,
    const uint32_t* __restrict__ listed, float* __restrict__ pref, float* __restrict__ pmass, float* __restrict__ psum) {
    typedef DistillTile<F> D;
    constexpr int FETCH = GRAD ? D::BYTES : 2 * D::PLANE, STAGES = D::STAGES_FORWARD;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const uint32_t work = di_work_index();
    const int64_t range = work / (uint32_t)blocks, block = work % (uint32_t)blocks;
    const int64_t t0 = range * tiles_per_range;
    const int64_t t1 = t0 + tiles_per_range < ytiles ? t0 + tiles_per_range : ytiles;
    const int64_t own0 = block * DI_OWN + wave * 32;
    const bool active = own0 < n;
    const float c = di_logit_factor(step, di_scale_exponent(parts) + di_scale_exponent(parts + DI_PARTS));

    u32x4 own[2][F / 16];
    if (active) di_load_own<F>(ximg + (own0 / 32) * D::BYTES, own);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i)
        if (t0 + i < t1) di_fetch<FETCH>(yimg + (t0 + i) * D::BYTES, lds + i * FETCH);
    f32x16 acc[F / 32] = {};
    float ref = -INFINITY, mass = 0.f;
    uint32_t* out_bits = reinterpret_cast<uint32_t*>(lds + STAGES * FETCH) + wave * 64;
    const uint32_t* entry = listed;
    int entries = 0;                      // from `entry` on
    uint32_t held = ~0u, next = ~0u;      // these 64 and the 64 behind them (no entry: behind every tile)
    if (REST && active) {
        out_bits[lane] = 0;
        const uint16_t* at = start + own0 / 32 * (ytiles + 1);
        const int e0 = at[t0];
        entries = at[t1] - e0;
        entry += own0 * k + e0;
        if (lane < entries) held = entry[lane];
        if (lane + 64 < entries) next = entry[lane + 64];
    }
    int cur = 0;   // the buffer of the current tile
    for (int64_t t = t0; t < t1; ++t, cur = cur + 1 < STAGES ? cur + 1 : 0) {
        const char* tile = lds + cur * FETCH;
        di_wait<STAGES - 2, FETCH / (DI_NW * 1024)>(t + STAGES - 2 < t1);
        __syncthreads();   // this tile has arrived, and every wavefront is done with the one before it
        if (t + STAGES - 1 < t1) di_fetch<FETCH>(yimg + (t + STAGES - 1) * D::BYTES, lds + (cur > 0 ? cur - 1 : STAGES - 1) * FETCH);
        if (!active) continue;
        bool some = false;   // of this tile's items is on a list
        uint32_t bits = 0;   // which of this lane's
        if (REST) {
            for (;;) {
                const bool here = held >> 10 == (uint32_t)t;
                if (__any(here)) {
                    some = true;
                    const int r = held >> 5 & 31, c_of = held & 31;
                    if (here) atomicOr(&out_bits[r + 32 * ((c_of >> 2) & 1)], 1u << (4 * (c_of >> 3) + (c_of & 3)));
                }
                if ((uint32_t)__builtin_amdgcn_readlane((int)held, 63) >> 10 > (uint32_t)t) break;
                entry += 64;
                entries -= 64;
                held = next;
                next = lane + 64 < entries ? entry[lane + 64] : ~0u;
            }
            if (some) {
                asm volatile("" ::: "memory");   // written by other lanes of this wavefront, in order
                bits = out_bits[lane];
                out_bits[lane] = 0;
            }
        }
        f32x16 z = di_logits<F>(tile, own);
        if (REST && some) {
#pragma unroll
            for (int r = 0; r < 16; ++r) z[r] = (bits >> r) & 1u ? -INFINITY : z[r];
        }
        if (t == ytiles - 1 && (m & 31)) {   // rows behind the last item
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (t * 32 + 8 * (r / 4) + 4 * half + r % 4 >= m) z[r] = -INFINITY;
        }
        float top = z[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, z[r]);
        top = fmaxf(top, __shfl_xor(top, 32, 64)) * c;
        // a row's reference follows its maximum only when that has grown by more than 8: a probability is then below 2^15
        if (__ballot(top > ref + 8.f)) {
            const float now = fmaxf(ref, top);
            const float back = now == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ref - now);
            mass *= back;
            if (GRAD) {
#pragma unroll
                for (int u = 0; u < F / 32; ++u) acc[u] *= back;
            }
            ref = now;
        }
        const float off = REST && ref == -INFINITY ? 0.f : DI_HEADROOM - ref;   // (no item so far: all terms are zero)
#pragma unroll
        for (int r = 0; r < 16; ++r) z[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[r], c, off));
        float sum = 0.f;
#pragma unroll
        for (int r = 0; r < 16; r += 4) sum += (z[r] + z[r + 1]) + (z[r + 2] + z[r + 3]);
        mass += sum;
        if (GRAD) di_accumulate<F>(tile, z, acc);
    }
    mass += __shfl_xor(mass, 32, 64);
    const int64_t row = own0 + (lane & 31);
    if (!active || row >= n) return;
    if (half == 0) {
        pref[range * n + row] = ref;
        pmass[range * n + row] = mass;
    }
    if (GRAD) {
#pragma unroll
        for (int u = 0; u < F / 32; ++u)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 q = {acc[u][4 * g], acc[u][4 * g + 1], acc[u][4 * g + 2], acc[u][4 * g + 3]};
                *reinterpret_cast<f32x4*>(psum + (range * n + row) * F + 32 * u + 8 * g + 4 * half) = q;
            }
    }
}

// First of the steps that workgroup w of `runs` takes.
__device__ __forceinline__ int64_t di_quotient(int64_t a, int64_t b) {   // (a 64-bit division takes half a microsecond)
    return a < ((int64_t)1 << 32) ? (int64_t)((uint32_t)a / (uint32_t)b) : a / b;
}
__device__ __forceinline__ int64_t di_run_begin(int64_t w, int64_t steps, int64_t runs) { return di_quotient(w * steps, runs); }

// The gradients of the items: 32 of them per wavefront, 256 per workgroup, against all tiles of rows.  The steps (block of
// items, row tile) are numbered block by block and cut into equal runs, one per workgroup, whatever the number of
// blocks: 106 or 782 blocks are 0.4 and 3.05 rounds of 256 workgroups.  A workgroup writes a block that it
// sees whole to its place, and what it has of a block at an end of its run to a slot of its own, which
// distill_join_kernel adds up in the order of the rows.
template <int F>
__global__ __launch_bounds__(64 * DI_NW) void distill_backward_kernel(
    const char* __restrict__ yimg, int64_t m, int64_t steps, const char* __restrict__ ximg, int64_t n, int64_t xtiles,
    float step, float temperature, const uint32_t* __restrict__ parts, const float* __restrict__ row_const,
    const uint16_t* __restrict__ start, int64_t ytiles, const uint16_t* __restrict__ place, const float* __restrict__ gval,
    int k, float* __restrict__ dY, float* __restrict__ slots) {
    typedef DistillTile<F> D;
    constexpr int STAGES = D::STAGES_BACKWARD;
    extern __shared__ __attribute__((aligned(1024))) char lds[];   // tiles, what their rows bring, list entries on their way
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), half = lane >> 5;
    const int64_t run0 = di_run_begin(blockIdx.x, steps, gridDim.x), run1 = di_run_begin(blockIdx.x + 1, steps, gridDim.x);
    const int sx = di_scale_exponent(parts), sy = di_scale_exponent(parts + DI_PARTS);
    // the weights of the rows; |q - p| is at most 1, and so is |q_r - p_r| e / S: S sums the e off the list
    const int sg = di_scale_exponent(parts + 2 * DI_PARTS);
    const float c = di_logit_factor(step, sx + sy);

    const float back = ldexpf(temperature, -sx - sg);

    // a tile of rows and what its rows bring (zero behind the last row), into a buffer
    char* row_lds = lds + STAGES * D::BYTES;
    auto fetch_tile = [&](int64_t t, int buffer) {
        di_fetch<D::BYTES>(ximg + t * D::BYTES, lds + buffer * D::BYTES);
        if (wave == 0 && half == 0)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(row_const + t * 128 + lane * 4),
                                             (__attribute__((address_space(3))) void*)(row_lds + buffer * 512), 16, 0, 0);
    };
    int cur = 0;   // the buffer of the current step
    // The list entries that fall on this wavefront's items and a tile's rows.  Where they begin and end is asked for
    // two steps ahead, the first 64 of them (one per lane) one step ahead.
    struct Step {
        int block, t;
    };
    const int xt = (int)xtiles;
    auto after = [&](Step p) { return p.t + 1 < xt ? Step{p.block, p.t + 1} : Step{p.block + 1, 0}; };
    int e0 = 0, e1 = 0;
    auto fetch_extent = [&](Step p) {
        const int64_t jt = (int64_t)p.block * DI_NW + wave;
        e0 = e1 = 0;
        if (jt < ytiles) {
            const uint16_t* at = start + p.t * (ytiles + 1) + jt;
            e0 = at[0];
            e1 = at[1];
            // whatever the workspace holds, the tile's entries are not left
            const int64_t have = (n - p.t * 32 < 32 ? n - p.t * 32 : 32) * k;
            e1 = e1 < have ? e1 : (int)have;
        }
    };
    int entries = 0, spot = 0;
    float val = 0.f;
    int64_t list0 = 0;
    auto fetch_entries = [&](Step p) {
        entries = __builtin_amdgcn_readfirstlane(e1 - e0);
        list0 = (int64_t)p.t * 32 * k + __builtin_amdgcn_readfirstlane(e0);
        if (lane < entries) {
            spot = place[list0 + lane] & 1023;
            val = gval[list0 + lane];
        }
    };
    // Their values on the way to the lanes and registers that hold their places: 16 values per lane (rows of 20: 16-byte
    // reads of neighbouring lanes fall into distinct banks) and a bit for each that is there.
    float* fix = reinterpret_cast<float*>(lds + STAGES * (D::BYTES + 512)) + wave * (64 * 20 + 64);
    uint32_t* fix_bits = reinterpret_cast<uint32_t*>(fix + 64 * 20);
    fix_bits[lane] = 0;
    const int block0 = (int)di_quotient(run0, xtiles);
    Step now = {block0, (int)(run0 - block0 * xtiles)};
    fetch_extent(now);
    Step ahead = now;   // the next tile to copy
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
        if (run0 + i < run1) fetch_tile(ahead.t, i);
        ahead = after(ahead);
    }
    fetch_entries(now);
    Step next = after(now);
    fetch_extent(next);
    bool first = true;
    for (int64_t left = run1 - run0; left > 0;) {   // block by block
        const int t0 = now.t, t1 = left < xt - t0 ? t0 + (int)left : xt;
        const int64_t block = now.block;
        const int64_t own0 = block * DI_OWN + wave * 32;
        const bool active = own0 < m;
        u32x4 own[2][F / 16];
        if (active) di_load_own<F>(yimg + own0 / 32 * D::BYTES, own);
        f32x16 acc[F / 32] = {};
        for (int t = t0; t < t1; ++t, cur = cur + 1 < STAGES ? cur + 1 : 0) {
            const char* tile = lds + cur * D::BYTES;
            const float* rows = reinterpret_cast<const float*>(row_lds + cur * 512);
            di_wait<STAGES - 2, D::BYTES / (DI_NW * 1024)>(left > STAGES - 2);
            __syncthreads();
            const int have = entries;
            for (int done = 0; done < have; done += 64) {
                if (done > 0 && lane < have - done) {
                    spot = place[list0 + done + lane] & 1023;
                    val = gval[list0 + done + lane];
                }
                if (lane < have - done) {
                    const int r = spot >> 5, to = (spot & 31) + 32 * ((r >> 2) & 1), reg = 4 * (r >> 3) + (r & 3);
                    fix[to * 20 + reg] = val * rows[64 + r];
                    atomicOr(&fix_bits[to], 1u << reg);
                }
            }
            now = next;
            next = after(next);
            if (--left > 0) {
                fetch_entries(now);
                fetch_extent(next);   // (behind the run's last step: read, not used)
            }
            if (left > STAGES - 2) fetch_tile(ahead.t, cur > 0 ? cur - 1 : STAGES - 1);
            ahead = after(ahead);
            if (!active) continue;
            f32x16 z = di_logits<F>(tile, own);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x4 off = *reinterpret_cast<const f32x4*>(rows + 8 * g + 4 * half);
                const f32x4 w = *reinterpret_cast<const f32x4*>(rows + 32 + 8 * g + 4 * half);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    z[4 * g + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[4 * g + i], c, off[i])) * w[i];
            }
            // where an item is on a row's list its gradient is q - p (with the class, what stands there may have overflowed)
            if (have > 0) {
                asm volatile("" ::: "memory");   // written by other lanes of this wavefront, in order
                const uint32_t bits = fix_bits[lane];
                fix_bits[lane] = 0;
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 v = *reinterpret_cast<const f32x4*>(fix + lane * 20 + 4 * g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) z[4 * g + i] = (bits >> (4 * g + i)) & 1u ? v[i] : z[4 * g + i];
                }
            }
            di_accumulate<F>(tile, z, acc);
        }
        const int64_t item = own0 + (lane & 31);
        if (active && item < m) {
            // a part of a block goes to slot 0 where the run begins with it, else to slot 1
            const int64_t slot = 2 * (int64_t)blockIdx.x + (first ? 0 : 1);
            float* out = t0 == 0 && t1 == xt ? dY + item * F : slots + (slot * DI_OWN + wave * 32 + (lane & 31)) * F;
#pragma unroll
            for (int u = 0; u < F / 32; ++u)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const f32x4 q = {acc[u][4 * g] * back, acc[u][4 * g + 1] * back, acc[u][4 * g + 2] * back, acc[u][4 * g + 3] * back};
                    *reinterpret_cast<f32x4*>(out + 32 * u + 8 * g + 4 * half) = q;
                }
        }
        first = false;
    }
}

// The blocks that no workgroup saw whole: the sum of their parts, in the order of the rows.  One workgroup column per
// run; it takes the block that its run begins inside of, if no run before it does.
__global__ __launch_bounds__(DI_THREADS) void distill_join_kernel(const float* __restrict__ slots, int64_t steps, int64_t runs,
                                                                  int64_t xtiles, int64_t m, int f, float* __restrict__ dY) {
    const int64_t begin = di_run_begin(blockIdx.x + 1, steps, runs), block = di_quotient(begin, xtiles);
    const int64_t s0 = block * xtiles, s1 = s0 + xtiles;
    const int64_t w0 = blockIdx.x, before = di_run_begin(w0, steps, runs);   // the run that ends inside the block
    if (begin == s0 || before > s0) return;
    // one past the last run with a part of the block: the first whose steps begin behind it
    int64_t w1 = di_quotient(s1 * runs + steps - 1, steps);
    w1 = w1 < runs ? w1 : runs;
    const int first_slot = before == s0 ? 0 : 1;
    const int64_t rows = m - block * DI_OWN < DI_OWN ? m - block * DI_OWN : DI_OWN;
    const int64_t e = ((int64_t)blockIdx.y * DI_THREADS + threadIdx.x) * 4;   // (the grid covers a block)
    if (e >= rows * f) return;
    f32x4 v = *reinterpret_cast<const f32x4*>(slots + (2 * w0 + first_slot) * DI_OWN * f + e);
    for (int64_t w = w0 + 1; w < w1; w += 8) {   // eight parts asked for at once
        f32x4 part[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (w + u < w1) part[u] = *reinterpret_cast<const f32x4*>(slots + 2 * (w + u) * DI_OWN * f + e);
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (w + u < w1) v += part[u];
    }
    *reinterpret_cast<f32x4*>(dY + block * DI_OWN * f + e) = v;
}

// ------------------------------------------------------------------------------------------------------- the lists

// One workgroup per row: joins the row's partial results (REST: with teacher_lse, those of the items off the list); the list
// without its excluded entries, entries that name the same item merged (their probabilities add); the row's loss; its dX
// but for the weight.  Latency, not bandwidth, is what a row costs (a chain of a dozen dependent steps): factor rows are
// read by sixteen lanes each, four rows of a group of lanes in flight, and what does not depend on each other is asked for
// at once.  NT threads: 256 finish a row
// soonest, 64 (no barriers, sixteen rows in flight on a compute unit instead of four) more rows than run at once with 256
// (DI_MANY_ROWS: 1024 lists of 50 at 64 columns 12 and 16 us, 1500 of 200 at 192 columns 52 and 40).  4096 lists of 100 at 128
// columns with the class 45 us, of which the factor rows, 0.2 GB from L2, are a third.  REST: two sums of the list's items in
// registers, three wavefronts per SIMD from 96 columns on (four spill and gain nothing).
template <int F, int NT, bool REST>
__global__ __launch_bounds__(NT, NT == 64 && F <= 128 ? (REST && F > 64 ? 3 : 4) : 2) void distill_list_kernel(
    const float* __restrict__ X, int64_t n, const float* __restrict__ Y, int64_t m, const int32_t* __restrict__ ids,
    const float* __restrict__ scores, int k, float temperature, const float* __restrict__ teacher_lse, int ranges,
    const float* __restrict__ pref, const float* __restrict__ pmass, const float* __restrict__ psum,
    const uint32_t* __restrict__ parts, float* __restrict__ loss, float* __restrict__ ref_out, float* __restrict__ mass_out,
    float* __restrict__ a_out, int32_t* __restrict__ count_out, int32_t* __restrict__ id_out, float* __restrict__ val_out,
    float* __restrict__ base) {
    constexpr int PIECES = F / 32;     // 8-byte pieces of a factor row per lane
    constexpr int ROWS = NT / 16;      // factor rows that the workgroup reads side by side
    constexpr int NWV = NT / 64, PER = DI_LIST / NT;
    extern __shared__ __attribute__((aligned(16))) char list_lds[];
    const int kp = (k + 63) & ~63;
    uint64_t* key = reinterpret_cast<uint64_t*>(list_lds);          // item and place, where an item is listed twice
    int32_t* table = reinterpret_cast<int32_t*>(key);               // before that: the items, hashed
    float* mp = reinterpret_cast<float*>(key);                      // after that: p and log p of the merged entries
    float* mlogp = mp + kp;
    int32_t* sid = reinterpret_cast<int32_t*>(key + kp);            // by ascending item
    float* sp = reinterpret_cast<float*>(sid + kp);                 // p, then q
    int32_t* mid = reinterpret_cast<int32_t*>(sp + kp);             // merged
    float* mz = reinterpret_cast<float*>(mid + kp);                 // log p, then logits
    int slots = 2 * kp;                                             // of the table: a power of two
    while (slots & (slots - 1)) slots &= slots - 1;
    __shared__ float red[NWV][F];
    __shared__ float range_w[DI_RANGES];
    __shared__ float row_ref, row_mass;
    __shared__ double partd[2][NWV];
    __shared__ int parti[NWV];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, group = tid >> 4, sub = tid & 15;
    const double inv_t = 1.0 / (double)temperature;
    const int sy = di_scale_exponent(parts + DI_PARTS);
    auto block_max = [&](double v) {
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) v = fmax(v, __shfl_xor(v, d, 64));
        if (NWV == 1) return v;
        if (lane == 0) partd[0][wave] = v;
        __syncthreads();
        v = partd[0][0];
        for (int w = 1; w < NWV; ++w) v = fmax(v, partd[0][w]);
        __syncthreads();
        return v;
    };
    auto block_sum = [&](double v, int which) {
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
        if (NWV == 1) return v;
        if (lane == 0) partd[which][wave] = v;
        __syncthreads();
        v = partd[which][0];
        for (int w = 1; w < NWV; ++w) v += partd[which][w];
        __syncthreads();
        return v;
    };

    for (int64_t b = blockIdx.x; b < n; b += gridDim.x) {
        f32x2 x[PIECES];
#pragma unroll
        for (int i = 0; i < PIECES; ++i) x[i] = *reinterpret_cast<const f32x2*>(X + b * F + 2 * (sub + 16 * i));
        __syncthreads();   // the row before is done with the shared arrays
        if (wave == 0) {   // the ranges' references and masses, some of them to a lane
            float r[DI_RANGES / 64], pm[DI_RANGES / 64], top = -INFINITY, sum = 0.f;
#pragma unroll
            for (int i = 0; i < DI_RANGES / 64; ++i) {
                const int at = lane + 64 * i;
                r[i] = at < ranges ? pref[at * n + b] : -INFINITY;
                pm[i] = at < ranges ? pmass[at * n + b] : 0.f;
                top = fmaxf(top, r[i]);
            }
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
            if (REST && top == -INFINITY) top = 0.f;   // every item is on the list
#pragma unroll
            for (int i = 0; i < DI_RANGES / 64; ++i) {
                r[i] = lane + 64 * i < ranges ? __builtin_amdgcn_exp2f(r[i] - top) : 0.f;
                sum = __builtin_fmaf(pm[i], r[i], sum);
            }
            sum = wave_sum(sum);
#pragma unroll
            for (int i = 0; i < DI_RANGES / 64; ++i) range_w[lane + 64 * i] = REST && sum == 0.f ? 0.f : ldexpf(r[i] / sum, -sy);
            if (lane == 0) {
                row_ref = top;
                row_mass = ldexpf(sum, -(int)DI_HEADROOM);
                ref_out[b] = row_ref;
                mass_out[b] = REST && sum == 0.f ? 1.f : row_mass;
            }
        }
        // The entries that count, the best of them, and whether two name the same item (a hash table, open addressing: at
        // least a quarter of it stays empty).
        int32_t my_id[PER];   // entry tid + NT i; -1: left out
        float my_s[PER];
        float top = -INFINITY;
        int valid = 0;
        bool twice = false;
        for (int e = tid; e < slots; e += NT) table[e] = -1;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int e = tid + NT * i;
            my_id[i] = e < k ? ids[b * k + e] : -1;
            my_s[i] = e < k ? scores[b * k + e] : 0.f;
            if (!di_counts(my_id[i], my_s[i], m)) my_id[i] = -1;
            if (my_id[i] >= 0) top = fmaxf(top, my_s[i]);
            valid += my_id[i] >= 0 ? 1 : 0;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i)
            if (my_id[i] >= 0) {
                uint32_t at = ((uint32_t)my_id[i] * 2654435769u >> 16) & (uint32_t)(slots - 1);
                for (;;) {
                    const int32_t there = atomicCAS(&table[at], -1, my_id[i]);
                    twice = twice || there == my_id[i];
                    if (there == -1 || there == my_id[i]) break;
                    at = (at + 1) & (uint32_t)(slots - 1);
                }
            }
#pragma unroll
        for (int d = 32; d > 0; d >>= 1) {
            top = fmaxf(top, __shfl_xor(top, d, 64));
            valid += __shfl_xor(valid, d, 64);
        }
        int again = __any(twice) ? 1 : 0;
        if (NWV > 1) {
            if (lane == 0) {
                sp[wave] = top;
                parti[wave] = 2 * valid + again;
            }
            __syncthreads();
            top = sp[0];
            valid = parti[0] >> 1;
            again = parti[0] & 1;
            for (int w = 1; w < NWV; ++w) {
                top = fmaxf(top, sp[w]);
                valid += parti[w] >> 1;
                again |= parti[w] & 1;
            }
        }
        __syncthreads();
        if (valid == 0) {   // nothing to learn from this row
            if (tid == 0) {
                loss[b] = 0.f;
                a_out[b] = 0.f;
                count_out[b] = 0;
            }
            if (base)
                for (int c = tid; c < F; c += NT) base[b * F + c] = 0.f;
            continue;
        }
        // log sum exp of the student's logits (of those off the list, with the class) and of the teacher's
        const double log_rest = REST && row_mass == 0.f ? -INFINITY : (double)row_ref * 0.69314718055994531 + log((double)row_mass);
        double log_mass = log_rest, teacher = 0.0;
        if (REST) {
            teacher = (double)teacher_lse[b] - (double)top * inv_t;
        } else {
            double mass = 0.0;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (my_id[i] >= 0) mass += my_s[i] == top ? 1.0 : (double)expf((float)(((double)my_s[i] - (double)top) * inv_t));
            teacher = log(block_sum(mass, 0));
        }
        auto logp_of = [&](float s) -> float { return (float)((s == top ? 0.0 : ((double)s - (double)top) * inv_t) - teacher); };
        // where the chosen entries of this step go: behind `done`, in order
        auto place_of = [&](bool chosen, int& done) -> int {
            const uint64_t votes = __ballot(chosen);
            int at = done + __popcll(votes & ((1ull << lane) - 1));
            if (NWV > 1) {
                if (lane == 0) parti[wave] = __popcll(votes);
                __syncthreads();
                for (int w = 0; w < NWV; ++w) {
                    at += w < wave ? parti[w] : 0;
                    done += parti[w];
                }
                __syncthreads();
            } else {
                done += __popcll(votes);
            }
            return at;
        };
        int merged = 0;
        if (!again) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int at = place_of(my_id[i] >= 0, merged);
                if (my_id[i] >= 0) {
                    const float lp = logp_of(my_s[i]);
                    mid[at] = my_id[i];
                    mp[at] = expf(lp);
                    mlogp[at] = lp;
                }
            }
        } else {   // by ascending item; entries of one item become one
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (tid + NT * i < kp) key[tid + NT * i] = my_id[i] >= 0 ? ((uint64_t)my_id[i] << 8) | (uint64_t)(tid + NT * i) : ~0ull;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (my_id[i] < 0) continue;
                const uint64_t mine = key[tid + NT * i];
                int rank = 0;
                const ulonglong2* kv = reinterpret_cast<const ulonglong2*>(key);
#pragma unroll 8
                for (int j = 0; j < kp / 2; ++j) rank += (kv[j].x < mine ? 1 : 0) + (kv[j].y < mine ? 1 : 0);
                const float lp = logp_of(my_s[i]);
                sid[rank] = my_id[i];
                mz[rank] = lp;
                sp[rank] = expf(lp);
            }
            __syncthreads();
            for (int e0 = 0; e0 < valid; e0 += NT) {
                const int e = e0 + tid;
                const bool head = e < valid && (e == 0 || sid[e] != sid[e - 1]);
                const int at = place_of(head, merged);
                if (head) {
                    float p = sp[e], lp = mz[e];
                    int j = e + 1;
                    for (; j < valid && sid[j] == sid[e]; ++j) p += sp[j];
                    if (j > e + 1) lp = logf(p);
                    mid[at] = sid[e];
                    mp[at] = p;
                    mlogp[at] = lp;
                }
            }
        }
        __syncthreads();
        // f(e, whether it is an entry, this lane's pieces of the item's factors) for the entries of this group of lanes
        auto each_entry = [&](auto&& f) {
            for (int e0 = group; e0 - group < merged; e0 += 4 * ROWS) {
                f32x2 y[4][PIECES];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int e = e0 + u * ROWS;
                    const float* v = Y + (int64_t)mid[e < merged ? e : 0] * F + 2 * sub;
#pragma unroll
                    for (int i = 0; i < PIECES; ++i) y[u][i] = *reinterpret_cast<const f32x2*>(v + 32 * i);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u) f(e0 + u * ROWS, e0 + u * ROWS < merged, y[u]);
            }
        };
        auto logit = [&](const f32x2 (&y)[PIECES]) -> float {
            float z = 0.f;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                z = __builtin_fmaf(x[i][0], y[i][0], z);
                z = __builtin_fmaf(x[i][1], y[i][1], z);
            }
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) z += __shfl_xor(z, o, 64);
            return z;
        };
        f32x2 sum[PIECES] = {};   // of dX but for its weight: the list's part
        auto add = [&](f32x2 (&to)[PIECES], float w, const f32x2 (&y)[PIECES]) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) to[i][j] = __builtin_fmaf(w, y[i][j], to[i][j]);
        };
        // The student's logits and probabilities on the list, and the sum of the list's items: a factor row is read once.  Without
        // the class q is known from the mass of all items and is in their mean; with it a group of lanes holds its q relative
        // to the largest it has met, until all of them complete the log-sum-exp.
        if (!REST) {
            each_entry([&](int e, bool real, const f32x2 (&y)[PIECES]) {
                const float z = logit(y);
                const float q = expf((float)((double)z * inv_t - log_mass)), p = mp[real ? e : 0];
                if (real) {
                    if (sub == 0) {
                        mz[e] = z;
                        sp[e] = q;
                    }
                    if (base) add(sum, -p, y);
                }
            });
        } else {
            f32x2 sum_q[PIECES] = {};
            double group_top = -INFINITY, group_mass = 0.0;
            each_entry([&](int e, bool real, const f32x2 (&y)[PIECES]) {
                const float z = logit(y);
                const double t = (double)z * inv_t;
                const float p = mp[real ? e : 0];
                if (real) {
                    if (sub == 0) mz[e] = z;
                    if (t > group_top) {
                        const float back = expf((float)(group_top - t));
                        group_mass *= (double)back;
#pragma unroll
                        for (int i = 0; i < PIECES; ++i) sum_q[i] *= back;
                        group_top = t;
                    }
                    const float q = expf((float)(t - group_top));
                    group_mass += (double)q;
                    if (base) {
                        add(sum, -p, y);
                        add(sum_q, q, y);
                    }
                }
            });
            const double top_log = block_max(fmax(group_top, log_rest));
            const double list_mass = block_sum(sub == 0 ? group_mass * (double)expf((float)(group_top - top_log)) : 0.0, 1);
            log_mass = top_log + log(list_mass + exp(log_rest - top_log));
            const float scale = expf((float)(group_top - log_mass));
            add(sum, scale, sum_q);
            for (int e = tid; e < merged; e += NT) sp[e] = expf((float)((double)mz[e] * inv_t - log_mass));
        }
        __syncthreads();
        double kl = 0.0, sum_p = 0.0;
        for (int e = tid; e < merged; e += NT) {
            const double logq = (double)mz[e] * inv_t - log_mass;
            const float p = mp[e];
            if (!(p <= 0.f)) kl += (double)p * ((double)mlogp[e] - logq);   // (a NaN probability stays in the sum)
            sum_p += (double)p;
        }
        kl = block_sum(kl, 0);
        float a = 1.f;   // what the mean counts for
        if (REST) {
            const double pr = fmax(1.0 - block_sum(sum_p, 1), 0.0);
            const double log_qr = log_rest - log_mass, qr = exp(log_qr);   // bounded below by 2^-24 beside p_r
            if (pr > 0.0) kl += pr * (log(pr) - fmax(log_qr, -24.0 * 0.69314718055994531));
            a = (float)(qr - pr * fmin(qr * 0x1p24, 1.0));
        }
        if (tid == 0) {
            loss[b] = (float)((double)temperature * (double)temperature * kl);
            a_out[b] = a;
            count_out[b] = merged;
        }
        if (!base) continue;
        for (int e = tid; e < merged; e += NT) {
            id_out[b * k + e] = mid[e];
            val_out[b * k + e] = sp[e] - mp[e];
        }
        // and the ranges' part
        for (int r0 = group; r0 - group < ranges; r0 += 4 * ROWS) {
            f32x2 y[4][PIECES];
            float w[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int r = r0 + u * ROWS;
                w[u] = r < ranges ? a * range_w[r] : 0.f;
                const float* v = psum + ((r < ranges ? r : 0) * n + b) * F + 2 * sub;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) y[u][i] = *reinterpret_cast<const f32x2*>(v + 32 * i);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const bool real = r0 + u * ROWS < ranges;
#pragma unroll
                for (int i = 0; i < PIECES; ++i) {
                    sum[i][0] = real ? __builtin_fmaf(w[u], y[u][i][0], sum[i][0]) : sum[i][0];
                    sum[i][1] = real ? __builtin_fmaf(w[u], y[u][i][1], sum[i][1]) : sum[i][1];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < PIECES; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                float v = sum[i][j];
                v += __shfl_xor(v, 16, 64);
                v += __shfl_xor(v, 32, 64);
                if (lane < 16) red[wave][2 * (sub + 16 * i) + j] = v;
            }
        __syncthreads();
        for (int c = tid; c < F; c += NT) {
            float v = red[0][c];
            for (int w = 1; w < NWV; ++w) v += red[w][c];
            base[b * F + c] = v;
        }
    }
}

// dX; and per tile of rows what they bring to the backward pass, 32 numbers each: minus the reference of a row's logits,
// the weight of its probabilities, the weight of its list entries, the two scaled by the power of two that the largest
// |grad| asks for (every workgroup finds that for itself; `parts` gets it for the backward pass).
__device__ __forceinline__ void di_weigh(int block, const float* __restrict__ base, const float* __restrict__ grad,
                                         float temperature, int64_t n, int f, float* __restrict__ dX,
                                         const float* __restrict__ ref, const float* __restrict__ mass, const float* __restrict__ a,
                                         float* __restrict__ rows, uint32_t* __restrict__ parts) {
    __shared__ uint32_t part[DI_PREPARE_THREADS / 64];
    uint32_t top = 0;
    for (int64_t b0 = threadIdx.x; b0 < n; b0 += 8 * DI_PREPARE_THREADS) {
        uint32_t u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int64_t b = b0 + i * DI_PREPARE_THREADS;
            u[i] = b < n ? __float_as_uint(grad[b]) & 0x7fffffffu : 0u;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) top = u[i] > top ? u[i] : top;
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)top, d, 64);
        top = o > top ? o : top;
    }
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int w = 0; w < DI_PREPARE_THREADS / 64; ++w) top = part[w] > top ? part[w] : top;
    if (block == 0 && threadIdx.x < DI_PARTS) parts[threadIdx.x] = top;
    const int sg = di_exponent_of(top);
    const int64_t mine = (int64_t)block * DI_PREPARE_THREADS + threadIdx.x, stride = (int64_t)DI_WEIGH_BLOCKS * DI_PREPARE_THREADS;
    if (dX)
        for (int64_t e = mine * 4; e < n * f; e += stride * 4) {
            const float g = grad[e / f] * temperature;
            *reinterpret_cast<f32x4*>(dX + e) = *reinterpret_cast<const f32x4*>(base + e) * g;
        }
    for (int64_t b = mine; b < ((n + 31) & ~(int64_t)31); b += stride) {
        float* to = rows + b / 32 * 128 + b % 32;
        const float g = b < n ? ldexpf(grad[b], sg) : 0.f;
        to[0] = b < n ? -ref[b] : 0.f;
        to[32] = b < n ? g * (a[b] / mass[b]) : 0.f;
        to[64] = g;
        to[96] = 0.f;
    }
}

// What the gradients need beside the two passes: workgroups 0 .. DI_WEIGH_BLOCKS - 1 weigh the rows, the others group the
// lists (one launch: each alone leaves most of the chip idle).
__global__ __launch_bounds__(DI_PREPARE_THREADS) void distill_prepare_kernel(
    const float* __restrict__ base, const float* __restrict__ grad, float temperature, int64_t n, int f, float* __restrict__ dX,
    const float* __restrict__ ref, const float* __restrict__ mass, const float* __restrict__ a, float* __restrict__ rows,
    uint32_t* __restrict__ parts, const int32_t* __restrict__ count, const int32_t* __restrict__ list_id,
    const float* __restrict__ list_val, int64_t m, int k, int64_t ytiles, uint16_t* __restrict__ start, uint16_t* __restrict__ place,
    float* __restrict__ val) {
    if (blockIdx.x < DI_WEIGH_BLOCKS)
        di_weigh((int)blockIdx.x, base, grad, temperature, n, f, dX, ref, mass, a, rows, parts);
    else
        di_group<true>((int64_t)blockIdx.x - DI_WEIGH_BLOCKS, count, list_id, list_val, n, m, k, ytiles, start, place, val, nullptr);
}

__global__ __launch_bounds__(DI_THREADS) void distill_zero_kernel(float* __restrict__ out, int64_t cnt) {
    for (int64_t e = (int64_t)blockIdx.x * DI_THREADS + threadIdx.x; e < cnt; e += (int64_t)gridDim.x * DI_THREADS) out[e] = 0.f;
}

static int distill_check(const char* who, const float* X, int64_t n, const float* Y, int64_t m, int f, int k,
                         float temperature) {
    MIREC_REQUIRE(n >= 0 && m >= 0, MIREC_E_INVALID, "%s: negative size", who);
    MIREC_REQUIRE(f >= 32 && f <= 192 && f % 32 == 0, MIREC_E_UNSUPPORTED,
                  "%s: factor width %d is not one of 32,64,96,128,160,192; zero-pad the columns", who, f);
    MIREC_REQUIRE(k >= 1, MIREC_E_INVALID, "%s: lists need at least one entry (got %d)", who, k);
    MIREC_REQUIRE(k <= DI_LIST, MIREC_E_UNSUPPORTED, "%s: lists of %d entries exceed the supported maximum of %d", who, k,
                  DI_LIST);
    MIREC_REQUIRE(temperature >= 1e-6f && temperature <= 1e6f, MIREC_E_INVALID,
                  "%s: temperature must lie in [1e-6, 1e6] (got %g)", who, (double)temperature);
    // (a launch has less than 2^32 threads: 1024 per 32 rows)
    MIREC_REQUIRE(n <= ((int64_t)1 << 26) && m <= ((int64_t)1 << 26), MIREC_E_UNSUPPORTED, "%s: more than 2^26 rows or items",
                  who);
    MIREC_REQUIRE(n == 0 || m >= 1, MIREC_E_INVALID, "%s: the catalogue is empty", who);
    MIREC_REQUIRE(n == 0 || (X && Y), MIREC_E_INVALID, "%s: null argument", who);
    MIREC_REQUIRE((((uintptr_t)X | (uintptr_t)Y) & 15) == 0, MIREC_E_INVALID, "%s: X and Y must be 16-byte aligned", who);
    return MIREC_OK;
}

static int distill_check_ws(const char* who, const void* ws, size_t ws_bytes, size_t need) {
    MIREC_REQUIRE(ws != nullptr && ((uintptr_t)ws & 255) == 0 && ws_bytes >= need, MIREC_E_WORKSPACE,
                  "%s: workspace of %zu bytes needed (256-byte aligned), %zu given", who, need, ws_bytes);
    return MIREC_OK;
}

// Dynamic LDS of the two passes (two to four tiles) needs an attribute once per kernel and device.
static int distill_lds(const void* kernel, int bytes, OncePerDevice& once, const char* who) {
    bool* done = once.slot();
    MIREC_REQUIRE(done, MIREC_E_HIP, "%s: cannot read the current device", who);
    if (!*done) {   // idempotent; a race only repeats the call
        MIREC_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        *done = true;
    }
    return MIREC_OK;
}

template <int F, bool GRAD, bool REST>
static int launch_forward(const DistillWorkspace& L, char* w, const float* X, int64_t n, const float* Y, int64_t m,
                          const int32_t* ids, const float* scores, int k, float temperature, const float* teacher_lse,
                          float* loss, hipStream_t stream) {
    const float step = (float)(1.4426950408889634 / (double)temperature);
    static OncePerDevice once;
    constexpr int LDS = DistillTile<F>::STAGES_FORWARD * (GRAD ? DistillTile<F>::BYTES : 2 * DistillTile<F>::PLANE) +
                        (REST ? DI_NW * 64 * 4 : 0);
    if (const int rc = distill_lds((const void*)distill_forward_kernel<F, GRAD, REST>, LDS, once, "mirec_distill_loss")) return rc;
    uint32_t* parts = (uint32_t*)(w + L.max_off);
    hipLaunchKernelGGL((distill_image_kernel<F>), dim3((unsigned)(L.xtiles + L.ytiles)), dim3(DI_THREADS), 0, stream, X, n,
                       L.xtiles, w + L.ximg_off, Y, m, w + L.yimg_off, parts);
    MIREC_LAUNCH_CHECK();
    const int64_t blocks = (n + DI_OWN - 1) / DI_OWN, per = (L.ytiles + L.splits_x - 1) / L.splits_x;
    const int64_t ranges = (L.ytiles + per - 1) / per;
    hipLaunchKernelGGL((distill_forward_kernel<F, GRAD, REST>), dim3((unsigned)(blocks * ranges)), dim3(64 * DI_NW), LDS, stream,
                       w + L.ximg_off, n, blocks, w + L.yimg_off, m, L.ytiles, per, step, parts, k, (const uint16_t*)(w + L.start_off),
                       (const uint32_t*)(w + L.gval_off), (float*)(w + L.pref_off), (float*)(w + L.pmass_off),
                       (float*)(w + L.part_off));
    MIREC_LAUNCH_CHECK();
    const int nt = n > DI_MANY_ROWS ? 64 : 256;
    hipLaunchKernelGGL(nt == 64 ? (distill_list_kernel<F, 64, REST>) : (distill_list_kernel<F, 256, REST>),
                       dim3((unsigned)(n < 262144 ? n : 262144)), dim3(nt), (size_t)((k + 63) & ~63) * 24, stream, X, n, Y, m,
                       ids, scores, k, temperature, teacher_lse, (int)ranges, (const float*)(w + L.pref_off),
                       (const float*)(w + L.pmass_off), (const float*)(w + L.part_off), parts, loss, (float*)(w + L.ref_off),
                       (float*)(w + L.mass_off), (float*)(w + L.a_off), (int32_t*)(w + L.count_off), (int32_t*)(w + L.id_off),
                       (float*)(w + L.val_off), GRAD ? (float*)(w + L.base_off) : nullptr);
    MIREC_LAUNCH_CHECK();
    return MIREC_OK;
}

template <int F>
static int launch_forward(bool grad, const DistillWorkspace& L, char* w, const float* X, int64_t n, const float* Y, int64_t m,
                          const int32_t* ids, const float* scores, int k, float temperature, const float* teacher_lse,
                          float* loss, hipStream_t stream) {
    auto* launch = grad ? (teacher_lse ? launch_forward<F, true, true> : launch_forward<F, true, false>)
                        : (teacher_lse ? launch_forward<F, false, true> : launch_forward<F, false, false>);
    return launch(L, w, X, n, Y, m, ids, scores, k, temperature, teacher_lse, loss, stream);
}

template <int F>
static int launch_backward(const DistillWorkspace& L, char* w, int64_t n, int64_t m, int k, float step, float temperature,
                           float* dY, hipStream_t stream) {
    static OncePerDevice once;
    constexpr int LDS = DistillTile<F>::STAGES_BACKWARD * (DistillTile<F>::BYTES + 512) + DI_NW * (64 * 20 + 64) * 4;
    if (const int rc = distill_lds((const void*)distill_backward_kernel<F>, LDS, once, "mirec_distill_grad")) return rc;
    const int64_t blocks = (m + DI_OWN - 1) / DI_OWN, steps = blocks * L.xtiles;
    float* slots = (float*)(w + L.part_off);
    hipLaunchKernelGGL((distill_backward_kernel<F>), dim3((unsigned)L.runs), dim3(64 * DI_NW), LDS, stream, w + L.yimg_off, m,
                       steps, w + L.ximg_off, n, L.xtiles, step, temperature, (const uint32_t*)(w + L.max_off),
                       (const float*)(w + L.row_off), (const uint16_t*)(w + L.start_off), L.ytiles,
                       (const uint16_t*)(w + L.place_off), (const float*)(w + L.gval_off), k, dY, slots);
    MIREC_LAUNCH_CHECK();
    if (blocks % L.runs != 0) {   // (else every run is of whole blocks)
        const dim3 grid((unsigned)(L.runs - 1), DI_OWN * F / (4 * DI_THREADS));
        hipLaunchKernelGGL(distill_join_kernel, grid, dim3(DI_THREADS), 0, stream, slots, steps,
                           L.runs, L.xtiles, m, F, dY);
        MIREC_LAUNCH_CHECK();
    }
    return MIREC_OK;
}

}  // namespace mirec

#define MIREC_DISTILL_WIDTHS(CASE) CASE(32) CASE(64) CASE(96) CASE(128) CASE(160) CASE(192)

extern "C" size_t mirec_distill_workspace_bytes(int64_t n, int64_t m, int f, int k) {
    if (n <= 0 || m <= 0 || f < 1 || k < 1) return 0;
    return mirec::distill_layout(n, m, f, k).bytes;
}

extern "C" int mirec_distill_loss(const float* X, int64_t n, const float* Y, int64_t m, int f, const int32_t* ids,
                                  const float* scores, int k, float temperature, const float* teacher_lse, int with_grad,
                                  float* loss, void* ws, size_t ws_bytes, mirec_stream_t stream_) {
    using namespace mirec;
    hipStream_t stream = (hipStream_t)stream_;
    if (const int rc = distill_check("mirec_distill_loss", X, n, Y, m, f, k, temperature)) return rc;
    if (n == 0) return MIREC_OK;
    MIREC_REQUIRE(ids && scores && loss, MIREC_E_INVALID, "mirec_distill_loss: null argument");
    const DistillWorkspace L = distill_layout(n, m, f, k);
    if (const int rc = distill_check_ws("mirec_distill_loss", ws, ws_bytes, L.bytes)) return rc;
    char* w = (char*)ws;
    hipLaunchKernelGGL(distill_scan_kernel, dim3((unsigned)(2 * DI_PARTS + (teacher_lse ? L.xtiles : 0))), dim3(DI_MAX_THREADS), 0,
                       stream, X, Y, f, (uint32_t*)(w + L.max_off), ids, scores, n, m, k, L.ytiles, (uint16_t*)(w + L.start_off),
                       (uint32_t*)(w + L.gval_off));
    MIREC_LAUNCH_CHECK();
    switch (f) {
#define MIREC_DISTILL_CASE(FW)                                                                                          \
    case FW:                                                                                                            \
        return launch_forward<FW>(with_grad != 0, L, w, X, n, Y, m, ids, scores, k, temperature, teacher_lse, loss, stream);
        MIREC_DISTILL_WIDTHS(MIREC_DISTILL_CASE)
#undef MIREC_DISTILL_CASE
    }
    return MIREC_OK;
}

extern "C" int mirec_distill_grad(const float* X, int64_t n, const float* Y, int64_t m, int f, int k, float temperature,
                                  const float* grad, float* dX, float* dY, void* ws, size_t ws_bytes,
                                  mirec_stream_t stream_) {
    using namespace mirec;
    hipStream_t stream = (hipStream_t)stream_;
    if (const int rc = distill_check("mirec_distill_grad", X, n, Y, m, f, k, temperature)) return rc;
    MIREC_REQUIRE(n == 0 || grad, MIREC_E_INVALID, "mirec_distill_grad: null argument");
    MIREC_REQUIRE((((uintptr_t)dX | (uintptr_t)dY) & 15) == 0, MIREC_E_INVALID,
                  "mirec_distill_grad: dX and dY must be 16-byte aligned");
    if (n == 0) {   // a step without rows
        if (dY && m > 0) {
            hipLaunchKernelGGL(distill_zero_kernel, dim3(1024), dim3(DI_THREADS), 0, stream, dY, m * f);
            MIREC_LAUNCH_CHECK();
        }
        return MIREC_OK;
    }
    const DistillWorkspace L = distill_layout(n, m, f, k);
    if (const int rc = distill_check_ws("mirec_distill_grad", ws, ws_bytes, L.bytes)) return rc;
    char* w = (char*)ws;
    // (without dY the lists need no grouping)
    hipLaunchKernelGGL(distill_prepare_kernel, dim3((unsigned)(DI_WEIGH_BLOCKS + (dY ? L.xtiles : 0))), dim3(DI_PREPARE_THREADS), 0,
                       stream, (const float*)(w + L.base_off), grad, temperature, n, f, dX, (const float*)(w + L.ref_off),
                       (const float*)(w + L.mass_off), (const float*)(w + L.a_off), (float*)(w + L.row_off),
                       (uint32_t*)(w + L.max_off) + 2 * DI_PARTS, (const int32_t*)(w + L.count_off),
                       (const int32_t*)(w + L.id_off), (const float*)(w + L.val_off), m, k, L.ytiles, (uint16_t*)(w + L.start_off),
                       (uint16_t*)(w + L.place_off), (float*)(w + L.gval_off));
    MIREC_LAUNCH_CHECK();
    if (!dY) return MIREC_OK;
    const float step = (float)(1.4426950408889634 / (double)temperature);
    switch (f) {
#define MIREC_DISTILL_CASE(FW) \
    case FW:                   \
        return launch_backward<FW>(L, w, n, m, k, step, temperature, dY, stream);
        MIREC_DISTILL_WIDTHS(MIREC_DISTILL_CASE)
#undef MIREC_DISTILL_CASE
    }
    return MIREC_OK;
}
