// Distilling a factor model from a teacher's ranked lists: per row the Kullback-Leibler divergence of the student's
// softmax over the whole catalogue from the teacher's distribution on its list, and its gradients, from the factor
// matrices -- as in the top-K pass the matrix of scores is never written.  The teacher's side is what the reference
// serves for a user (recommenders/als_recommender.py:181-186): ids and scores, best first.
//
//   z_bj = x_b . y_j / T,  q_b = softmax(z_b) over all m items,  p_b = softmax(t_b / T) over the list (or
//   exp(t / T - lse) with the teacher's log-sum-exp given: what the list leaves, p_r = 1 - sum p, is one class more,
//   which the student gives q_r = 1 - sum over the list of q)
//   loss_b = T^2 [ sum_list p (log p - log q) + p_r (log p_r - log q_r) ]
//   d loss_b / d (x_b . y_j) = T (q_j - p_j) on the list, T A_b q_j elsewhere, A_b = 1 - p_r / q_r (1 without the class)
//
// so with mean_b = sum_j q_bj y_j
//   dX_b = grad_b T [ A_b mean_b + sum_list ((1 - A_b) q_k - p_k) y_k ],   dY_j = sum_b grad_b T g_bj x_b,
//   g_bj = A_b q_bj, or q_k - p_k where j is on row b's list.
//
// The two passes over the n x m logits have one form: a wavefront owns 32 rows of one side (in registers), the other
// side streams through LDS in tiles of 32 rows, a tile's 32 x 32 logits come off the matrix cores with the owned rows
// as columns, so that a lane holds 16 logits of ONE owned row, become probabilities in registers and go straight back
// into the matrix cores as the operand that weights the streamed rows: the streamed side's image is laid out for that
// (below) and no logit passes through LDS or memory.
//   distill_forward_kernel   owns rows of X, streams Y: running maximum, mass and mean of the items (dX's dense part)
//   distill_backward_kernel  owns rows of Y, streams X: dY; the logits are formed a second time (three of twelve
//                            matrix products) because keeping them would write and read n m of them
//
// fp32 on the fp16 matrix cores: an operand is two fp16 planes, hi = fp16(v), mid = fp16(v - hi), of the value scaled
// by a power of two that puts its matrix's largest entry just below 2^15, and a product is hi hi + hi mid + mid hi in
// fp32 (mid mid is below 2^-24 of it).  Entries within 2^-18 of the largest keep 22 bits or more, smaller ones an
// absolute error of 2^-40 of the largest, which is what a sum with the large ones leaves of them anyway.
#include <float.h>

#include "common.h"

namespace mirec {

constexpr int DI_LIST = MIREC_DISTILL_MAX_LIST;   // longest list; one thread per entry in distill_list_kernel
constexpr int DI_THREADS = 256;
constexpr int DI_NW = 8;                          // wavefronts of a workgroup of the two passes
constexpr int DI_OWN = 32 * DI_NW;                // rows it owns
constexpr int DI_PARTS = 256;                     // partial maxima of a matrix
constexpr int DI_CUS = 256;                       // workgroups that run at once
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
};

// Workspace of a call pair (host side): what mirec_distill_loss leaves for mirec_distill_grad, and scratch.
struct DistillWorkspace {
    size_t max_off, ref_off, mass_off, a_off, count_off, id_off, val_off, start_off, base_off, ximg_off, yimg_off, pref_off,
        pmass_off, part_off, bytes;
    int64_t xtiles, ytiles;
    int splits_x, splits_y;   // ranges the streamed side is cut into: of Y in the forward pass, of X in the backward
};

// Into how many ranges to cut the streamed tiles: the fewest rounds of 256 workgroups, each paying for its start (four
// tiles' time) and for the partial results (written and read once more: 0.05 of a tile's time per owned block).
static int distill_splits(int64_t blocks, int64_t tiles) {
    int best = 1;
    double cost = 1e300;
    for (int64_t s = 1; s <= 64 && s <= tiles; ++s) {
        const double rounds = (double)((blocks * s + DI_CUS - 1) / DI_CUS);
        const double c = rounds * ((double)((tiles + s - 1) / s) + 4.0) + (s > 1 ? 0.05 * (double)(blocks * s) : 0.0);
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
    w.splits_x = distill_splits(xblocks, w.ytiles);
    w.splits_y = distill_splits(yblocks, w.xtiles);
    w.max_off = take(3 * DI_PARTS * 4);       // partial maxima of |X|, |Y|, |grad|
    w.ref_off = take((size_t)n * 4);          // M_b: log2 reference of a row's mass
    w.mass_off = take((size_t)n * 4);         // sum_j 2^(z_bj log2 e - M_b)
    w.a_off = take((size_t)n * 4);            // A_b
    w.count_off = take((size_t)n * 4);        // entries of the merged list
    w.id_off = take((size_t)n * k * 4);       // merged list, ascending ids
    w.val_off = take((size_t)n * k * 4);      // q - p of those
    w.start_off = take((size_t)n * (w.ytiles + 1) * 2);   // where the entries of an item tile begin in the list
    w.base_off = take((size_t)n * f * 4);     // dX_b / (grad_b T)
    w.ximg_off = take((size_t)w.xtiles * 256 * f);
    w.yimg_off = take((size_t)w.ytiles * 256 * f);
    w.pref_off = take((size_t)w.splits_x * n * 4);
    w.pmass_off = take((size_t)w.splits_x * n * 4);
    const size_t px = (size_t)w.splits_x * n * f * 4, py = w.splits_y > 1 ? (size_t)w.splits_y * m * f * 4 : 0;
    w.part_off = take(px > py ? px : py);     // partial means, later partial dY
    w.bytes = at;
    return w;
}

__device__ __forceinline__ float di_block_max(float v, float* part) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int w = 0; w < DI_THREADS / 64; ++w) v = fmaxf(v, part[w]);
    return v;
}

__device__ __forceinline__ double di_block_sum(double v, double* part) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int w = 0; w < DI_THREADS / 64; ++w) v += part[w];
    return v;
}

// ------------------------------------------------------------------------------------------------ operand images

// Largest magnitude of up to two arrays (blockIdx.y), as DI_PARTS partial maxima of bit patterns each (a NaN's is
// above every number's).
__global__ __launch_bounds__(DI_THREADS) void distill_absmax_kernel(const float* __restrict__ a, int64_t na,
                                                                    const float* __restrict__ b, int64_t nb,
                                                                    uint32_t* __restrict__ parts) {
    __shared__ uint32_t part[DI_THREADS / 64];
    const float* v = blockIdx.y ? b : a;
    const int64_t cnt = blockIdx.y ? nb : na;
    uint32_t top = 0;
    for (int64_t e = ((int64_t)blockIdx.x * DI_THREADS + threadIdx.x) * 4; e < cnt; e += (int64_t)DI_PARTS * DI_THREADS * 4) {
        const f32x4 q = *reinterpret_cast<const f32x4*>(v + e);   // the widths are multiples of 32: no tail
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t u = __float_as_uint(q[i]) & 0x7fffffffu;
            top = u > top ? u : top;
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
        for (int w = 1; w < DI_THREADS / 64; ++w) top = part[w] > top ? part[w] : top;
        parts[blockIdx.y * DI_PARTS + blockIdx.x] = top;
    }
}

// Power of two that puts the largest magnitude into [2^14, 2^15), within 2^+-100 (1 where there is none, or it is not
// finite).  Called by a whole wavefront.
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
    const int e = (int)(top >> 23);   // |v| in [2^(e - 127), 2^(e - 126))
    if (top == 0 || e == 255) return 0;
    const int s = 14 + 127 - e;
    return s > 100 ? 100 : (s < -100 ? -100 : s);
}

__device__ __forceinline__ uint32_t di_pack(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{a, b}), f16x2));
}

// (a, b) -> packed pairs hi, mid; both roundings to nearest, the remainder is exact.
__device__ __forceinline__ void di_split(float a, float b, uint32_t& hi, uint32_t& mid) {
    hi = di_pack(a, b);
    const f16x2 h = __builtin_bit_cast(f16x2, hi);
    mid = di_pack(a - (float)h[0], b - (float)h[1]);
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

// Queue the copy of `bytes` (a multiple of 8 KiB) of a tile's image into LDS: 1 KiB per wavefront and instruction.
__device__ __forceinline__ void di_fetch(const char* __restrict__ src, char* lds, int bytes) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int o = wave * 1024; o < bytes; o += DI_NW * 1024)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + o + lane * 16),
                                         (__attribute__((address_space(3))) void*)(lds + o), 16, 0, 0);
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
__device__ __forceinline__ int64_t di_work_index() {
    const int64_t total = gridDim.x, per = total / 8, i = blockIdx.x;
    return i < per * 8 ? (i % 8) * per + i / 8 : i;
}

// Rows [32 w, 32 w + 32) of the block per wavefront against a range of item tiles: reference, mass and (GRAD) the
// weighted sum of the items, per row and range.
template <int F, bool GRAD>
__global__ __launch_bounds__(64 * DI_NW) void distill_forward_kernel(
    const char* __restrict__ ximg, int64_t n, int64_t blocks, const char* __restrict__ yimg, int64_t m, int64_t ytiles,
    int64_t tiles_per_range, float step, const uint32_t* __restrict__ parts, float* __restrict__ pref,
    float* __restrict__ pmass, float* __restrict__ psum) {
    typedef DistillTile<F> D;
    constexpr int FETCH = GRAD ? D::BYTES : 2 * D::PLANE;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, half = lane >> 5;
    const int64_t work = di_work_index();
    const int64_t range = work / blocks, block = work % blocks;
    const int64_t t0 = range * tiles_per_range;
    const int64_t t1 = t0 + tiles_per_range < ytiles ? t0 + tiles_per_range : ytiles;
    const int64_t own0 = block * DI_OWN + wave * 32;
    const bool active = own0 < n;
    const float c = ldexpf(step, -di_scale_exponent(parts) - di_scale_exponent(parts + DI_PARTS));

    di_fetch(yimg + t0 * D::BYTES, lds, FETCH);
    u32x4 own[2][F / 16];
    if (active) di_load_own<F>(ximg + (own0 / 32) * D::BYTES, own);
    f32x16 acc[F / 32] = {};
    float ref = -INFINITY, mass = 0.f;
    for (int64_t t = t0; t < t1; ++t) {
        const char* tile = lds + ((t - t0) & 1) * D::BYTES;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();   // this tile has arrived, and every wavefront is done with the one before it
        if (t + 1 < t1) di_fetch(yimg + (t + 1) * D::BYTES, lds + ((t + 1 - t0) & 1) * D::BYTES, FETCH);
        if (!active) continue;
        f32x16 z = di_logits<F>(tile, own);
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
        const float off = DI_HEADROOM - ref;
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

// Items [32 w, 32 w + 32) of the block per wavefront against a range of row tiles: their gradient from those rows.
template <int F>
__global__ __launch_bounds__(64 * DI_NW) void distill_backward_kernel(
    const char* __restrict__ yimg, int64_t m, int64_t blocks, const char* __restrict__ ximg, int64_t n, int64_t xtiles,
    int64_t tiles_per_range, float step, float temperature, const uint32_t* __restrict__ parts, const float* __restrict__ ref,
    const float* __restrict__ mass, const float* __restrict__ a, const float* __restrict__ grad,
    const uint16_t* __restrict__ start, int64_t ytiles, const int32_t* __restrict__ list_id,
    const float* __restrict__ list_val, int k, float* __restrict__ out) {
    typedef DistillTile<F> D;
    extern __shared__ __attribute__((aligned(1024))) char lds[];
    __shared__ __attribute__((aligned(16))) float row_off[2][32], row_w[2][32], row_v[2][32];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, half = lane >> 5;
    const int64_t work = di_work_index();
    const int64_t range = work / blocks, block = work % blocks;
    const int64_t t0 = range * tiles_per_range;
    const int64_t t1 = t0 + tiles_per_range < xtiles ? t0 + tiles_per_range : xtiles;
    const int64_t own0 = block * DI_OWN + wave * 32, jt = own0 / 32;
    const bool active = own0 < m;
    const int sx = di_scale_exponent(parts), sy = di_scale_exponent(parts + DI_PARTS);
    const int sg = di_scale_exponent(parts + 2 * DI_PARTS);   // the weights of the rows; |q - p| and |A q| are at most 1
    const float c = ldexpf(step, -sx - sy);

    // what a row brings besides its factors: the reference of its logits, the weight of a probability, that of a list entry
    float p_ref = 0.f, p_w = 0.f, p_v = 0.f;
    auto fetch_rows = [&](int64_t t) {
        if (tid < 32) {
            const int64_t b = t * 32 + tid;
            const float w = b < n ? ldexpf(grad[b], sg) : 0.f;
            p_ref = b < n ? -ref[b] : 0.f;
            p_v = w;
            p_w = b < n ? w * a[b] / mass[b] : 0.f;
        }
    };
    auto store_rows = [&](int64_t t) {
        if (tid < 32) {
            row_off[(t - t0) & 1][tid] = p_ref;
            row_w[(t - t0) & 1][tid] = p_w;
            row_v[(t - t0) & 1][tid] = p_v;
        }
    };
    // a lane's row (of the tile) on the lists: where the entries of this wavefront's items begin and end
    int e0 = 0, e1 = 0;
    auto fetch_list = [&](int64_t t) {
        const int64_t b = t * 32 + (lane & 31);
        e0 = e1 = 0;
        if (active && b < n) {
            e0 = start[b * (ytiles + 1) + jt];
            e1 = start[b * (ytiles + 1) + jt + 1];
            e1 = e1 < k ? e1 : k;   // whatever the workspace holds, the list is not left
        }
    };
    di_fetch(ximg + t0 * D::BYTES, lds, D::BYTES);
    fetch_rows(t0);
    fetch_list(t0);
    u32x4 own[2][F / 16];
    if (active) di_load_own<F>(yimg + jt * D::BYTES, own);
    f32x16 acc[F / 32] = {};
    for (int64_t t = t0; t < t1; ++t) {
        const int cur = (int)((t - t0) & 1);
        const char* tile = lds + cur * D::BYTES;
        store_rows(t);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        // the first entry of each row's part of the list
        const int f0 = e0, f1 = e1;
        const int64_t lrow = (t * 32 + (lane & 31)) * k;
        int32_t id = 0;
        float val = 0.f;
        if (f1 > f0) {
            id = list_id[lrow + f0];
            val = list_val[lrow + f0];
        }
        if (t + 1 < t1) {
            di_fetch(ximg + (t + 1) * D::BYTES, lds + (cur ^ 1) * D::BYTES, D::BYTES);
            fetch_rows(t + 1);
            fetch_list(t + 1);
        }
        if (!active) continue;
        f32x16 z = di_logits<F>(tile, own);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 o = *reinterpret_cast<const f32x4*>(&row_off[cur][8 * g + 4 * half]);
            const f32x4 w = *reinterpret_cast<const f32x4*>(&row_w[cur][8 * g + 4 * half]);
#pragma unroll
            for (int i = 0; i < 4; ++i) z[4 * g + i] = __builtin_amdgcn_exp2f(__builtin_fmaf(z[4 * g + i], c, o[i])) * w[i];
        }
        // where an item is on a row's list, its gradient is not A q but q - p
        uint32_t rows = (uint32_t)__ballot(half == 0 && f1 > f0);
        while (rows) {
            const int r = __builtin_ctz(rows);
            rows &= rows - 1;
            const int n_e = __builtin_amdgcn_readlane(f1 - f0, r);
            int32_t item = __builtin_amdgcn_readlane(id, r);
            float v = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(val), r));
            const int first = __builtin_amdgcn_readlane(f0, r);
            for (int e = 0;;) {
                const bool here = lane == (int)(item - own0) + 32 * ((r >> 2) & 1);
                const float gv = v * row_v[cur][r];
                const int reg = 4 * (r >> 3) + (r & 3);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (i == reg) z[i] = here ? gv : z[i];
                if (++e >= n_e) break;
                item = list_id[(t * 32 + r) * k + first + e];
                v = list_val[(t * 32 + r) * k + first + e];
            }
        }
        di_accumulate<F>(tile, z, acc);
    }
    const int64_t item = own0 + (lane & 31);
    if (!active || item >= m) return;
    const float back = ldexpf(temperature, -sx - sg);
#pragma unroll
    for (int u = 0; u < F / 32; ++u)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 q = {acc[u][4 * g] * back, acc[u][4 * g + 1] * back, acc[u][4 * g + 2] * back, acc[u][4 * g + 3] * back};
            *reinterpret_cast<f32x4*>(out + (range * m + item) * F + 32 * u + 8 * g + 4 * half) = q;
        }
}

// The sum of the ranges' partial gradients, in their order.
__global__ __launch_bounds__(DI_THREADS) void distill_join_kernel(const float* __restrict__ part, int ranges, int64_t cnt,
                                                                  float* __restrict__ out) {
    for (int64_t e = ((int64_t)blockIdx.x * DI_THREADS + threadIdx.x) * 4; e < cnt; e += (int64_t)gridDim.x * DI_THREADS * 4) {
        f32x4 v = *reinterpret_cast<const f32x4*>(part + e);
        for (int r = 1; r < ranges; ++r) v += *reinterpret_cast<const f32x4*>(part + r * cnt + e);
        *reinterpret_cast<f32x4*>(out + e) = v;
    }
}

// ------------------------------------------------------------------------------------------------------- the lists

// One workgroup per row, one thread per list entry: joins the row's partial results; the list without its excluded
// entries, ordered by item, entries that name the same item merged (their probabilities add), and where the entries of
// every item tile begin in it; the row's loss; its dX but for the weight.
__global__ __launch_bounds__(DI_LIST) void distill_list_kernel(
    const float* __restrict__ X, int64_t n, const float* __restrict__ Y, int64_t m, int f, const int32_t* __restrict__ ids,
    const float* __restrict__ scores, int k, float temperature, const float* __restrict__ teacher_lse, int ranges,
    const float* __restrict__ pref, const float* __restrict__ pmass, const float* __restrict__ psum,
    const uint32_t* __restrict__ parts, float* __restrict__ loss, float* __restrict__ ref_out, float* __restrict__ mass_out,
    float* __restrict__ a_out, int32_t* __restrict__ count_out, int32_t* __restrict__ id_out, float* __restrict__ val_out,
    uint16_t* __restrict__ start_out, float* __restrict__ base) {
    __shared__ uint64_t key[DI_LIST];
    __shared__ int32_t sid[DI_LIST];     // by ascending item
    __shared__ float st[DI_LIST];        // log p, then the coefficient of y in dX
    __shared__ float sp[DI_LIST];        // p
    __shared__ int32_t mid[DI_LIST];     // merged
    __shared__ float mlogp[DI_LIST], mp[DI_LIST], mz[DI_LIST];
    __shared__ float partf[DI_THREADS / 64];
    __shared__ double partd[DI_THREADS / 64];
    __shared__ int parti[DI_THREADS / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const double inv_t = 1.0 / (double)temperature;
    const int64_t ytiles = (m + 31) / 32;
    const int sy = di_scale_exponent(parts + DI_PARTS);

    for (int64_t b = blockIdx.x; b < n; b += gridDim.x) {
        float ref = -INFINITY, mass2 = 0.f, mean = 0.f;
        for (int r = 0; r < ranges; ++r) ref = fmaxf(ref, pref[r * n + b]);
        for (int r = 0; r < ranges; ++r) {
            const float w = __builtin_amdgcn_exp2f(pref[r * n + b] - ref);
            mass2 = __builtin_fmaf(pmass[r * n + b], w, mass2);
            if (base && tid < f) mean = __builtin_fmaf(psum[(r * n + b) * f + tid], w, mean);
        }
        mean = ldexpf(mean / mass2, -sy);
        mass2 = ldexpf(mass2, -(int)DI_HEADROOM);
        const double log_mass = (double)ref * 0.69314718055994531 + log((double)mass2);   // log sum exp of the logits

        const int32_t id = tid < k ? ids[b * k + tid] : -1;
        const float s = tid < k ? scores[b * k + tid] : 0.f;
        const bool valid = id >= 0 && id < m && s > -FLT_MAX;
        const float top = di_block_max(valid ? s : -INFINITY, partf);
        // log p of the entry (before merging)
        const double d = s == top ? 0.0 : ((double)s - (double)top) * inv_t;
        const double mass = di_block_sum(valid ? (double)expf((float)d) : 0.0, partd);
        const int nvalid = __syncthreads_count(valid);
        if (tid == 0) {
            ref_out[b] = ref;
            mass_out[b] = mass2;
        }
        if (nvalid == 0) {   // nothing to learn from this row
            if (tid == 0) {
                loss[b] = 0.f;
                a_out[b] = 0.f;
                count_out[b] = 0;
            }
            if (base) {
                if (tid < f) base[b * f + tid] = 0.f;
                for (int64_t t = tid; t <= ytiles; t += DI_LIST) start_out[b * (ytiles + 1) + t] = 0;
            }
            continue;
        }
        const float logp = (float)(teacher_lse ? (double)s * inv_t - (double)teacher_lse[b] : d - log(mass));
        key[tid] = valid ? ((uint64_t)id << 8) | (uint64_t)tid : ~0ull;
        __syncthreads();
        if (valid) {
            int rank = 0;
            const uint64_t mine = key[tid];
            for (int j = 0; j < k; ++j) rank += key[j] < mine ? 1 : 0;
            sid[rank] = id;
            st[rank] = logp;
            sp[rank] = expf(logp);
        }
        __syncthreads();
        const bool head = tid < nvalid && (tid == 0 || sid[tid] != sid[tid - 1]);
        const uint64_t votes = __ballot(head);
        if (lane == 0) parti[wave] = __popcll(votes);
        __syncthreads();
        int at = __popcll(votes & ((1ull << lane) - 1)), merged = 0;
        for (int w = 0; w < DI_THREADS / 64; ++w) {
            at += w < wave ? parti[w] : 0;
            merged += parti[w];
        }
        if (head) {
            float p = sp[tid], lp = st[tid];
            int j = tid + 1;
            for (; j < nvalid && sid[j] == sid[tid]; ++j) p += sp[j];
            if (j > tid + 1) lp = logf(p);
            mid[at] = sid[tid];
            mp[at] = p;
            mlogp[at] = lp;
        }
        __syncthreads();
        // the student's logits on the list: half a wavefront per entry
        for (int e = tid >> 5; e < merged; e += DI_THREADS / 32) {
            const float* y = Y + (int64_t)mid[e] * f;
            float z = 0.f;
            for (int c = tid & 31; c < f; c += 32) z = __builtin_fmaf(X[b * f + c], y[c], z);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) z += __shfl_xor(z, o, 64);
            if ((tid & 31) == 0) mz[e] = z;
        }
        __syncthreads();
        const bool mine = tid < merged;
        const double logq = mine ? (double)mz[tid] * inv_t - log_mass : 0.0;
        const float q = mine ? expf((float)logq) : 0.f;
        const float p = mine ? mp[tid] : 0.f;
        // (a NaN probability stays in the sum)
        double kl = di_block_sum(mine && !(p <= 0.f) ? (double)p * ((double)mlogp[tid] - logq) : 0.0, partd);
        float a = 1.f;
        if (teacher_lse) {
            const double pr = fmax(1.0 - di_block_sum((double)p, partd), 0.0);
            const double qr = fmax(1.0 - di_block_sum((double)q, partd), 0x1p-24);
            if (pr > 0.0) {
                kl += pr * log(pr / qr);
                a = (float)(1.0 - pr / qr);
            }
        }
        if (tid == 0) {
            loss[b] = (float)((double)temperature * (double)temperature * kl);
            a_out[b] = a;
            count_out[b] = merged;
        }
        if (mine) st[tid] = (1.f - a) * q - p;
        if (base) {
            if (mine) {
                id_out[b * k + tid] = mid[tid];
                val_out[b * k + tid] = q - p;
            }
            for (int64_t t = tid; t <= ytiles; t += DI_LIST) {
                int lo = 0, hi = merged;
                while (lo < hi) {
                    const int c = (lo + hi) >> 1;
                    if ((int64_t)mid[c] < t * 32) lo = c + 1;
                    else hi = c;
                }
                start_out[b * (ytiles + 1) + t] = (uint16_t)lo;
            }
            __syncthreads();
            if (tid < f) {
                float acc = a * mean;
                for (int e = 0; e < merged; ++e) acc = __builtin_fmaf(st[e], Y[(int64_t)mid[e] * f + tid], acc);
                base[b * f + tid] = acc;
            }
        }
        __syncthreads();
    }
}

// dX, and the partial maxima of |grad| that scale the weights of the backward pass.
__global__ __launch_bounds__(DI_THREADS) void distill_dx_kernel(const float* __restrict__ base, const float* __restrict__ grad,
                                                                float temperature, int64_t n, int f, float* __restrict__ dX,
                                                                uint32_t* __restrict__ parts) {
    __shared__ uint32_t part[DI_THREADS / 64];
    uint32_t top = 0;
    if (dX)
        for (int64_t e = ((int64_t)blockIdx.x * DI_THREADS + threadIdx.x) * 4; e < n * f; e += (int64_t)DI_PARTS * DI_THREADS * 4) {
            const float g = grad[e / f] * temperature;
            *reinterpret_cast<f32x4*>(dX + e) = *reinterpret_cast<const f32x4*>(base + e) * g;
        }
    for (int64_t b = (int64_t)blockIdx.x * DI_THREADS + threadIdx.x; b < n; b += (int64_t)DI_PARTS * DI_THREADS) {
        const uint32_t u = __float_as_uint(grad[b]) & 0x7fffffffu;
        top = u > top ? u : top;
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) {
        const uint32_t o = (uint32_t)__shfl_xor((int)top, d, 64);
        top = o > top ? o : top;
    }
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < DI_THREADS / 64; ++w) top = part[w] > top ? part[w] : top;
        parts[blockIdx.x] = top;
    }
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
    MIREC_REQUIRE(n <= ((int64_t)1 << 28) && m <= ((int64_t)1 << 28), MIREC_E_UNSUPPORTED, "%s: more than 2^28 rows or items",
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

// Dynamic LDS of the two passes (two tiles) needs an attribute once per kernel and device.
static int distill_lds(const void* kernel, int bytes, OncePerDevice& once, const char* who) {
    bool* done = once.slot();
    MIREC_REQUIRE(done, MIREC_E_HIP, "%s: cannot read the current device", who);
    if (!*done) {   // idempotent; a race only repeats the call
        MIREC_HIP(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes));
        *done = true;
    }
    return MIREC_OK;
}

template <int F, bool GRAD>
static int launch_forward(const DistillWorkspace& L, char* w, const float* X, int64_t n, const float* Y, int64_t m, float step,
                          hipStream_t stream) {
    static OncePerDevice once;
    constexpr int LDS = 2 * DistillTile<F>::BYTES;
    if (const int rc = distill_lds((const void*)distill_forward_kernel<F, GRAD>, LDS, once, "mirec_distill_loss")) return rc;
    uint32_t* parts = (uint32_t*)(w + L.max_off);
    hipLaunchKernelGGL((distill_image_kernel<F>), dim3((unsigned)(L.xtiles + L.ytiles)), dim3(DI_THREADS), 0, stream, X, n,
                       L.xtiles, w + L.ximg_off, Y, m, w + L.yimg_off, parts);
    MIREC_LAUNCH_CHECK();
    const int64_t blocks = (n + DI_OWN - 1) / DI_OWN, per = (L.ytiles + L.splits_x - 1) / L.splits_x;
    const int64_t ranges = (L.ytiles + per - 1) / per;
    hipLaunchKernelGGL((distill_forward_kernel<F, GRAD>), dim3((unsigned)(blocks * ranges)), dim3(64 * DI_NW), LDS, stream,
                       w + L.ximg_off, n, blocks, w + L.yimg_off, m, L.ytiles, per, step, parts, (float*)(w + L.pref_off),
                       (float*)(w + L.pmass_off), (float*)(w + L.part_off));
    MIREC_LAUNCH_CHECK();
    return MIREC_OK;
}

template <int F>
static int launch_backward(const DistillWorkspace& L, char* w, int64_t n, int64_t m, int k, float step, float temperature,
                           const float* grad, float* dY, hipStream_t stream) {
    static OncePerDevice once;
    constexpr int LDS = 2 * DistillTile<F>::BYTES;
    if (const int rc = distill_lds((const void*)distill_backward_kernel<F>, LDS, once, "mirec_distill_grad")) return rc;
    const int64_t blocks = (m + DI_OWN - 1) / DI_OWN, per = (L.xtiles + L.splits_y - 1) / L.splits_y;
    const int64_t ranges = (L.xtiles + per - 1) / per;
    float* out = ranges > 1 ? (float*)(w + L.part_off) : dY;
    hipLaunchKernelGGL((distill_backward_kernel<F>), dim3((unsigned)(blocks * ranges)), dim3(64 * DI_NW), LDS, stream,
                       w + L.yimg_off, m, blocks, w + L.ximg_off, n, L.xtiles, per, step, temperature,
                       (const uint32_t*)(w + L.max_off), (const float*)(w + L.ref_off), (const float*)(w + L.mass_off),
                       (const float*)(w + L.a_off), grad, (const uint16_t*)(w + L.start_off), L.ytiles,
                       (const int32_t*)(w + L.id_off), (const float*)(w + L.val_off), k, out);
    MIREC_LAUNCH_CHECK();
    if (ranges > 1) {
        const int64_t jb = (m * F / 4 + DI_THREADS - 1) / DI_THREADS;
        hipLaunchKernelGGL(distill_join_kernel, dim3((unsigned)(jb < 4096 ? jb : 4096)), dim3(DI_THREADS), 0, stream, out,
                           (int)ranges, m * F, dY);
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
    const float step = (float)(1.4426950408889634 / (double)temperature);
    hipLaunchKernelGGL(distill_absmax_kernel, dim3(DI_PARTS, 2), dim3(DI_THREADS), 0, stream, X, n * f, Y, m * f,
                       (uint32_t*)(w + L.max_off));
    MIREC_LAUNCH_CHECK();
    int rc = MIREC_OK;
    switch (f) {
#define MIREC_DISTILL_CASE(FW)                                                                                  case FW:                                                                                                        rc = with_grad ? launch_forward<FW, true>(L, w, X, n, Y, m, step, stream)                                                  : launch_forward<FW, false>(L, w, X, n, Y, m, step, stream);                                 break;
        MIREC_DISTILL_WIDTHS(MIREC_DISTILL_CASE)
#undef MIREC_DISTILL_CASE
    }
    if (rc) return rc;
    const int64_t per = (L.ytiles + L.splits_x - 1) / L.splits_x;
    hipLaunchKernelGGL(distill_list_kernel, dim3((unsigned)(n < 262144 ? n : 262144)), dim3(DI_LIST), 0, stream, X, n, Y, m, f,
                       ids, scores, k, temperature, teacher_lse, (int)((L.ytiles + per - 1) / per),
                       (const float*)(w + L.pref_off), (const float*)(w + L.pmass_off), (const float*)(w + L.part_off),
                       (const uint32_t*)(w + L.max_off), loss, (float*)(w + L.ref_off), (float*)(w + L.mass_off),
                       (float*)(w + L.a_off), (int32_t*)(w + L.count_off), (int32_t*)(w + L.id_off), (float*)(w + L.val_off),
                       (uint16_t*)(w + L.start_off), with_grad ? (float*)(w + L.base_off) : nullptr);
    MIREC_LAUNCH_CHECK();
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
    hipLaunchKernelGGL(distill_dx_kernel, dim3(DI_PARTS), dim3(DI_THREADS), 0, stream, (const float*)(w + L.base_off), grad,
                       temperature, n, f, dX, (uint32_t*)(w + L.max_off) + 2 * DI_PARTS);
    MIREC_LAUNCH_CHECK();
    if (!dY) return MIREC_OK;
    const float step = (float)(1.4426950408889634 / (double)temperature);
    switch (f) {
#define MIREC_DISTILL_CASE(FW) \
    case FW:                   \
        return launch_backward<FW>(L, w, n, m, k, step, temperature, grad, dY, stream);
        MIREC_DISTILL_WIDTHS(MIREC_DISTILL_CASE)
#undef MIREC_DISTILL_CASE
    }
    return MIREC_OK;
}
