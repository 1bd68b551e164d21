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
#include <float.h>

#include "common.h"

namespace mirec {

constexpr int DI_LIST = MIREC_DISTILL_MAX_LIST;   // longest list; one thread per entry in distill_list_kernel
constexpr int DI_THREADS = 256;

// Workspace of a call pair (host side): what mirec_distill_loss leaves for mirec_distill_grad.
struct DistillWorkspace {
    size_t lse_off, a_off, count_off, id_off, val_off, base_off, bytes;
};

static DistillWorkspace distill_layout(int64_t n, int64_t m, int f, int k) {
    (void)m;
    DistillWorkspace w;
    size_t at = 0;
    auto take = [&](size_t b) {
        const size_t o = at;
        at += align_up(b, 256);
        return o;
    };
    w.lse_off = take((size_t)n * 4);          // log sum exp of z_b
    w.a_off = take((size_t)n * 4);            // A_b
    w.count_off = take((size_t)n * 4);        // entries of the merged list
    w.id_off = take((size_t)n * k * 4);       // merged list, ascending ids
    w.val_off = take((size_t)n * k * 4);      // q - p of those
    w.base_off = take((size_t)n * f * 4);     // mean_b, then dX_b / (grad_b T)
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

// One workgroup per row: log sum exp of the row's logits and, where `mean` is given, the mean of the items under the
// row's softmax.
__global__ __launch_bounds__(DI_THREADS) void distill_dense_kernel(const float* __restrict__ X, int64_t n,
                                                                   const float* __restrict__ Y, int64_t m, int f,
                                                                   float inv_t, float* __restrict__ lse,
                                                                   float* __restrict__ mean) {
    __shared__ float x[192];
    __shared__ float q[DI_THREADS];
    __shared__ float partf[DI_THREADS / 64];
    __shared__ double partd[DI_THREADS / 64];
    const int tid = threadIdx.x;
    for (int64_t b = blockIdx.x; b < n; b += gridDim.x) {
        __syncthreads();
        if (tid < f) x[tid] = X[b * f + tid];
        __syncthreads();
        auto logit = [&](int64_t j) -> float {
            float z = 0.f;
            for (int c = 0; c < f; ++c) z = __builtin_fmaf(x[c], Y[j * f + c], z);
            return z * inv_t;
        };
        float top = -INFINITY;
        for (int64_t j = tid; j < m; j += DI_THREADS) top = fmaxf(top, logit(j));
        top = di_block_max(top, partf);
        double mass = 0;
        for (int64_t j = tid; j < m; j += DI_THREADS) mass += (double)expf(logit(j) - top);
        mass = di_block_sum(mass, partd);
        const float l = (float)((double)top + log(mass));
        if (tid == 0) lse[b] = l;
        if (mean) {
            float acc = 0.f;
            for (int64_t j0 = 0; j0 < m; j0 += DI_THREADS) {
                __syncthreads();
                q[tid] = j0 + tid < m ? expf(logit(j0 + tid) - l) : 0.f;
                __syncthreads();
                const int cnt = (int)(m - j0 < DI_THREADS ? m - j0 : DI_THREADS);
                if (tid < f)
                    for (int j = 0; j < cnt; ++j) acc = __builtin_fmaf(q[j], Y[(j0 + j) * f + tid], acc);
            }
            if (tid < f) mean[b * f + tid] = acc;
        }
    }
}

// One workgroup per row, one thread per list entry: the list without its excluded entries, ordered by item, entries
// that name the same item merged (their probabilities add); the row's loss; what the gradients need of it.
__global__ __launch_bounds__(DI_LIST) void distill_list_kernel(
    const float* __restrict__ X, int64_t n, const float* __restrict__ Y, int64_t m, int f, const int32_t* __restrict__ ids,
    const float* __restrict__ scores, int k, float temperature, const float* __restrict__ teacher_lse,
    const float* __restrict__ lse, float* __restrict__ loss, float* __restrict__ a_out, int32_t* __restrict__ count_out,
    int32_t* __restrict__ id_out, float* __restrict__ val_out, float* __restrict__ base) {
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
    const float inv_t = 1.f / temperature;

    for (int64_t b = blockIdx.x; b < n; b += gridDim.x) {
        const int32_t id = tid < k ? ids[b * k + tid] : -1;
        const float s = tid < k ? scores[b * k + tid] : 0.f;
        const bool valid = id >= 0 && id < m && s > -FLT_MAX;
        const float top = di_block_max(valid ? s : -INFINITY, partf);
        // log p of the entry (before merging)
        const float d = s == top ? 0.f : (s - top) * inv_t;
        const double mass = di_block_sum(valid ? (double)expf(d) : 0.0, partd);
        const int nvalid = __syncthreads_count(valid);
        if (nvalid == 0) {   // nothing to learn from this row
            if (tid == 0) {
                loss[b] = 0.f;
                a_out[b] = 0.f;
                count_out[b] = 0;
            }
            if (base && tid < f) base[b * f + tid] = 0.f;
            continue;
        }
        const float logp = teacher_lse ? (float)((double)s * (double)inv_t - (double)teacher_lse[b])
                                       : d - (float)log(mass);
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
            if ((tid & 31) == 0) mz[e] = z * inv_t;
        }
        __syncthreads();
        const bool mine = tid < merged;
        const float logq = mine ? mz[tid] - lse[b] : 0.f;
        const float q = mine ? expf(logq) : 0.f;
        const float p = mine ? mp[tid] : 0.f;
        double kl = di_block_sum(mine && p > 0.f ? (double)p * ((double)mlogp[tid] - (double)logq) : mine ? 0.0 * p : 0.0, partd);
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
        if (mine) {
            id_out[b * k + tid] = mid[tid];
            val_out[b * k + tid] = q - p;
            st[tid] = (1.f - a) * q - p;
        }
        __syncthreads();
        if (base && tid < f) {
            float acc = a * base[b * f + tid];
            for (int e = 0; e < merged; ++e) acc = __builtin_fmaf(st[e], Y[(int64_t)mid[e] * f + tid], acc);
            base[b * f + tid] = acc;
        }
        __syncthreads();
    }
}

__global__ __launch_bounds__(DI_THREADS) void distill_dx_kernel(const float* __restrict__ base, const float* __restrict__ grad,
                                                                float temperature, int64_t n, int f,
                                                                float* __restrict__ dX) {
    for (int64_t e = (int64_t)blockIdx.x * DI_THREADS + threadIdx.x; e < n * f; e += (int64_t)gridDim.x * DI_THREADS)
        dX[e] = grad[e / f] * temperature * base[e];
}

// One workgroup per item: its gradient over all rows.
__global__ __launch_bounds__(DI_THREADS) void distill_dy_kernel(
    const float* __restrict__ X, int64_t n, const float* __restrict__ Y, int64_t m, int f, float temperature,
    const float* __restrict__ lse, const float* __restrict__ a_in, const int32_t* __restrict__ count,
    const int32_t* __restrict__ list_id, const float* __restrict__ list_val, int k, const float* __restrict__ grad,
    float* __restrict__ dY) {
    __shared__ float y[192];
    __shared__ float g[DI_THREADS];
    const int tid = threadIdx.x;
    const float inv_t = 1.f / temperature;
    for (int64_t j = blockIdx.x; j < m; j += gridDim.x) {
        __syncthreads();
        if (tid < f) y[tid] = Y[j * f + tid];
        float acc = 0.f;
        for (int64_t b0 = 0; b0 < n; b0 += DI_THREADS) {
            __syncthreads();
            const int64_t b = b0 + tid;
            g[tid] = 0.f;
            if (b < n) {
                float z = 0.f;
                for (int c = 0; c < f; ++c) z = __builtin_fmaf(X[b * f + c], y[c], z);
                float v = a_in[b] * expf(z * inv_t - lse[b]);
                int lo = 0, hi = count[b];
                while (lo < hi) {
                    const int mid = (lo + hi) >> 1;
                    if (list_id[b * k + mid] < j) lo = mid + 1;
                    else hi = mid;
                }
                if (lo < count[b] && list_id[b * k + lo] == j) v = list_val[b * k + lo];
                g[tid] = v * grad[b] * temperature;
            }
            __syncthreads();
            const int cnt = (int)(n - b0 < DI_THREADS ? n - b0 : DI_THREADS);
            if (tid < f)
                for (int i = 0; i < cnt; ++i) acc = __builtin_fmaf(g[i], X[(b0 + i) * f + tid], acc);
        }
        if (tid < f) dY[j * f + tid] = acc;
    }
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
    MIREC_REQUIRE(n < ((int64_t)1 << 31) && m < ((int64_t)1 << 31), MIREC_E_UNSUPPORTED, "%s: more than 2^31 rows or items",
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

}  // namespace mirec

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
    float* lse = (float*)(w + L.lse_off);
    float* base = with_grad ? (float*)(w + L.base_off) : nullptr;
    const unsigned rows = (unsigned)(n < 262144 ? n : 262144);
    hipLaunchKernelGGL(distill_dense_kernel, dim3(rows), dim3(DI_THREADS), 0, stream, X, n, Y, m, f, 1.f / temperature, lse,
                       base);
    MIREC_LAUNCH_CHECK();
    hipLaunchKernelGGL(distill_list_kernel, dim3(rows), dim3(DI_LIST), 0, stream, X, n, Y, m, f, ids, scores, k, temperature,
                       teacher_lse, lse, loss, (float*)(w + L.a_off), (int32_t*)(w + L.count_off), (int32_t*)(w + L.id_off),
                       (float*)(w + L.val_off), base);
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
    const DistillWorkspace L = distill_layout(n, m, f, k);
    if (n > 0)
        if (const int rc = distill_check_ws("mirec_distill_grad", ws, ws_bytes, L.bytes)) return rc;
    char* w = (char*)ws;
    if (dX && n > 0) {
        const int64_t blocks = (n * f + DI_THREADS - 1) / DI_THREADS;
        hipLaunchKernelGGL(distill_dx_kernel, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(DI_THREADS), 0, stream,
                           (const float*)(w + L.base_off), grad, temperature, n, f, dX);
        MIREC_LAUNCH_CHECK();
    }
    if (dY && m > 0) {
        hipLaunchKernelGGL(distill_dy_kernel, dim3((unsigned)(m < 262144 ? m : 262144)), dim3(DI_THREADS), 0, stream, X, n, Y,
                           m, f, temperature, (const float*)(w + L.lse_off), (const float*)(w + L.a_off),
                           (const int32_t*)(w + L.count_off), (const int32_t*)(w + L.id_off), (const float*)(w + L.val_off), k,
                           grad, dY);
        MIREC_LAUNCH_CHECK();
    }
    return MIREC_OK;
}
