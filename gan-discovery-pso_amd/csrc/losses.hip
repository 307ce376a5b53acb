// Losses over the logits of a choice (codes of a codebook, classes of an assessor, experts of a router), with
// their gradients:
//
//   balance   p_i = softmax(row i), P[c] = mean of p over the kept rows, f[c] = choices of c / all counted choices,
//             loss = E sum_c f[c] P[c],            d loss / d s[i,c] = (E / rows) p[i,c] (f[c] - sum_j f[j] p[i,j])
//   distill   q_i = softmax(teacher's kept logits / t), p_i = softmax(row i / t),
//             loss = t^2 mean_i sum_j q_ij (log q_ij - log p_i[idx_ij]),
//                                                  d loss / d s[i,c] = (t / rows) (p[i,c] - sum of q_ij with idx_ij = c)
//
// All softmax statistics, sums and gradients are fp32 (joins of many partial sums fp64); a gradient is rounded once,
// to the logits' type, when it is stored.  A row without a finite logit has p = 0; NaN and +inf propagate.
#include "common.h"

#include <math.h>

namespace gdpso {
namespace {

constexpr int LOSS_THREADS = 256;
constexpr int BAL_MAX_E = GDPSO_BALANCE_MAX_E;
constexpr int DIST_MAX_K = GDPSO_DISTILL_MAX_K;

// log2(e) / temperature as hi + lo, hi below the exact value so that lo > 0: then d * lo of d = -inf is -inf, not NaN.
struct ExpScale {
    float hi, lo;
};
inline ExpScale exp_scale(double temperature) {
    const double c = 1.4426950408889634074 / temperature;
    ExpScale s;
    s.hi = (float)c;
    if ((double)s.hi >= c) s.hi = nextafterf(s.hi, 0.f);
    s.lo = (float)(c - (double)s.hi);
    return s;
}
// exp(d / temperature) for d <= 0.  The second term keeps the argument's rounding error of a long way below the
// maximum out of the result; the instruction returns 0 where the result would be subnormal.
__device__ __forceinline__ float exp_scaled(float d, ExpScale s) { return __builtin_amdgcn_exp2f(fmaf(d, s.hi, d * s.lo)); }

template <typename E>
__device__ __forceinline__ float to_f32(E v) { return (float)v; }

__device__ __forceinline__ float block_max(float v, float *s_red) {
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s_red[0];
    for (int w = 1; w < LOSS_THREADS / 64; ++w) v = fmaxf(v, s_red[w]);
    return v;
}
__device__ __forceinline__ float block_sum(float v, float *s_red) {
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s_red[0];
    for (int w = 1; w < LOSS_THREADS / 64; ++w) v += s_red[w];
    return v;
}
// Maximum (0 where there is none, so that differences stay defined) and sum of exp of a row, over the workgroup.
template <typename E>
__device__ __forceinline__ void row_stats(const E *row, int e, ExpScale sc, float *s_red, float &m, float &l) {
    m = -INFINITY;
    for (int c = threadIdx.x; c < e; c += LOSS_THREADS) m = fmaxf(m, to_f32(row[c]));
    m = block_max(m, s_red);
    if (m == -INFINITY) m = 0.f;
    l = 0.f;
    for (int c = threadIdx.x; c < e; c += LOSS_THREADS) l += exp_scaled(to_f32(row[c]) - m, sc);
    l = block_sum(l, s_red);
}

__device__ __forceinline__ long long load_index(const void *idx, int index_bytes, long long i) {
    return index_bytes == 8 ? ((const long long *)idx)[i] : (long long)((const int *)idx)[i];
}

__global__ void fill_zero_kernel(long long *p, int n) {
    const int i = blockIdx.x * LOSS_THREADS + threadIdx.x;
    if (i < n) p[i] = 0;
}

// counts[c] += choices of c, counts[e] += rows kept, counts[e + 1] += choices counted (whole numbers: any order gives
// the same sums)
__global__ __launch_bounds__(LOSS_THREADS) void bal_count_kernel(int n, int e, int k, const void *__restrict__ idx, int index_bytes,
                                                                 const unsigned char *__restrict__ mask, unsigned long long *counts) {
    int rows = 0, chosen = 0;
    for (long long i = (long long)blockIdx.x * LOSS_THREADS + threadIdx.x; i < n; i += (long long)gridDim.x * LOSS_THREADS) {
        if (mask && !mask[i]) continue;
        ++rows;
        for (int j = 0; j < k; ++j) {
            const long long c = load_index(idx, index_bytes, i * k + j);
            if (c < 0 || c >= e) continue;
            ++chosen;
            atomicAdd(&counts[c], 1ull);
        }
    }
    if (rows) atomicAdd(&counts[e], (unsigned long long)rows);
    if (chosen) atomicAdd(&counts[e + 1], (unsigned long long)chosen);
}

// Column sums of p over this workgroup's rows -> part[blockIdx][e]; gradients of its rows when GRAD.
template <typename E, bool SUMS, bool GRAD>
__global__ __launch_bounds__(LOSS_THREADS) void bal_rows_kernel(int n, int e, const E *__restrict__ logits, long long row_stride,
                                                                const unsigned char *__restrict__ mask, const long long *__restrict__ counts,
                                                                float grad_scale, const float *__restrict__ upstream, float *__restrict__ part,
                                                                E *__restrict__ grad, ExpScale sc) {
    extern __shared__ float s_col[];
    __shared__ float s_red[LOSS_THREADS / 64];
    float inv_n = 0.f, factor = 0.f;
    if (GRAD) {
        const long long rows = counts[e], chosen = counts[e + 1];
        inv_n = chosen > 0 ? 1.f / (float)chosen : 0.f;
        factor = rows > 0 ? (upstream ? *upstream : grad_scale) * (float)e / (float)rows : 0.f;
    }
    if (SUMS)
        for (int c = threadIdx.x; c < e; c += LOSS_THREADS) s_col[c] = 0.f;
    for (long long i = blockIdx.x; i < n; i += gridDim.x) {
        const E *row = logits + i * row_stride;
        if (mask && !mask[i]) {
            if (GRAD)
                for (int c = threadIdx.x; c < e; c += LOSS_THREADS) grad[i * e + c] = (E)0.f;
            continue;
        }
        float m, l;
        row_stats(row, e, sc, s_red, m, l);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        float dot = 0.f;
        for (int c = threadIdx.x; c < e; c += LOSS_THREADS) {
            const float p = exp_scaled(to_f32(row[c]) - m, sc) * inv;
            if (SUMS) s_col[c] += p;
            if (GRAD) dot = fmaf(p, (float)counts[c] * inv_n, dot);
        }
        if (GRAD) {
            dot = block_sum(dot, s_red);
            for (int c = threadIdx.x; c < e; c += LOSS_THREADS) {
                const float p = exp_scaled(to_f32(row[c]) - m, sc) * inv;
                grad[i * e + c] = (E)(factor * p * ((float)counts[c] * inv_n - dot));
            }
        }
    }
    if (SUMS)
        for (int c = threadIdx.x; c < e; c += LOSS_THREADS) part[(size_t)blockIdx.x * e + c] = s_col[c];
}

__global__ __launch_bounds__(LOSS_THREADS) void bal_finish_kernel(int e, int nparts, const float *__restrict__ part,
                                                                  const long long *__restrict__ counts, float *__restrict__ mean_prob,
                                                                  float *__restrict__ loss) {
    __shared__ double s_sum[LOSS_THREADS];
    const double inv_t = counts[e] > 0 ? 1. / (double)counts[e] : 0., inv_n = counts[e + 1] > 0 ? 1. / (double)counts[e + 1] : 0.;
    double dot = 0.;
    for (int c = threadIdx.x; c < e; c += LOSS_THREADS) {
        double s = 0.;
        for (int g = 0; g < nparts; ++g) s += part[(size_t)g * e + c];
        s *= inv_t;
        mean_prob[c] = (float)s;
        dot += s * ((double)counts[c] * inv_n);
    }
    s_sum[threadIdx.x] = dot;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.;
        for (int i = 0; i < LOSS_THREADS; ++i) t += s_sum[i];
        *loss = (float)(t * e);
    }
}

// stats[2n] = 1 / rows the mask keeps (0: none)
__global__ __launch_bounds__(LOSS_THREADS) void dist_rows_kept_kernel(int n, const unsigned char *__restrict__ mask, float *inv_rows) {
    __shared__ long long s_cnt[LOSS_THREADS];
    long long cnt = 0;
    for (int i = threadIdx.x; i < n; i += LOSS_THREADS) cnt += !mask || mask[i] != 0;
    s_cnt[threadIdx.x] = cnt;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < LOSS_THREADS; ++i) cnt += s_cnt[i];
        *inv_rows = cnt > 0 ? (float)(1. / (double)cnt) : 0.f;
    }
}

__device__ __forceinline__ float load_typed(const void *p, int dtype, long long i) {
    if (dtype == DT_F32) return ((const float *)p)[i];
    if (dtype == DT_BF16) return (float)((const bf16_t *)p)[i];
    return (float)((const f16_t *)p)[i];
}

// One workgroup per row.  VALUE: row_loss and stats (maximum, sum) are written; else the stats are read.
template <typename E, bool VALUE, bool GRAD>
__global__ __launch_bounds__(LOSS_THREADS) void dist_rows_kernel(int n, int v, int k, const E *__restrict__ logits, long long row_stride,
                                                                 const void *__restrict__ t_logits, int t_dtype, const void *__restrict__ t_idx,
                                                                 int index_bytes, const unsigned char *__restrict__ mask, float temperature,
                                                                 ExpScale sc, float grad_scale, const float *__restrict__ upstream,
                                                                 float *__restrict__ stats, const float *__restrict__ inv_rows,
                                                                 float *__restrict__ row_loss, E *__restrict__ grad) {
    __shared__ float s_red[LOSS_THREADS / 64];
    __shared__ float s_q[DIST_MAX_K];
    __shared__ int s_i[DIST_MAX_K];
    const float inv_t = 1.f / temperature;
    for (long long i = blockIdx.x; i < n; i += gridDim.x) {
        const E *row = logits + i * row_stride;
        E *grow = grad + i * v;
        if (mask && !mask[i]) {
            if (VALUE && threadIdx.x == 0) {
                row_loss[i] = 0.f;
                stats[2 * i] = 0.f;
                stats[2 * i + 1] = 0.f;
            }
            if (GRAD)
                for (int c = threadIdx.x; c < v; c += LOSS_THREADS) grow[c] = (E)0.f;
            continue;
        }
        // the teacher's entries: an index outside the row is no entry
        float tm = -INFINITY;
        __syncthreads();
        for (int j = threadIdx.x; j < k; j += LOSS_THREADS) {
            const long long c = load_index(t_idx, index_bytes, i * k + j);
            const bool in = c >= 0 && c < v;
            const float t = in ? load_typed(t_logits, t_dtype, i * k + j) : -INFINITY;
            s_i[j] = in ? (int)c : -1;
            s_q[j] = t;
            tm = fmaxf(tm, t);
        }
        tm = block_max(tm, s_red);
        if (tm == -INFINITY) tm = 0.f;
        float tl = 0.f;
        for (int j = threadIdx.x; j < k; j += LOSS_THREADS) tl += exp_scaled(s_q[j] - tm, sc);
        tl = block_sum(tl, s_red);
        float m, l;
        if (VALUE) {
            row_stats(row, v, sc, s_red, m, l);
            if (threadIdx.x == 0) {
                stats[2 * i] = m;
                stats[2 * i + 1] = l;
            }
        } else {
            m = stats[2 * i];
            l = stats[2 * i + 1];
        }
        const bool empty = l == 0.f || tl == 0.f;
        const float inv_tl = empty ? 0.f : 1.f / tl, inv_l = empty ? 0.f : 1.f / l;
        float part = 0.f;
        for (int j = threadIdx.x; j < k; j += LOSS_THREADS) {
            const float t = s_q[j], q = exp_scaled(t - tm, sc) * inv_tl;
            s_q[j] = q;
            if (VALUE && q != 0.f) part += q * ((t - tm) - (to_f32(row[s_i[j]]) - m)) * inv_t;
        }
        if (VALUE) {
            part = block_sum(part, s_red);
            if (threadIdx.x == 0) row_loss[i] = empty ? 0.f : temperature * temperature * (part + (logf(l) - logf(tl)));
        }
        if (GRAD) {
            const float factor = (upstream ? *upstream : grad_scale) * temperature * *inv_rows;
            for (int c = threadIdx.x; c < v; c += LOSS_THREADS)
                grow[c] = empty ? (E)0.f : (E)(factor * (exp_scaled(to_f32(row[c]) - m, sc) * inv_l));
            __syncthreads();
            // the columns the teacher names: the first entry of a column stores for all entries of it
            if (!empty)
                for (int j = threadIdx.x; j < k; j += LOSS_THREADS) {
                    const int c = s_i[j];
                    bool first = c >= 0;
                    for (int h = 0; h < j && first; ++h) first = s_i[h] != c;
                    if (!first) continue;
                    float q = s_q[j];
                    for (int h = j + 1; h < k; ++h)
                        if (s_i[h] == c) q += s_q[h];
                    grow[c] = (E)(factor * (exp_scaled(to_f32(row[c]) - m, sc) * inv_l - q));
                }
        }
    }
}

__global__ __launch_bounds__(LOSS_THREADS) void dist_finish_kernel(int n, const float *__restrict__ row_loss, const float *__restrict__ inv_rows,
                                                                   float *__restrict__ loss) {
    __shared__ double s_sum[LOSS_THREADS];
    double s = 0.;
    for (int i = threadIdx.x; i < n; i += LOSS_THREADS) s += row_loss[i];
    s_sum[threadIdx.x] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < LOSS_THREADS; ++i) s += s_sum[i];
        *loss = (float)(s * (double)*inv_rows);
    }
}

constexpr int LOSS_GRID = 512;
inline int loss_grid(int n) { return n < LOSS_GRID ? (n > 0 ? n : 1) : LOSS_GRID; }

int balance_check(const char *what, int n, int e, const void *logits, long long row_stride, int dtype) {
    const std::string w(what);
    GDPSO_REQUIRE(n >= 0 && e > 0, w + ": n >= 0 and e > 0 are required");
    GDPSO_REQUIRE(e <= BAL_MAX_E, w + ": more than 16384 experts");
    GDPSO_REQUIRE(dtype_ok(dtype), w + ": unknown element type");
    GDPSO_REQUIRE(n == 0 || logits, w + ": null argument");
    GDPSO_REQUIRE(row_stride >= 0, w + ": negative row stride");
    return GDPSO_OK;
}

}  // namespace
}  // namespace gdpso

using namespace gdpso;

extern "C" size_t gdpso_balance_workspace_bytes(int n, int e) {
    if (n < 0 || e <= 0) return 0;
    return (size_t)loss_grid(n) * e * sizeof(float);
}

extern "C" int gdpso_balance(void *stream_, int n, int e, int k, const void *logits, long long row_stride, int dtype, const void *indices,
                             int index_bytes, const unsigned char *mask, float grad_scale, float *loss, long long *counts, float *mean_prob,
                             void *grad, void *workspace, size_t workspace_bytes) {
    int rc = balance_check("balance", n, e, logits, row_stride, dtype);
    if (rc) return rc;
    GDPSO_REQUIRE(k > 0, "balance: k > 0 is required");
    GDPSO_REQUIRE(index_bytes == 4 || index_bytes == 8, "balance: indices are 4 or 8 bytes");
    GDPSO_REQUIRE((n == 0 || indices) && loss && counts && mean_prob && workspace, "balance: null argument");
    if (workspace_bytes < gdpso_balance_workspace_bytes(n, e)) return fail(GDPSO_ERR_WORKSPACE, "balance: workspace too small");
    hipStream_t stream = (hipStream_t)stream_;
    const ExpScale sc = exp_scale(1.);
    const int g = loss_grid(n);
    float *part = (float *)workspace;
    hipLaunchKernelGGL(fill_zero_kernel, dim3(ceil_div(e + 2, LOSS_THREADS)), dim3(LOSS_THREADS), 0, stream, counts, e + 2);
    hipLaunchKernelGGL(bal_count_kernel, dim3(ceil_div(n, LOSS_THREADS) < 256 ? ceil_div(n, LOSS_THREADS) + 1 : 256), dim3(LOSS_THREADS), 0, stream, n,
                       e, k, indices, index_bytes, mask, (unsigned long long *)counts);
    const size_t lds = (size_t)e * sizeof(float);
    if (grad)
        GDPSO_WITH_DTYPE(dtype, hipLaunchKernelGGL((bal_rows_kernel<E, true, true>), dim3(g), dim3(LOSS_THREADS), lds, stream, n, e, (const E *)logits,
                                                   row_stride, mask, counts, grad_scale, (const float *)nullptr, part, (E *)grad, sc));
    else
        GDPSO_WITH_DTYPE(dtype, hipLaunchKernelGGL((bal_rows_kernel<E, true, false>), dim3(g), dim3(LOSS_THREADS), lds, stream, n, e, (const E *)logits,
                                                   row_stride, mask, counts, 0.f, (const float *)nullptr, part, (E *)nullptr, sc));
    hipLaunchKernelGGL(bal_finish_kernel, dim3(1), dim3(LOSS_THREADS), 0, stream, e, g, part, counts, mean_prob, loss);
    GDPSO_HIP(hipGetLastError());
    return GDPSO_OK;
}

extern "C" int gdpso_balance_grad(void *stream_, int n, int e, const void *logits, long long row_stride, int dtype, const unsigned char *mask,
                                  const long long *counts, const float *upstream, void *grad) {
    int rc = balance_check("balance_grad", n, e, logits, row_stride, dtype);
    if (rc) return rc;
    GDPSO_REQUIRE(n == 0 || (counts && upstream && grad), "balance_grad: null argument");
    if (n == 0) return GDPSO_OK;
    hipStream_t stream = (hipStream_t)stream_;
    GDPSO_WITH_DTYPE(dtype, hipLaunchKernelGGL((bal_rows_kernel<E, false, true>), dim3(loss_grid(n)), dim3(LOSS_THREADS), 0, stream, n, e,
                                               (const E *)logits, row_stride, mask, counts, 0.f, upstream, (float *)nullptr, (E *)grad, exp_scale(1.)));
    GDPSO_HIP(hipGetLastError());
    return GDPSO_OK;
}

namespace gdpso {
namespace {
int distill_check(const char *what, int n, int v, int k, const void *logits, long long row_stride, int dtype, const void *t_logits, int t_dtype,
                  const void *t_idx, int index_bytes, float temperature) {
    const std::string w(what);
    GDPSO_REQUIRE(n >= 0 && v > 0 && k > 0, w + ": n >= 0, v > 0 and k > 0 are required");
    GDPSO_REQUIRE(k <= DIST_MAX_K, w + ": more than 1024 teacher logits a row");
    GDPSO_REQUIRE(dtype_ok(dtype) && dtype_ok(t_dtype), w + ": unknown element type");
    GDPSO_REQUIRE(index_bytes == 4 || index_bytes == 8, w + ": indices are 4 or 8 bytes");
    GDPSO_REQUIRE(temperature > 0.f && temperature <= 1e6f && temperature >= 1e-6f, w + ": temperature must lie in [1e-6, 1e6]");
    GDPSO_REQUIRE(n == 0 || (logits && t_logits && t_idx), w + ": null argument");
    GDPSO_REQUIRE(row_stride >= 0, w + ": negative row stride");
    return GDPSO_OK;
}
}  // namespace
}  // namespace gdpso

extern "C" size_t gdpso_distill_workspace_bytes(int n, int v, int k) { return 0; }

extern "C" int gdpso_distill(void *stream_, int n, int v, int k, const void *logits, long long row_stride, int dtype, const void *t_logits, int t_dtype,
                             const void *t_indices, int index_bytes, const unsigned char *mask, float temperature, float grad_scale, float *loss,
                             float *row_loss, float *row_stats, void *grad, void *workspace, size_t workspace_bytes) {
    int rc = distill_check("distill", n, v, k, logits, row_stride, dtype, t_logits, t_dtype, t_indices, index_bytes, temperature);
    if (rc) return rc;
    GDPSO_REQUIRE(loss && row_stats && (n == 0 || row_loss), "distill: null argument");
    if (workspace_bytes < gdpso_distill_workspace_bytes(n, v, k)) return fail(GDPSO_ERR_WORKSPACE, "distill: workspace too small");
    hipStream_t stream = (hipStream_t)stream_;
    const ExpScale sc = exp_scale(temperature);
    float *inv_rows = row_stats + 2 * (size_t)n;
    hipLaunchKernelGGL(dist_rows_kept_kernel, dim3(1), dim3(LOSS_THREADS), 0, stream, n, mask, inv_rows);
    const int g = n < 8192 ? (n > 0 ? n : 1) : 8192;
    if (grad)
        GDPSO_WITH_DTYPE(dtype, hipLaunchKernelGGL((dist_rows_kernel<E, true, true>), dim3(g), dim3(LOSS_THREADS), 0, stream, n, v, k, (const E *)logits,
                                                   row_stride, t_logits, t_dtype, t_indices, index_bytes, mask, temperature, sc, grad_scale,
                                                   (const float *)nullptr, row_stats, inv_rows, row_loss, (E *)grad));
    else
        GDPSO_WITH_DTYPE(dtype, hipLaunchKernelGGL((dist_rows_kernel<E, true, false>), dim3(g), dim3(LOSS_THREADS), 0, stream, n, v, k, (const E *)logits,
                                                   row_stride, t_logits, t_dtype, t_indices, index_bytes, mask, temperature, sc, 0.f,
                                                   (const float *)nullptr, row_stats, inv_rows, row_loss, (E *)nullptr));
    hipLaunchKernelGGL(dist_finish_kernel, dim3(1), dim3(LOSS_THREADS), 0, stream, n, row_loss, inv_rows, loss);
    GDPSO_HIP(hipGetLastError());
    return GDPSO_OK;
}

extern "C" int gdpso_distill_grad(void *stream_, int n, int v, int k, const void *logits, long long row_stride, int dtype, const void *t_logits,
                                  int t_dtype, const void *t_indices, int index_bytes, const unsigned char *mask, float temperature,
                                  const float *row_stats, const float *upstream, void *grad) {
    int rc = distill_check("distill_grad", n, v, k, logits, row_stride, dtype, t_logits, t_dtype, t_indices, index_bytes, temperature);
    if (rc) return rc;
    GDPSO_REQUIRE(n == 0 || (row_stats && upstream && grad), "distill_grad: null argument");
    if (n == 0) return GDPSO_OK;
    const int g = n < 8192 ? n : 8192;
    GDPSO_WITH_DTYPE(dtype, hipLaunchKernelGGL((dist_rows_kernel<E, false, true>), dim3(g), dim3(LOSS_THREADS), 0, (hipStream_t)stream_, n, v, k,
                                               (const E *)logits, row_stride, t_logits, t_dtype, t_indices, index_bytes, mask, temperature,
                                               exp_scale(temperature), 0.f, upstream, (float *)row_stats, row_stats + 2 * (size_t)n, (float *)nullptr,
                                               (E *)grad));
    GDPSO_HIP(hipGetLastError());
    return GDPSO_OK;
}
