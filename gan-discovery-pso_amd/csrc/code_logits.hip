// Logits of a soft assignment of latents to codes and their gradients, the differentiable counterpart of the
// nearest-code search (row i, code c, temperature t):
//
//   s[i,c]    = (2 <x_i, code_c> - |code_c|^2) / t     (minus the squared distance over t, less the row's constant |x_i|^2)
//   d x_i     = (2 / t) sum_c g[i,c] code_c
//   d code_c  = (2 / t) (sum_i g[i,c] x_i - code_c sum_i g[i,c])
//
// Three products; the logits and their gradient are fp32 whatever the type of latents and codes, and so is every sum.
#include "common.h"

#include <math.h>

namespace gdpso {
namespace {

constexpr int T = 16;  // output tile of a workgroup of T x T threads
constexpr int CL_MAX_D = 4096;

template <typename E>
__global__ __launch_bounds__(T *T) void code_logits_kernel(int n, int d, int k, const E *__restrict__ x, const E *__restrict__ cb, float inv_t,
                                                           float *__restrict__ out) {
    __shared__ float s_x[T][T + 1], s_c[T][T + 1];
    const int tx = threadIdx.x % T, ty = threadIdx.x / T;
    const long i0 = (long)blockIdx.x * T;
    const int c0 = blockIdx.y * T;
    float acc = 0.f, sq = 0.f;
    for (int j0 = 0; j0 < d; j0 += T) {
        s_x[ty][tx] = i0 + ty < n && j0 + tx < d ? (float)x[(i0 + ty) * d + j0 + tx] : 0.f;
        s_c[ty][tx] = c0 + ty < k && j0 + tx < d ? (float)cb[(size_t)(c0 + ty) * d + j0 + tx] : 0.f;
        __syncthreads();
        for (int j = 0; j < T; ++j) {
            acc = fmaf(s_x[ty][j], s_c[tx][j], acc);
            sq = fmaf(s_c[tx][j], s_c[tx][j], sq);
        }
        __syncthreads();
    }
    if (i0 + ty < n && c0 + tx < k) out[(i0 + ty) * k + c0 + tx] = fmaf(2.f, acc, -sq) * inv_t;
}

template <typename E>
__global__ __launch_bounds__(T *T) void code_dx_kernel(int n, int d, int k, const float *__restrict__ g, const E *__restrict__ cb, float scale,
                                                       E *__restrict__ dx) {
    __shared__ float s_g[T][T + 1], s_c[T][T + 1];
    const int tx = threadIdx.x % T, ty = threadIdx.x / T;
    const long i0 = (long)blockIdx.x * T;
    const int j0 = blockIdx.y * T;
    float acc = 0.f;
    for (int c0 = 0; c0 < k; c0 += T) {
        s_g[ty][tx] = i0 + ty < n && c0 + tx < k ? g[(i0 + ty) * k + c0 + tx] : 0.f;
        s_c[ty][tx] = c0 + ty < k && j0 + tx < d ? (float)cb[(size_t)(c0 + ty) * d + j0 + tx] : 0.f;
        __syncthreads();
        for (int c = 0; c < T; ++c) acc = fmaf(s_g[ty][c], s_c[c][tx], acc);
        __syncthreads();
    }
    if (i0 + ty < n && j0 + tx < d) dx[(i0 + ty) * d + j0 + tx] = (E)(scale * acc);
}

// part[split][c][j] = sum of g[i,c] x[i,j] over the split's rows, part[split][k * d + c] = sum of g[i,c]
template <typename E>
__global__ __launch_bounds__(T *T) void code_dcode_kernel(int n, int d, int k, const float *__restrict__ g, const E *__restrict__ x, int rows_per_split,
                                                          float *__restrict__ part) {
    __shared__ float s_g[T][T + 1], s_x[T][T + 1];
    const int tx = threadIdx.x % T, ty = threadIdx.x / T;
    const int c0 = blockIdx.x * T, j0 = blockIdx.y * T;
    const long lo = (long)blockIdx.z * rows_per_split, hi = lo + rows_per_split < n ? lo + rows_per_split : n;
    float acc = 0.f, sum = 0.f;
    for (long i0 = lo; i0 < hi; i0 += T) {
        s_g[ty][tx] = i0 + ty < hi && c0 + tx < k ? g[(i0 + ty) * k + c0 + tx] : 0.f;
        s_x[ty][tx] = i0 + ty < hi && j0 + tx < d ? (float)x[(i0 + ty) * d + j0 + tx] : 0.f;
        __syncthreads();
        for (int i = 0; i < T; ++i) {
            acc = fmaf(s_g[i][ty], s_x[i][tx], acc);
            sum += s_g[i][ty];
        }
        __syncthreads();
    }
    float *p = part + (size_t)blockIdx.z * k * (d + 1);
    if (c0 + ty < k && j0 + tx < d) p[(size_t)(c0 + ty) * d + j0 + tx] = acc;
    if (c0 + ty < k && j0 + tx == 0) p[(size_t)k * d + c0 + ty] = sum;
}

template <typename E>
__global__ __launch_bounds__(256) void code_dcode_finish_kernel(int d, int k, int splits, const float *__restrict__ part, const E *__restrict__ cb,
                                                                float scale, E *__restrict__ dcode) {
    const long e = (long)blockIdx.x * 256 + threadIdx.x;
    if (e >= (long)k * d) return;
    const int c = (int)(e / d);
    float acc = 0.f, sum = 0.f;
    for (int s = 0; s < splits; ++s) {
        const float *p = part + (size_t)s * k * (d + 1);
        acc += p[e];
        sum += p[(size_t)k * d + c];
    }
    dcode[e] = (E)(scale * fmaf(-sum, (float)cb[e], acc));
}

constexpr int CL_SPLIT_ROWS = 1024;
inline int code_splits(int n) { return n > 0 ? ceil_div(n, CL_SPLIT_ROWS) : 0; }

int code_check(const char *what, int n, int d, int k, int dtype, float temperature) {
    const std::string w(what);
    GDPSO_REQUIRE(n >= 0 && k > 0 && d > 0, w + ": n >= 0, k > 0 and d > 0 are required");
    GDPSO_REQUIRE(d <= CL_MAX_D, w + ": embedding size above 4096");
    GDPSO_REQUIRE(k <= (1 << 20), w + ": more than 2^20 codes");
    GDPSO_REQUIRE(dtype_ok(dtype), w + ": unknown element type");
    GDPSO_REQUIRE(temperature >= 1e-6f && temperature <= 1e6f, w + ": temperature must lie in [1e-6, 1e6]");
    return GDPSO_OK;
}

}  // namespace
}  // namespace gdpso

using namespace gdpso;

extern "C" int gdpso_code_logits(void *stream_, int n, int d, int k, const void *inputs, const void *codebook, int dtype, float temperature,
                                 float *logits) {
    int rc = code_check("code_logits", n, d, k, dtype, temperature);
    if (rc) return rc;
    GDPSO_REQUIRE(n == 0 || (inputs && codebook && logits), "code_logits: null argument");
    if (n == 0) return GDPSO_OK;
    GDPSO_WITH_DTYPE(dtype, hipLaunchKernelGGL((code_logits_kernel<E>), dim3(ceil_div(n, T), ceil_div(k, T)), dim3(T * T), 0, (hipStream_t)stream_, n, d, k,
                                               (const E *)inputs, (const E *)codebook, 1.f / temperature, logits));
    GDPSO_HIP(hipGetLastError());
    return GDPSO_OK;
}

extern "C" size_t gdpso_code_logits_grad_workspace_bytes(int n, int d, int k) {
    if (n <= 0 || d <= 0 || k <= 0) return 0;
    return (size_t)code_splits(n) * k * (d + 1) * sizeof(float);
}

extern "C" int gdpso_code_logits_grad(void *stream_, int n, int d, int k, const float *grad_logits, const void *inputs, const void *codebook, int dtype,
                                      float temperature, void *grad_inputs, void *grad_codebook, void *workspace, size_t workspace_bytes) {
    int rc = code_check("code_logits_grad", n, d, k, dtype, temperature);
    if (rc) return rc;
    GDPSO_REQUIRE(n == 0 || (grad_logits && inputs), "code_logits_grad: null argument");
    GDPSO_REQUIRE(codebook, "code_logits_grad: null argument");
    GDPSO_REQUIRE(!grad_codebook || n == 0 || workspace, "code_logits_grad: null workspace");
    if (grad_codebook && workspace_bytes < gdpso_code_logits_grad_workspace_bytes(n, d, k))
        return fail(GDPSO_ERR_WORKSPACE, "code_logits_grad: workspace too small");
    hipStream_t stream = (hipStream_t)stream_;
    const float scale = 2.f / temperature;
    if (grad_inputs && n > 0)
        GDPSO_WITH_DTYPE(dtype, hipLaunchKernelGGL((code_dx_kernel<E>), dim3(ceil_div(n, T), ceil_div(d, T)), dim3(T * T), 0, stream, n, d, k, grad_logits,
                                                   (const E *)codebook, scale, (E *)grad_inputs));
    if (grad_codebook) {
        const int splits = code_splits(n);
        if (splits)
            GDPSO_WITH_DTYPE(dtype, hipLaunchKernelGGL((code_dcode_kernel<E>), dim3(ceil_div(k, T), ceil_div(d, T), splits), dim3(T * T), 0, stream, n, d, k,
                                                       grad_logits, (const E *)inputs, CL_SPLIT_ROWS, (float *)workspace));
        GDPSO_WITH_DTYPE(dtype, hipLaunchKernelGGL((code_dcode_finish_kernel<E>), dim3(ceil_div((long)k * d, 256)), dim3(256), 0, stream, d, k, splits,
                                                   (const float *)workspace, (const E *)codebook, scale, (E *)grad_codebook));
    }
    GDPSO_HIP(hipGetLastError());
    return GDPSO_OK;
}
