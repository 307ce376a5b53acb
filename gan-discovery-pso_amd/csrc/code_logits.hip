// Logits of a soft assignment of latents to codes and their gradients, the differentiable counterpart of the
// nearest-code search (row i, code c, temperature t):
//
//   s[i,c]    = (2 <x_i, code_c> - |code_c|^2) / t     (minus the squared distance over t, less the row's constant |x_i|^2)
//   d x_i     = (2 / t) sum_c g[i,c] code_c
//   d code_c  = (2 / t) (sum_i g[i,c] x_i - code_c sum_i g[i,c])
//
// Three products; the logits and their gradient are fp32 whatever the type of latents and codes, and so is every sum.
//
// The products run on the 16-bit matrix instructions, sixteen times the rate of the fp32 ones, without giving up
// fp32 accuracy: a value is cut into bf16 parts, each the rounded rest of the one before, so that an fp32 value is three
// parts (3 x 8 bits), an fp16 value two, a bf16 value itself, and the product of two values is the sum of the products of
// their parts.  Those of order 2^-24 and below are left out (two middle parts of order 2^-16 are kept): six matrix
// instructions for fp32 x fp32, five for fp32 x fp16, three for fp32 x bf16.  Parts multiply exactly and add up in fp32.  The
// forward product of two 16-bit operands needs no cutting.
#include "loss_rows.h"

namespace gdpso {
namespace {

constexpr int CL_MAX_D = 4096;
constexpr int CL_THREADS = 256;  // four waves, one below the other over the output tile's rows
constexpr int KT = 32;           // summed elements a stage: one 16x16x32 matrix instruction deep
// LDS elements from one row of a stage to the next: 80 bytes put the sixteen rows of a fragment read on disjoint banks
constexpr int LROW = KT + 8;

using bf16x8 = __attribute__((ext_vector_type(8))) bf16_t;
using f16x8 = __attribute__((ext_vector_type(8))) f16_t;
template <typename M>
using Frag = __attribute__((ext_vector_type(8))) M;

// Cuts eight values into P parts of type M: parts[p] is the rounded rest of what the parts before it leave.
template <int P, typename M, typename E>
__device__ __forceinline__ void cut(const E (&v)[8], Frag<M> (&parts)[P]) {
    if constexpr (__is_same(E, M) && P == 1) {
#pragma unroll
        for (int e = 0; e < 8; ++e) parts[0][e] = v[e];
    } else {
        float rest[8], most = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            rest[e] = (float)v[e];
            most = fmaxf(most, fabsf(rest[e]));
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
#pragma unroll
            for (int e = 0; e < 8; ++e) parts[p][e] = (M)rest[e];
            if (p + 1 < P)
#pragma unroll
                for (int e = 0; e < 8; ++e) rest[e] -= (float)parts[p][e];
        }
        if (P > 1 && most > 3.3895e38f) {  // an infinite first part (inf, or rounded up to it) has no rest: inf - inf made it NaN
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (__builtin_isinf((float)parts[0][e]))
#pragma unroll
                    for (int p = 1; p < P; ++p) parts[p][e] = (M)0.f;
        }
    }
}

enum Product { LOGITS, GRAD_X, GRAD_CODE };

// The operand on the output rows' side.  Every wave has rows of its own, so its fragments come straight from global
// memory into registers, a stage ahead, and no value passes through LDS.  KC: the summed side is contiguous, a lane reads
// its eight values of a row in one piece; else the rows' side is, and a lane reads MT neighbouring rows at eight summed
// indices (tile t of the wave then holds rows t, MT + t, 2 MT + t ...).
template <typename E, bool KC, int MT, int P, typename M>
struct RowsOperand {
    E v[MT][8];

    __device__ __forceinline__ static long row(long wave_row0, int i, int fr) { return KC ? wave_row0 + i * 16 + fr : wave_row0 + fr * MT + i; }
    // values [k, kend) of this lane's rows; indices beyond read as 0, rows beyond as the last one (KC) or 0: nothing uses them
    __device__ __forceinline__ void load(const E *__restrict__ p, long ld, long wave_row0, long rows, int fr, long k, long kend) {
        if constexpr (KC) {
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const E *q = p + min(row(wave_row0, i, fr), rows - 1) * ld + k;
                if (k + 8 <= kend) {
                    constexpr int W = 16 / sizeof(E);
#pragma unroll
                    for (int w = 0; w < 8 / W; ++w) {
                        const auto x = *(const typename VecAt<E, W>::type *)(q + w * W);
#pragma unroll
                        for (int e = 0; e < W; ++e) v[i][w * W + e] = x[e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[i][e] = k + e < kend ? q[e] : (E)0.f;
                }
            }
        } else {
            const long r = row(wave_row0, 0, fr);
            const E *q = p + k * ld + r;
            if (r + MT <= rows && k + 8 <= kend) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const auto x = *(const typename VecAt<E, MT>::type *)(q + e * ld);
#pragma unroll
                    for (int i = 0; i < MT; ++i) v[i][e] = x[i];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
#pragma unroll
                    for (int i = 0; i < MT; ++i) v[i][e] = r + i < rows && k + e < kend ? q[e * ld + i] : (E)0.f;
            }
        }
    }
};

// The operand on the output columns' side, shared by the waves: BN columns by KT of the summed side per stage, through
// registers (a stage ahead) into P planes of parts in LDS, [P][BN][LROW].  KC: the summed side is contiguous in
// memory; else the columns' side is, and the eight values of a fragment are gathered from eight rows by one thread.
template <typename E, bool KC, int BN, int P, typename M>
struct ColsOperand {
    static constexpr int CW = KC ? 1 : (BN * 4 > CL_THREADS ? BN * 4 / CL_THREADS : 1);  // columns a unit
    static constexpr int UNITS = BN * 4 / CW;
    static constexpr int NU = (UNITS + CL_THREADS - 1) / CL_THREADS;
    E v[NU][CW][8];

    __device__ __forceinline__ static bool unit(int i, int &col, int &kc) {
        const int u = threadIdx.x + i * CL_THREADS;
        if constexpr (KC) {
            col = u >> 2;
            kc = u & 3;
        } else {
            col = u % (BN / CW) * CW;
            kc = u / (BN / CW);
        }
        return UNITS % CL_THREADS == 0 || u < UNITS;
    }
    // columns [col0, cols) and summed indices [k0, kend) of p, what lies beyond reads as 0
    __device__ __forceinline__ void load(const E *__restrict__ p, long ld, long col0, long cols, long k0, long kend) {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            int c0, kc;
            if (!unit(i, c0, kc)) continue;
            const long col = col0 + c0, k = k0 + kc * 8;
            if constexpr (KC) {
                const E *q = p + col * ld + k;
                if (col < cols && k + 8 <= kend) {
                    constexpr int W = 16 / sizeof(E);
#pragma unroll
                    for (int w = 0; w < 8 / W; ++w) {
                        const auto x = *(const typename VecAt<E, W>::type *)(q + w * W);
#pragma unroll
                        for (int e = 0; e < W; ++e) v[i][0][w * W + e] = x[e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[i][0][e] = col < cols && k + e < kend ? q[e] : (E)0.f;
                }
            } else {
                const E *q = p + k * ld + col;
                if (col + CW <= cols && k + 8 <= kend) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const auto x = *(const typename VecAt<E, CW>::type *)(q + e * ld);
#pragma unroll
                        for (int c = 0; c < CW; ++c) v[i][c][e] = x[c];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
#pragma unroll
                        for (int c = 0; c < CW; ++c) v[i][c][e] = col + c < cols && k + e < kend ? q[e * ld + c] : (E)0.f;
                }
            }
        }
    }
    __device__ __forceinline__ void add_squares(float (&sums)[NU]) const {
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) sums[i] = fmaf((float)v[i][0][e], (float)v[i][0][e], sums[i]);
    }
    __device__ __forceinline__ void store(M *lds) const {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            int c0, kc;
            if (!unit(i, c0, kc)) continue;
#pragma unroll
            for (int c = 0; c < CW; ++c) {
                Frag<M> parts[P];
                cut<P, M>(v[i][c], parts);
#pragma unroll
                for (int p = 0; p < P; ++p) *(Frag<M> *)(lds + (p * BN + c0 + c) * LROW + kc * 8) = parts[p];
            }
        }
    }
};

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

struct ProductArgs {
    const void *m, *n;  // operands: output rows' side and output columns' side
    void *out;          // LOGITS, GRAD_X: result; GRAD_CODE: partial sums [split][rows * cols + rows]
    long rows, cols, sum;
    long ld_m, ld_n;
    int tiles_m, tiles_n, splits;
    long sum_per_split;  // a multiple of KT
    float scale;
};

// An output tile of 64 MT x 16 NT a workgroup: each wave 16 MT rows of it and all its columns.
template <Product OP, typename EM, typename EN, int PM, int PN, typename M, int MT, int NT, typename EO>
__global__ __launch_bounds__(CL_THREADS) void product_kernel(ProductArgs a) {
    constexpr bool KC_M = OP != GRAD_CODE, KC_N = OP == LOGITS;
    constexpr int BN = NT * 16;
    using OpM = RowsOperand<EM, KC_M, MT, PM, M>;
    using OpN = ColsOperand<EN, KC_N, BN, PN, M>;
    __shared__ __attribute__((aligned(16))) M s_n[2][PN][BN][LROW];
    __shared__ float s_norm[OP == LOGITS ? BN : 1];
    // Workgroups b and b + 8 run on one XCD: the tiles that share rows (GRAD_CODE: a split) go to the same one, whose L2
    // then serves the shared operand once.
    const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
    int tm, tn, split;
    if constexpr (OP == GRAD_CODE) {
        const int per = a.tiles_m * a.tiles_n;
        split = slot / per * 8 + xcd;
        tm = slot % per % a.tiles_m;
        tn = slot % per / a.tiles_m;
        if (split >= a.splits) return;
    } else {
        split = 0;
        tm = slot / a.tiles_n * 8 + xcd;
        tn = slot % a.tiles_n;
        if (tm >= a.tiles_m) return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long m0 = ((long)tm * 4 + wave) * (MT * 16), n0 = (long)tn * BN;
    const long k0 = split * a.sum_per_split, kend = min(k0 + a.sum_per_split, a.sum);
    const int fr = lane & 15, fk = (lane >> 4) * 8;  // this lane's row and first summed element of a fragment

    OpM om;
    OpN on;
    float sq[OpN::NU] = {}, sum_m[MT] = {};
    f32x4 acc[MT][NT] = {};
    om.load((const EM *)a.m, a.ld_m, m0, a.rows, fr, k0 + fk, kend);
    on.load((const EN *)a.n, a.ld_n, n0, a.cols, k0, kend);
    on.store(&s_n[0][0][0][0]);
    if constexpr (OP == LOGITS) on.add_squares(sq);
    int buf = 0;
    for (long k = k0; k < kend; k += KT, buf ^= 1) {
        Frag<M> fm[MT][PM];
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            if constexpr (OP == GRAD_CODE)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum_m[i] += (float)om.v[i][e];
            cut<PM, M>(om.v[i], fm[i]);
        }
        const bool more = k + KT < kend;
        if (more) {
            om.load((const EM *)a.m, a.ld_m, m0, a.rows, fr, k + KT + fk, kend);
            on.load((const EN *)a.n, a.ld_n, n0, a.cols, k + KT, kend);
        }
        // The barrier orders this stage's plane after its stores and the other plane's next stores after its last reads.
        __syncthreads();
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            Frag<M> fn[PN];
#pragma unroll
            for (int p = 0; p < PN; ++p) fn[p] = *(const Frag<M> *)&s_n[buf][p][j * 16 + fr][fk];
            // the small products first
#pragma unroll
            for (int order = 2; order >= 0; --order)
#pragma unroll
                for (int p = 0; p < PM; ++p) {
                    const int q = order - p;
                    if (q < 0 || q >= PN) continue;
#pragma unroll
                    for (int i = 0; i < MT; ++i) acc[i][j] = mfma(fn[q], fm[i][p], acc[i][j]);
                }
        }
        if (more) {
            on.store(&s_n[buf ^ 1][0][0][0]);
            if constexpr (OP == LOGITS) on.add_squares(sq);
        }
    }

    if constexpr (OP == LOGITS) {  // |code|^2: four neighbouring threads hold a row's chunks
#pragma unroll
        for (int i = 0; i < OpN::NU; ++i) {
            int c, kc;
            if (!OpN::unit(i, c, kc)) continue;
            float s = sq[i];
            s += __shfl_xor(s, 1, 64);
            s += __shfl_xor(s, 2, 64);
            if (kc == 0) s_norm[c] = s;
        }
        __syncthreads();
    }
    if constexpr (OP == GRAD_CODE) {
        if (tn == 0) {
            float *p = (float *)a.out + split * (a.rows * a.cols + a.rows) + a.rows * a.cols;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                float s = sum_m[i];
                s += __shfl_xor(s, 16, 64);
                s += __shfl_xor(s, 32, 64);
                const long m = OpM::row(m0, i, fr);
                if (lane < 16 && m < a.rows) p[m] = s;
            }
        }
    }
    // A lane holds four consecutive columns of one row of each 16 x 16 tile.
    EO *out = (EO *)a.out + (OP == GRAD_CODE ? split * (a.rows * a.cols + a.rows) : 0);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const long m = OpM::row(m0, i, fr);
        if (m >= a.rows) continue;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int nl = j * 16 + (lane >> 4) * 4;
            const long n = n0 + nl;
            EO *dst = out + m * a.cols + n;
            typename VecAt<EO, 4>::type r;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x = acc[i][j][e];
                if constexpr (OP == LOGITS) x = fmaf(2.f, x, -s_norm[nl + e]) * a.scale;
                if constexpr (OP == GRAD_X) x *= a.scale;
                r[e] = (EO)x;
            }
            if (n + 4 <= a.cols) *(typename VecAt<EO, 4>::type *)dst = r;
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < a.cols) dst[e] = r[e];
        }
    }
}

// Joins the splits' partial sums in a fixed order: 64 neighbouring elements a workgroup, the splits dealt to its waves.
constexpr int JOIN_WAVES = 8;
template <typename E>
__global__ __launch_bounds__(64 * JOIN_WAVES) void code_join_kernel(int d, int k, int splits, const float *__restrict__ part, const E *__restrict__ cb,
                                                                    float scale, E *__restrict__ dcode) {
    __shared__ float s_acc[JOIN_WAVES][64], s_sum[JOIN_WAVES][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long size = (long)k * d, e = (long)blockIdx.x * 64 + lane;
    float acc = 0.f, sum = 0.f;
    if (e < size) {
        const float *p = part + e, *ps = part + size + e / d;
#pragma unroll 4
        for (int s = wave; s < splits; s += JOIN_WAVES) {
            acc += p[s * (size + k)];
            sum += ps[s * (size + k)];
        }
    }
    s_acc[wave][lane] = acc;
    s_sum[wave][lane] = sum;
    __syncthreads();
    if (wave == 0 && e < size) {
        for (int w = 1; w < JOIN_WAVES; ++w) {
            acc += s_acc[w][lane];
            sum += s_sum[w][lane];
        }
        dcode[e] = (E)(scale * fmaf(-sum, (float)cb[e], acc));
    }
}

// Output tile: the largest that still gives every CU a workgroup; a side of at most 64 takes 64.
constexpr int CL_WANT = 256;
struct Tile {
    int m, n;
};
inline Tile pick_tile(long rows, long cols, long splits) {
    const Tile tiles[] = {{128, 128}, {128, 64}, {64, 64}};
    for (const Tile &t : tiles) {
        if (t.n == 128 && cols <= 64) continue;
        if ((long)ceil_div(rows, t.m) * ceil_div(cols, t.n) * splits >= CL_WANT) return t;
    }
    return {64, 32};
}

// Splits of the summed rows of the codebook's gradient: about two workgroups of 128 x 128 or 128 x 64 per CU, at least
// 128 rows a split (the partial sums a split writes and the join reads have to stay small beside its rows).
inline int code_splits(int n, int d, int k) {
    if (n <= 0) return 0;
    const long tiles = (long)ceil_div(k, 128) * ceil_div(d, d <= 64 ? 64 : 128);
    const long want = ceil_div(512, tiles), most = ceil_div(n, 128);
    return (int)(want < most ? want : most);
}

template <Product OP, typename EM, typename EN, int PM, int PN, typename M, typename EO>
int launch_product(hipStream_t stream, ProductArgs a) {
    const Tile t = pick_tile(a.rows, a.cols, a.splits);
    a.tiles_m = ceil_div(a.rows, t.m);
    a.tiles_n = ceil_div(a.cols, t.n);
    const long grid = OP == GRAD_CODE ? (long)ceil_div(a.splits, 8) * 8 * a.tiles_m * a.tiles_n : (long)ceil_div(a.tiles_m, 8) * 8 * a.tiles_n;
    GDPSO_REQUIRE(grid < (1l << 31), "code_logits: too many rows for one call");
#define CL_LAUNCH(MT, NT) hipLaunchKernelGGL((product_kernel<OP, EM, EN, PM, PN, M, MT, NT, EO>), dim3((unsigned)grid), dim3(CL_THREADS), 0, stream, a)
    if (t.n == 128) CL_LAUNCH(2, 8);
    else if (t.m == 128) CL_LAUNCH(2, 4);
    else if (t.n == 64) CL_LAUNCH(1, 4);
    else CL_LAUNCH(1, 2);
#undef CL_LAUNCH
    GDPSO_HIP(hipGetLastError());
    return GDPSO_OK;
}

template <typename E>
constexpr int grad_parts() {
    return is_f32<E>() ? 3 : (__is_same(E, f16_t) ? 2 : 1);
}

template <typename E>
int logits_product(hipStream_t stream, const ProductArgs &a) {
    if constexpr (is_f32<E>()) return launch_product<LOGITS, float, float, 3, 3, bf16_t, float>(stream, a);
    else return launch_product<LOGITS, E, E, 1, 1, E, float>(stream, a);
}

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
    ProductArgs a = {inputs, codebook, logits, n, k, d, d, d, 0, 0, 1, ceil_div(d, KT) * (long)KT, 1.f / temperature};
    GDPSO_WITH_DTYPE(dtype, rc = logits_product<E>((hipStream_t)stream_, a));
    return rc;
}

extern "C" size_t gdpso_code_logits_grad_workspace_bytes(int n, int d, int k) {
    if (n <= 0 || d <= 0 || k <= 0) return 0;
    return (size_t)code_splits(n, d, k) * k * (d + 1) * sizeof(float);
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
    if (grad_inputs && n > 0) {
        const ProductArgs a = {grad_logits, codebook, grad_inputs, n, d, k, k, d, 0, 0, 1, ceil_div(k, KT) * (long)KT, scale};
        GDPSO_WITH_DTYPE(dtype, rc = (launch_product<GRAD_X, float, E, 3, grad_parts<E>(), bf16_t, E>(stream, a)));
        if (rc) return rc;
    }
    if (grad_codebook) {
        const int splits = code_splits(n, d, k);
        if (splits) {
            const long per = ceil_div(ceil_div(n, splits), KT) * (long)KT;
            const ProductArgs a = {grad_logits, inputs, workspace, k, d, n, k, d, 0, 0, splits, per, 1.f};
            GDPSO_WITH_DTYPE(dtype, rc = (launch_product<GRAD_CODE, float, E, 3, grad_parts<E>(), bf16_t, float>(stream, a)));
            if (rc) return rc;
        }
        GDPSO_WITH_DTYPE(dtype, hipLaunchKernelGGL((code_join_kernel<E>), dim3(ceil_div((long)k * d, 64)), dim3(64 * JOIN_WAVES), 0, stream, d, k, splits,
                                                   (const float *)workspace, (const E *)codebook, scale, (E *)grad_codebook));
        GDPSO_HIP(hipGetLastError());
    }
    return GDPSO_OK;
}
