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
// their parts.  Those of order 2^-24 and below are left out: six matrix instructions for fp32 x fp32, five for fp32 x fp16,
// three for fp32 x bf16.  Parts multiply exactly and add up in fp32.  The forward product of two 16-bit operands needs no cutting.
//
// What bounds them: the fp32 logits or their gradient, [n, k], against which latents and codes are small, and with fp32 operands the
// matrix instructions as much.  Calls with inputs in rotation: latents 65536 x 64, 512 codes, fp32, logits 38 us (134 MB written, 3.6 TB/s,
// and 26 GFLOP of bf16 products), both gradients with their join 74 (the same 134 MB read for each, and 52 GFLOP).  50007 x 256 and 1024
// codes, bf16: logits 75 us (205 MB, 2.7 TB/s), gradients with planes and join 174 (2 x 205 MB and 157 GFLOP); fp16 77 and 274.
#include "loss_rows.h"

#include <algorithm>
#include <type_traits>

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

// p[off] for a pointer that is the same in the whole wave and a lane's offset in bytes: a scalar base and one register.
template <typename V, typename E>
__device__ __forceinline__ V at_bytes(const E *p, unsigned off) {
    return *(const V *)((const char *)p + off);
}

// Cuts a pair of values into P parts: words[p] holds the two p-th parts, the rounded rest of what the parts before leave.  One
// conversion instruction packs both.  BIG: values that the first part would round up to infinity have the largest bf16 for it, and an
// infinity is the last part alone.  A third part meets nothing but the other value's first one, which has its sign and is 0 only where
// the value is; a 16-bit type's infinity meets second parts too, and what comes out may be NaN.
template <int P, bool BIG>
__device__ __forceinline__ void cut_pair(float a, float b, unsigned (&words)[P]) {
    using f32x2 = __attribute__((ext_vector_type(2))) float;
    using bf16x2 = __attribute__((ext_vector_type(2))) bf16_t;
    constexpr float MOST = 3.38953139e38f;
    f32x2 rest = {a, b};
#pragma unroll
    for (int p = 0; p < P; ++p) {
        f32x2 x = rest;
        if (BIG && p == 0) {  // (a NaN stays one: comparisons with it are false)
            x[0] = fabsf(a) > MOST ? __builtin_copysignf(MOST, a) : a;
            x[1] = fabsf(b) > MOST ? __builtin_copysignf(MOST, b) : b;
        }
        words[p] = __builtin_bit_cast(unsigned, __builtin_convertvector(x, bf16x2));
        rest[0] -= __builtin_bit_cast(float, words[p] << 16);
        rest[1] -= __builtin_bit_cast(float, words[p] & 0xffff0000u);
    }
    if (BIG) {
        const unsigned low = fabsf(a) == INFINITY ? 0xffffu : 0u, high = fabsf(b) == INFINITY ? 0xffff0000u : 0u;
#pragma unroll
        for (int p = 0; p < P; ++p) words[p] &= ~(low | high);
        words[P - 1] |= (low & (__builtin_bit_cast(unsigned, a) >> 16)) | (high & __builtin_bit_cast(unsigned, b));
    }
}

// Cuts eight values into P parts of type M.
template <int P, typename M, typename E>
__device__ __forceinline__ void cut(const E (&v)[8], Frag<M> (&parts)[P]) {
    if constexpr (__is_same(E, M) && P == 1) {
#pragma unroll
        for (int e = 0; e < 8; ++e) parts[0][e] = v[e];
    } else {
        static_assert(__is_same(M, bf16_t), "parts are bf16");
        using u32x4 = __attribute__((ext_vector_type(4))) unsigned;
        u32x4 words[P];
        const auto all = [&](auto huge) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                unsigned pair[P];
                cut_pair<P, decltype(huge)::value>((float)v[2 * w], (float)v[2 * w + 1], pair);
#pragma unroll
                for (int p = 0; p < P; ++p) words[p][w] = pair[p];
            }
        };
        float most = 0.f;
        if (P > 1)
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, fabsf((float)v[e]));
        if (P > 1 && most > 3.3895e38f) all(std::true_type{});
        else all(std::false_type{});
#pragma unroll
        for (int p = 0; p < P; ++p) parts[p] = __builtin_bit_cast(Frag<M>, words[p]);
    }
}

enum Product { LOGITS, GRAD_X, GRAD_CODE };

// The operand on the output rows' side.  Every wave has rows of its own, so its fragments come straight from global
// memory into registers, a stage ahead, and no value passes through LDS.  KC: the summed side is contiguous, a lane reads
// its eight values of a row in one piece; else the rows' side is, and a lane reads MT neighbouring rows at eight summed
// indices (tile t of the wave then holds rows t, MT + t, 2 MT + t ...).
//
// Loads have one form for every position, without a branch, and what they return stays as it came until it is cut: only then
// does the compiler leave later stages' loads on the way while it waits for this one's.  Rows beyond the matrix are
// clamped into it; a vector of MT rows is clamped as a whole and may so begin before the lane's first row (shift()).
template <typename E, bool KC, int MT, int P, typename M>
struct RowsOperand {
    static constexpr int W = KC ? 16 / (int)sizeof(E) : MT;      // elements a load
    static constexpr int LOADS = KC ? MT * (8 / W) : 8;
    static constexpr int ROWS = KC ? 1 : MT;                     // fewest rows of the matrix
    typename VecAt<E, W>::type raw[LOADS];

    __device__ __forceinline__ static long row(long wave_row0, int i, int fr) { return KC ? wave_row0 + i * 16 + fr : wave_row0 + fr * MT + i; }
    __device__ __forceinline__ static long clamped(long r, long rows) { return min(r, rows - ROWS); }
    // The row that value i of this lane belongs to, and whether it is this lane's to write.
    __device__ __forceinline__ static long held(long wave_row0, long rows, int i, int fr, bool &mine) {
        const long r = row(wave_row0, i, fr);
        if constexpr (KC) {
            mine = r < rows;
            return r;
        } else {
            const long first = row(wave_row0, 0, fr), h = clamped(first, rows) + i;
            mine = h >= first;
            return h;
        }
    }
    __device__ __forceinline__ static long first_row(long wave_row0, long rows) { return clamped(wave_row0, rows); }
    // Byte offsets of this lane's loads from the wave's first row at a stage's first summed element.
    __device__ __forceinline__ static void offsets(long ld, long wave_row0, long rows, int fr, int fk, unsigned (&off)[KC ? MT : 1]) {
#pragma unroll
        for (int i = 0; i < (KC ? MT : 1); ++i) {
            const long r = clamped(row(wave_row0, i, fr), rows) - first_row(wave_row0, rows);
            off[i] = (unsigned)((KC ? r * ld + fk : fk * ld + r) * (long)sizeof(E));
        }
    }
    __device__ __forceinline__ void load_whole(const E *__restrict__ stage, long ld, const unsigned (&off)[KC ? MT : 1]) {
#pragma unroll
        for (int l = 0; l < LOADS; ++l) {
            if constexpr (KC) raw[l] = at_bytes<typename VecAt<E, W>::type>(stage + l % (8 / W) * W, off[l / (8 / W)]);
            else raw[l] = at_bytes<typename VecAt<E, W>::type>(stage + l * ld, off[0]);
        }
    }
    // The stage that the sum's end cuts: `left` elements of it are there, the others read as 0.
    __device__ __forceinline__ void load_part(const E *__restrict__ stage, long ld, const unsigned (&off)[KC ? MT : 1], int fk, int left) {
#pragma unroll
        for (int l = 0; l < LOADS; ++l)
#pragma unroll
            for (int w = 0; w < (KC ? W : 1); ++w) {
                const int e = KC ? l % (8 / W) * W + w : l;
                const int back = max(0, fk + e - (left - 1));  // elements beyond the last one that is there
                if constexpr (KC) {
                    const E x = at_bytes<E>(stage, (unsigned)(off[l / (8 / W)] + ((long)e - back) * (long)sizeof(E)));
                    raw[l][w] = back == 0 ? x : (E)0.f;
                } else {
                    const auto x = at_bytes<typename VecAt<E, W>::type>(stage, (unsigned)(off[0] + ((long)e - back) * ld * (long)sizeof(E)));
#pragma unroll
                    for (int c = 0; c < W; ++c) raw[l][c] = back == 0 ? x[c] : (E)0.f;
                }
            }
    }
    // the eight values of row i
    __device__ __forceinline__ void values(int i, E (&v)[8]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = KC ? raw[i * (8 / W) + e / W][e % W] : raw[e][i];
    }
};

// The operand on the output columns' side, shared by the waves: BN columns by KT of the summed side per stage, through
// registers (a stage ahead) into P planes of parts in LDS, [P][PLANE][LROW].  KC: the summed side is contiguous in
// memory; else the columns' side is, and the eight values of a fragment are gathered from eight rows by one thread, CW
// neighbouring columns at a time.  Loads as RowsOperand's: columns beyond the matrix are clamped into it, a vector of CW
// as a whole, and land in LDS where they belong (what belongs to no column of the matrix is never used).
template <typename E, bool KC, int BN, int P, typename M>
struct ColsOperand {
    static constexpr int CW = KC ? 1 : (BN * 4 > CL_THREADS ? BN * 4 / CL_THREADS : 1);  // columns a unit
    static constexpr int UNITS = BN * 4 / CW;
    static constexpr int NU = (UNITS + CL_THREADS - 1) / CL_THREADS;
    static constexpr int W = KC ? 16 / (int)sizeof(E) : CW, LOADS = KC ? 8 / W : 8;
    static constexpr int AHEAD = CW > 1 ? CW : 0;  // rows of a plane ahead of the tile's columns, for vectors that begin before it
    static constexpr int PLANE = BN + AHEAD;       // rows of a plane
    typename VecAt<E, W>::type raw[NU][LOADS];

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
    // Columns from the tile's first one to the first one that unit i holds: a clamped vector may begin before the tile.
    __device__ __forceinline__ static int base(long col0, long cols, int i, int &kc) {
        int c0;
        unit(i, c0, kc);
        kc &= 3;
        return (int)(min(col0 + c0, cols - CW) - col0);
    }
    // The column that a stage's address and the offsets count from.
    __device__ __forceinline__ static long origin(long col0) { return CW == 1 ? col0 : max(col0 - CW, 0l); }
    __device__ __forceinline__ static void offsets(long ld, long col0, long cols, unsigned (&off)[NU]) {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            int kc;
            const long col = base(col0, cols, i, kc) + col0 - origin(col0);
            off[i] = (unsigned)((KC ? col * ld + kc * 8 : kc * 8 * ld + col) * (long)sizeof(E));
        }
    }
    __device__ __forceinline__ void load_whole(const E *__restrict__ stage, long ld, const unsigned (&off)[NU]) {
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int l = 0; l < LOADS; ++l) raw[i][l] = at_bytes<typename VecAt<E, W>::type>(KC ? stage + l * W : stage + l * ld, off[i]);
    }
    __device__ __forceinline__ void load_part(const E *__restrict__ stage, long ld, const unsigned (&off)[NU], int left) {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            int c0, kc;
            unit(i, c0, kc);
#pragma unroll
            for (int l = 0; l < LOADS; ++l)
#pragma unroll
                for (int w = 0; w < (KC ? W : 1); ++w) {
                    const int e = KC ? l * W + w : l;
                    const int back = max(0, (kc & 3) * 8 + e - (left - 1));
                    const unsigned at = (unsigned)(off[i] + ((long)e - back) * (KC ? 1 : ld) * (long)sizeof(E));
                    if constexpr (KC) {
                        const E x = at_bytes<E>(stage, at);
                        raw[i][l][w] = back == 0 ? x : (E)0.f;
                    } else {
                        const auto x = at_bytes<typename VecAt<E, W>::type>(stage, at);
#pragma unroll
                        for (int c = 0; c < W; ++c) raw[i][l][c] = back == 0 ? x[c] : (E)0.f;
                    }
                }
        }
    }
    __device__ __forceinline__ E value(int i, int c, int e) const { return KC ? raw[i][e / W][e % W] : raw[i][e][c]; }
    __device__ __forceinline__ void add_squares(float (&sums)[NU]) const {
        using E2 = __attribute__((ext_vector_type(2))) E;
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const E2 x = {value(i, 0, e), value(i, 0, e + 1)};
                if constexpr (is_f32<E>()) sums[i] = fmaf(x[1], x[1], fmaf(x[0], x[0], sums[i]));
                else if constexpr (__is_same(E, bf16_t)) sums[i] = __builtin_amdgcn_fdot2_f32_bf16(x, x, sums[i], false);
                else sums[i] = __builtin_amdgcn_fdot2(x, x, sums[i], false);
            }
    }
    __device__ __forceinline__ void store(M *lds, long col0, long cols) const {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            int c0, kc;
            if (!unit(i, c0, kc)) continue;
            const int row = AHEAD + (CW == 1 ? c0 : base(col0, cols, i, kc));
#pragma unroll
            for (int c = 0; c < CW; ++c) {
                E v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = value(i, c, e);
                Frag<M> parts[P];
                cut<P, M>(v, parts);
#pragma unroll
                for (int p = 0; p < P; ++p) *(Frag<M> *)(lds + (p * PLANE + row + c) * LROW + kc * 8) = parts[p];
            }
        }
    }
};

// The same for the gradients of 16-bit codes and latents, from planes that planes_kernel has cut and transposed: P planes of bf16, each
// [pitch / KT][cols][KT] with `pitch` the sum's length rounded up to whole stages, zeros behind its end.  A stage passes
// through registers as it is, where gathering takes every workgroup eight loads of two bytes a value pair and the cut (a call, gathering
// and from planes with their launch: bf16, 20000 x 2048 x 256 171 and 157 us, 50007 x 1024 x 256 177 and 174; fp16, whose tile of 256
// columns would leave one wave a SIMD, 374 and 231, 411 and 271; up to 128 columns there is little between them, 50007 x 512 x 128 70 and
// 72, fp16 65536 x 512 x 64 61 and 67).  With fp32 the six matrix instructions a product hide the gathering, and the planes' own launch
// is a loss (65536 x 512 x 64: 68 us, 67 from planes and 14 for those).
template <int BN, int P>
struct PlanesOperand {
    static constexpr int UNITS = BN * 4, NU = (UNITS + CL_THREADS - 1) / CL_THREADS, AHEAD = 0, PLANE = BN;
    bf16x8 raw[NU][P];

    __device__ __forceinline__ static void unit(int i, int &col, int &kc) {
        const int u = threadIdx.x + i * CL_THREADS;
        col = u >> 2;
        kc = u & 3;
    }
    __device__ __forceinline__ static void offsets(long, long col0, long cols, unsigned (&off)[NU]) {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            int c, kc;
            unit(i, c, kc);
            off[i] = (unsigned)(((min(col0 + c, cols - 1) - col0) * KT + kc * 8) * 2);
        }
    }
    __device__ __forceinline__ void load(const bf16_t *__restrict__ stage, long plane, const unsigned (&off)[NU]) {
#pragma unroll
        for (int i = 0; i < NU; ++i)
#pragma unroll
            for (int p = 0; p < P; ++p) raw[i][p] = at_bytes<bf16x8>(stage + p * plane, off[i]);
    }
    __device__ __forceinline__ void store(bf16_t *lds, long, long) const {
#pragma unroll
        for (int i = 0; i < NU; ++i) {
            int c, kc;
            unit(i, c, kc);
            if (UNITS % CL_THREADS == 0 || c < BN)
#pragma unroll
                for (int p = 0; p < P; ++p) *(bf16x8 *)(lds + (p * BN + c) * LROW + kc * 8) = raw[i][p];
        }
    }
};

// Squared norms of the codes of a tile: four neighbouring threads hold a code's chunks.
template <typename OpN, typename At>
__device__ __forceinline__ void norms(const float (&sq)[OpN::NU], At at) {
#pragma unroll
    for (int i = 0; i < OpN::NU; ++i) {
        int c, kc;
        if (!OpN::unit(i, c, kc)) continue;
        float s = sq[i];
        s += __shfl_xor(s, 1, 64);
        s += __shfl_xor(s, 2, 64);
        if (kc == 0) *at(c) = s;
    }
}

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 mfma(f16x8 a, f16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

struct ProductArgs {
    const void *m, *n;  // operands: output rows' side and output columns' side
    void *out;          // result; with several splits partial sums, float [split][rows * cols + rows] (GRAD_X: [rows * cols])
    long rows, cols, sum;
    long ld_m, ld_n;    // ld_n: GRAD_*: pitch of the planes, whose size is cols * ld_n
    int tiles_m, tiles_n, splits;
    long sum_per_split;  // a multiple of KT
    float scale;
    const void *code;    // GRAD_CODE with one split: the codebook
};
// How a tile's columns' operand lies in memory and in LDS.
template <typename E>
constexpr bool from_planes() {
    return !is_f32<E>();
}
template <Product OP, typename E, int P, typename M, int NT>
using ColumnsOperand = std::conditional_t<OP != LOGITS && from_planes<E>(), PlanesOperand<NT * 16, P>, ColsOperand<E, OP == LOGITS, NT * 16, P, M>>;
// LDS of a tile: two stages of the columns' operand, and the norms of its codes.
template <Product OP, typename E, int P, int NT>
constexpr int tile_lds() {
    return 2 * P * ColumnsOperand<OP, E, P, bf16_t, NT>::PLANE * LROW * 2 + (OP == LOGITS ? NT * 16 * 4 : 0);
}

// Four consecutive columns of a row.
template <typename EO>
__device__ __forceinline__ void put4(EO *row, long n, long cols, const float (&x)[4]) {
    typename VecAt<EO, 4>::type r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = (EO)x[e];
    if (n + 4 <= cols) *(typename VecAt<EO, 4>::type *)(row + n) = r;
    else
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < cols) row[n + e] = r[e];
}

// One workgroup's tile of 64 MT x 16 NT outputs: each wave 16 MT rows of it and all its columns.  Two stages of both
// operands are on the way while one multiplies: a stage's matrix instructions take less time than memory to answer.
template <Product OP, typename EM, typename EN, int PM, int PN, typename M, int MT, int NT, typename EO>
__device__ __forceinline__ void product_tile(const ProductArgs &a, const int block, char *lds) {
    constexpr bool KC_M = OP != GRAD_CODE, KC_N = OP == LOGITS, PLANES = OP != LOGITS && from_planes<EN>();
    constexpr int BN = NT * 16;
    using OpM = RowsOperand<EM, KC_M, MT, PM, M>;
    using OpN = ColumnsOperand<OP, EN, PN, M, NT>;
    using MN = std::conditional_t<PLANES, bf16_t, EN>;  // what the columns' operand lies in memory as
    M(*s_n)[PN][OpN::PLANE][LROW] = (M(*)[PN][OpN::PLANE][LROW])lds;
    float *s_norm = (float *)(lds + 2 * PN * OpN::PLANE * LROW * sizeof(M));
    // Workgroups b and b + 8 run on one XCD: the tiles that share rows (GRAD_CODE: a split) go to the same one, whose L2
    // then serves the shared operand once.
    const int xcd = block & 7, slot = block >> 3;
    int tm, tn, split;
    if constexpr (OP == GRAD_CODE) {
        const int per = a.tiles_m * a.tiles_n;
        split = slot / per * 8 + xcd;
        tm = slot % per % a.tiles_m;
        tn = slot % per / a.tiles_m;
        if (split >= a.splits) return;
    } else {
        const int per = a.tiles_n * a.splits, rest = slot % per;
        tm = slot / per * 8 + xcd;
        tn = rest % a.tiles_n;
        split = rest / a.tiles_n;
        if (tm >= a.tiles_m) return;
    }
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long m0 = ((long)tm * 4 + wave) * (MT * 16), n0 = (long)tn * BN;
    const long k0 = split * a.sum_per_split, kend = min(k0 + a.sum_per_split, a.sum);
    const int fr = lane & 15, fk = (lane >> 4) * 8;  // this lane's row and first summed element of a fragment

    constexpr int DEPTH = 2;
    OpM om[DEPTH];
    OpN on[DEPTH];
    float sq[OpN::NU] = {}, sum_m[MT] = {};
    f32x4 acc[MT][NT] = {};
    unsigned off_m[KC_M ? MT : 1];
    unsigned off_n[OpN::NU];
    OpM::offsets(a.ld_m, m0, a.rows, fr, fk, off_m);
    OpN::offsets(a.ld_n, n0, a.cols, off_n);
    const EM *const pm = (const EM *)a.m + OpM::first_row(m0, a.rows) * (KC_M ? a.ld_m : 1);
    const MN *pn = (const MN *)a.n;
    if constexpr (PLANES) pn += n0 * KT;
    else pn += OpN::origin(n0) * (KC_N ? a.ld_n : 1);
    const auto stage = [&](OpN &n, int buf, bool there) {
        n.store(&s_n[buf][0][0][0], n0, a.cols);
        if constexpr (OP == LOGITS)
            if (there) n.add_squares(sq);
    };
    const auto rows_fragments = [&](const OpM &m, Frag<M> (&fm)[MT][PM]) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            EM v[8];
            m.values(i, v);
            if constexpr (OP == GRAD_CODE)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum_m[i] += (float)v[e];
            cut<PM, M>(v, fm[i]);
        }
    };
    const auto multiply = [&](const Frag<M> (&fm)[MT][PM], int buf) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            Frag<M> fn[PN];
#pragma unroll
            for (int p = 0; p < PN; ++p) fn[p] = *(const Frag<M> *)&s_n[buf][p][OpN::AHEAD + j * 16 + fr][fk];
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
    };
    // Whole stages: the loads ahead are never skipped (past the last stage they repeat it), so that the compiler can tell how
    // many are behind the one it waits for.
    const int stages = (int)((kend - k0) / KT);
    const auto load = [&](OpM &m, OpN &n, int s) {
        const long k = k0 + (long)min(s, stages - 1) * KT;
        m.load_whole(pm + (KC_M ? k : k * a.ld_m), a.ld_m, off_m);
        if constexpr (PLANES) n.load(pn + k * a.cols, a.cols * a.ld_n, off_n);
        else n.load_whole(pn + (KC_N ? k : k * a.ld_n), a.ld_n, off_n);
    };
    // stage s: its rows' operand is in om[CUR], its columns' in plane CUR & 1
    const auto step = [&](auto which, int s) {
        constexpr int CUR = decltype(which)::value, NEXT = (CUR + 1) % DEPTH;
        Frag<M> fm[MT][PM];
        rows_fragments(om[CUR], fm);
        load(om[CUR], on[CUR], s + DEPTH);
        // The barrier orders this plane's reads after its stores, and the other plane's next stores after its last reads.
        __syncthreads();
        multiply(fm, CUR & 1);
        stage(on[NEXT], NEXT & 1, s + 1 < stages);
    };
    if (stages > 0) {
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) load(om[i], on[i], i);
        stage(on[0], 0, true);
        for (int s = 0; s < stages; s += DEPTH) {
            step(std::integral_constant<int, 0>{}, s);
            if (s + 1 >= stages) break;
            step(std::integral_constant<int, 1>{}, s + 1);
        }
    }
    const long done = k0 + (long)stages * KT;
    if (done < kend) {  // what is left of the sum
        const int left = (int)(kend - done);
        om[0].load_part(pm + (KC_M ? done : done * a.ld_m), a.ld_m, off_m, fk, left);
        if constexpr (PLANES) on[0].load(pn + done * a.cols, a.cols * a.ld_n, off_n);
        else on[0].load_part(pn + (KC_N ? done : done * a.ld_n), a.ld_n, off_n, left);
        Frag<M> fm[MT][PM];
        rows_fragments(om[0], fm);
        __syncthreads();
        stage(on[0], 0, true);
        __syncthreads();
        multiply(fm, 0);
    }

    if constexpr (OP == LOGITS) {  // |code|^2: four neighbouring threads hold a row's chunks
        norms<OpN>(sq, [&](int c) { return s_norm + c; });
        __syncthreads();
    }
    if constexpr (OP == GRAD_CODE) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
            sum_m[i] += __shfl_xor(sum_m[i], 16, 64);
            sum_m[i] += __shfl_xor(sum_m[i], 32, 64);
        }
    }
    const bool part = OP != LOGITS && a.splits > 1;
    float *partial = (float *)a.out + split * (a.rows * a.cols + (OP == GRAD_CODE ? a.rows : 0));
    // A lane holds four consecutive columns of one row of each 16 x 16 tile.
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        bool mine;
        const long m = OpM::held(m0, a.rows, i, fr, mine);
        if (!mine) continue;
        if (OP == GRAD_CODE && part && tn == 0 && lane < 16) partial[a.rows * a.cols + m] = sum_m[i];
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int nl = j * 16 + (lane >> 4) * 4;
            const long n = n0 + nl;
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = acc[i][j][e];
                if constexpr (OP == LOGITS) x[e] = fmaf(2.f, x[e], -s_norm[nl + e]) * a.scale;
                if constexpr (OP == GRAD_X) x[e] *= part ? 1.f : a.scale;
                if constexpr (OP == GRAD_CODE)
                    if (!part && n + e < a.cols) x[e] = a.scale * fmaf(-sum_m[i], (float)((const EN *)a.code)[m * a.cols + n + e], x[e]);
            }
            if (part) put4(partial + m * a.cols, n, a.cols, x);
            else put4((EO *)a.out + m * a.cols, n, a.cols, x);
        }
    }
}

// The logits of long rows (those whose fragments logits_kernel could not keep in registers).
template <typename E, int P, typename M, int MT, int NT>
__global__ __launch_bounds__(CL_THREADS, 2) void logits_tile_kernel(ProductArgs a) {
    __shared__ __attribute__((aligned(16))) char lds[tile_lds<LOGITS, E, P, NT>()];
    product_tile<LOGITS, E, E, P, P, M, MT, NT, float>(a, blockIdx.x, lds);
}

// The logits: a workgroup keeps the fragments of its 64 MT rows for all NS stages of the sum in registers, cut once, and
// walks over its share of the codes, 16 NT at a time.  The output is what has to move (d is small against the number of codes),
// and nothing else is read twice.  Two sets of codes in LDS: the next ones are there before this tile's results are stored,
// because loads and stores complete in order, and a wait for codes behind the stores was a wait for the stores (bf16,
// 50007 x 1024 x 256: 66 us, against 42 for the products alone and 30 for the stores alone).
template <typename E, int P, typename M, int NS, int MT>
__global__ __launch_bounds__(CL_THREADS) void logits_kernel(ProductArgs a) {
    constexpr int NT = 4, BN = NT * 16;
    constexpr bool AHEAD = NS * P <= 8;  // two sets are 80 KB at most, for two workgroups a CU; longer fp32 rows have one
    using OpM = RowsOperand<E, true, MT, P, M>;
    using OpN = ColsOperand<E, true, BN, P, M>;
    __shared__ __attribute__((aligned(16))) M s_n[AHEAD ? 2 : 1][NS][P][BN][LROW];
    // a code's norm lies in the padding behind its first piece
    const auto norm_at = [&](int buf, int c) { return (float *)&s_n[buf][0][0][c][KT]; };
    // tiles_n here: workgroups that share a tile of rows
    const int xcd = blockIdx.x & 7, slot = blockIdx.x >> 3;
    const int tm = slot / a.tiles_n * 8 + xcd, first = slot % a.tiles_n;
    if (tm >= a.tiles_m) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long m0 = ((long)tm * 4 + wave) * (MT * 16);
    const int fr = lane & 15, fk = (lane >> 4) * 8;
    const int col_tiles = (int)((a.cols + BN - 1) / BN);
    OpN on[NS];
    const auto load_codes = [&](int t) {
        unsigned off[OpN::NU];
        OpN::offsets(a.ld_n, (long)t * BN, a.cols, off);
        const E *p = (const E *)a.n + (long)t * BN * a.ld_n;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int left = (int)a.sum - s * KT;  // only the last stage may be cut
            if (s + 1 < NS || left >= KT) on[s].load_whole(p + s * KT, a.ld_n, off);
            else on[s].load_part(p + s * KT, a.ld_n, off, left);
        }
    };
    const auto keep_codes = [&](int buf) {
        float sq[OpN::NU] = {};
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            on[s].store(&s_n[buf][s][0][0][0], 0, 0);
            on[s].add_squares(sq);
        }
        norms<OpN>(sq, [&](int c) { return norm_at(buf, c); });
    };
    Frag<M> fm[NS][MT][P];
    {
        OpM om[NS];
        unsigned off[MT];
        OpM::offsets(a.ld_m, m0, a.rows, fr, fk, off);
        const E *p = (const E *)a.m + OpM::first_row(m0, a.rows) * a.ld_m;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            const int left = (int)a.sum - s * KT;
            if (s + 1 < NS || left >= KT) om[s].load_whole(p + s * KT, a.ld_m, off);
            else om[s].load_part(p + s * KT, a.ld_m, off, fk, left);
        }
        load_codes(first);
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                E v[8];
                om[s].values(i, v);
                cut<P, M>(v, fm[s][i]);
            }
    }
    if (AHEAD) keep_codes(0);
    int buf = 0;
    for (int t = first; t < col_tiles; t += a.tiles_n, buf ^= AHEAD) {
        if (!AHEAD) {
            if (t != first) __syncthreads();
            keep_codes(0);
        }
        // these codes are there, and all waves are through with the ones before
        __syncthreads();
        const bool more = t + a.tiles_n < col_tiles;
        if (more) load_codes(t + a.tiles_n);
        f32x4 acc[MT][NT] = {};
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                Frag<M> fn[P];
#pragma unroll
                for (int p = 0; p < P; ++p) fn[p] = *(const Frag<M> *)&s_n[buf][s][p][j * 16 + fr][fk];
#pragma unroll
                for (int order = 2; order >= 0; --order)
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        const int q = order - p;
                        if (q < 0 || q >= P) continue;
#pragma unroll
                        for (int i = 0; i < MT; ++i) acc[i][j] = mfma(fn[q], fm[s][i][p], acc[i][j]);
                    }
            }
        if (AHEAD && more) keep_codes(buf ^ 1);
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            const int nl = j * 16 + (lane >> 4) * 4;
            float norm[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) norm[e] = *norm_at(buf, nl + e);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const long m = OpM::row(m0, i, fr);
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = fmaf(2.f, acc[i][j][e], -norm[e]) * a.scale;
                if (m < a.rows) put4((float *)a.out + m * a.cols, (long)t * BN + nl, a.cols, x);
            }
        }
    }
}

// A tile of 16 x 32 outputs of a small product, whose time is the length of its sum: the four waves take every fourth stage each,
// with both operands straight from memory and no barrier, and add up in LDS at the end.
constexpr int SMALL_NT = 2;
template <Product OP, typename E, int P>
__device__ __forceinline__ void small_tile(const ProductArgs &a, const int block, f32x4 (&s_acc)[4][SMALL_NT][64], float (&s_sum)[4][16]) {
    constexpr bool KC_M = OP == GRAD_X;
    constexpr int WAVES = CL_THREADS / 64, DEPTH = 2;
    using OpM = RowsOperand<float, KC_M, 1, 3, bf16_t>;
    using OpN = RowsOperand<E, false, 1, P, bf16_t>;  // sixteen columns as rows
    const int tm = block % a.tiles_m, rest = block / a.tiles_m, tn = rest % a.tiles_n, split = rest / a.tiles_n;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long m0 = (long)tm * 16, n0 = (long)tn * (16 * SMALL_NT);
    const long k0 = split * a.sum_per_split, kend = min(k0 + a.sum_per_split, a.sum);
    const int fr = lane & 15, fk = (lane >> 4) * 8;
    unsigned off_m[1], off_n[SMALL_NT][1];
    OpM::offsets(a.ld_m, m0, a.rows, fr, fk, off_m);
    const float *const pm = (const float *)a.m + OpM::first_row(m0, a.rows) * (KC_M ? a.ld_m : 1);
    const E *pn[SMALL_NT];
#pragma unroll
    for (int j = 0; j < SMALL_NT; ++j) {
        OpN::offsets(a.ld_n, n0 + j * 16, a.cols, fr, fk, off_n[j]);
        pn[j] = (const E *)a.n + OpN::first_row(n0 + j * 16, a.cols);
    }
    float sum_m = 0.f;
    f32x4 acc[SMALL_NT] = {};
    const auto multiply = [&](const OpM &m, const OpN (&n)[SMALL_NT]) {
        Frag<bf16_t> fm[3], fn[SMALL_NT][P];
        float v[8];
        m.values(0, v);
        if constexpr (OP == GRAD_CODE)
#pragma unroll
            for (int e = 0; e < 8; ++e) sum_m += v[e];
        cut<3, bf16_t>(v, fm);
#pragma unroll
        for (int j = 0; j < SMALL_NT; ++j) {
            E w[8];
            n[j].values(0, w);
            cut<P, bf16_t>(w, fn[j]);
        }
#pragma unroll
        for (int order = 2; order >= 0; --order)
#pragma unroll
            for (int p = 0; p < 3; ++p) {
                const int q = order - p;
                if (q < 0 || q >= P) continue;
#pragma unroll
                for (int j = 0; j < SMALL_NT; ++j) acc[j] = mfma(fn[j][q], fm[p], acc[j]);
            }
    };
    const int whole = (int)((kend - k0) / KT), mine = whole > wave ? (whole - wave + WAVES - 1) / WAVES : 0;  // whole stages, this wave's
    const auto load = [&](OpM &m, OpN (&n)[SMALL_NT], int t) {
        const long k = k0 + (long)(wave + min(t, mine - 1) * WAVES) * KT;
        m.load_whole(pm + (KC_M ? k : k * a.ld_m), a.ld_m, off_m);
#pragma unroll
        for (int j = 0; j < SMALL_NT; ++j) n[j].load_whole(pn[j] + k * a.ld_n, a.ld_n, off_n[j]);
    };
    OpM om[DEPTH];
    OpN on[DEPTH][SMALL_NT];
    if (mine > 0) {
#pragma unroll
        for (int i = 0; i < DEPTH; ++i) load(om[i], on[i], i);
        for (int t = 0; t < mine; t += DEPTH) {
            multiply(om[0], on[0]);
            if (t + 1 >= mine) break;
            load(om[0], on[0], t + 2);
            multiply(om[1], on[1]);
            load(om[1], on[1], t + 3);
        }
    }
    const long done = k0 + (long)whole * KT;
    if (done < kend && wave == whole % WAVES) {  // what is left of the sum
        om[0].load_part(pm + (KC_M ? done : done * a.ld_m), a.ld_m, off_m, fk, (int)(kend - done));
#pragma unroll
        for (int j = 0; j < SMALL_NT; ++j) on[0][j].load_part(pn[j] + done * a.ld_n, a.ld_n, off_n[j], fk, (int)(kend - done));
        multiply(om[0], on[0]);
    }
    if constexpr (OP == GRAD_CODE) {
        sum_m += __shfl_xor(sum_m, 16, 64);
        sum_m += __shfl_xor(sum_m, 32, 64);
        if (lane < 16) s_sum[wave][lane] = sum_m;
    }
#pragma unroll
    for (int j = 0; j < SMALL_NT; ++j) s_acc[wave][j][lane] = acc[j];
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int j = 0; j < SMALL_NT; ++j) acc[j] = (s_acc[0][j][lane] + s_acc[1][j][lane]) + (s_acc[2][j][lane] + s_acc[3][j][lane]);
    const long m = m0 + fr;
    if (m >= a.rows) return;
    if constexpr (OP == GRAD_CODE) sum_m = (s_sum[0][fr] + s_sum[1][fr]) + (s_sum[2][fr] + s_sum[3][fr]);
    const bool part = OP == GRAD_CODE && a.splits > 1;
    float *partial = (float *)a.out + split * (a.rows * a.cols + a.rows);
    if (part && tn == 0 && lane < 16) partial[a.rows * a.cols + m] = sum_m;
#pragma unroll
    for (int j = 0; j < SMALL_NT; ++j) {
        const long n = n0 + j * 16 + (lane >> 4) * 4;
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = acc[j][e];
            if constexpr (OP == GRAD_X) x[e] *= a.scale;
            if constexpr (OP == GRAD_CODE)
                if (!part && n + e < a.cols) x[e] = a.scale * fmaf(-sum_m, (float)((const E *)a.code)[m * a.cols + n + e], x[e]);
        }
        if (part) put4(partial + m * a.cols, n, a.cols, x);
        else put4((E *)a.out + m * a.cols, n, a.cols, x);
    }
}
template <typename E, int P>
__global__ __launch_bounds__(CL_THREADS) void grads_small_kernel(ProductArgs code, int code_blocks, ProductArgs x) {
    __shared__ f32x4 s_acc[4][SMALL_NT][64];
    __shared__ float s_sum[4][16];
    if ((int)blockIdx.x < code_blocks) small_tile<GRAD_CODE, E, P>(code, blockIdx.x, s_acc, s_sum);
    else small_tile<GRAD_X, E, P>(x, blockIdx.x - code_blocks, s_acc, s_sum);
}

// Cuts and transposes a matrix [rows][cols] into P planes [pitch / KT][cols][KT] of bf16, zeros behind the last row: 64 x 64
// elements a workgroup, through LDS.  The codebook's workgroups first, then the latents'.
struct PlanesArgs {
    const void *src[2];
    bf16_t *dst[2];
    long rows[2], pitch[2];
    int cols, first;  // workgroups of the first matrix
};
template <typename E, int P>
__global__ __launch_bounds__(CL_THREADS) void planes_kernel(PlanesArgs a) {
    using V = typename VecAt<E, 8>::type;
    __shared__ E s_x[64][64 + 2];
    const int which = (int)blockIdx.x >= a.first, block = blockIdx.x - (which ? a.first : 0);
    const int col_tiles = (a.cols + 63) / 64;
    const long r0 = (long)(block / col_tiles) * 64, rows = a.rows[which], pitch = a.pitch[which];
    const int c0 = block % col_tiles * 64;
    const E *src = (const E *)a.src[which];
    const int c = (threadIdx.x & 7) * 8;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int lr = i * 32 + (threadIdx.x >> 3);
        const long r = r0 + lr;
        const E *p = src + r * a.cols + c0 + c;
        V x = {};
        if (r < rows && c0 + c + 8 <= a.cols) x = *(const V *)p;
        else if (r < rows)
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c0 + c + e < a.cols) x[e] = p[e];
#pragma unroll
        for (int e = 0; e < 8; ++e) s_x[lr][c + e] = x[e];
    }
    __syncthreads();
    const int oc = threadIdx.x >> 2, orow = (threadIdx.x & 3) * 16;
    if (c0 + oc >= a.cols) return;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const long r = r0 + orow + h * 8;
        if (r >= pitch) break;
        E v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = s_x[orow + h * 8 + e][oc];
        Frag<bf16_t> parts[P];
        cut<P, bf16_t>(v, parts);
#pragma unroll
        for (int p = 0; p < P; ++p) *(bf16x8 *)(a.dst[which] + p * a.cols * pitch + (r / KT * a.cols + c0 + oc) * KT + r % KT) = parts[p];
    }
}

// Both gradients in one launch, the codebook's workgroups first (they run longer).  The logits' gradient keeps all three parts also
// for results of 16 bits: its rows sum to about nothing, so a common offset of the codes has to cancel in the products, and two parts
// leave 2^-17 of the offset there (fp16 codes of 1024 and their neighbours: twice the result's own rounding).
template <typename E, int P, int MT, int NT>
__global__ __launch_bounds__(CL_THREADS, 2) void grads_kernel(ProductArgs code, int code_blocks, ProductArgs x) {
    __shared__ __attribute__((aligned(16))) char lds[tile_lds<GRAD_X, E, P, NT>()];
    if ((int)blockIdx.x < code_blocks) product_tile<GRAD_CODE, float, E, 3, P, bf16_t, MT, NT, E>(code, blockIdx.x, lds);
    else product_tile<GRAD_X, float, E, 3, P, bf16_t, MT, NT, E>(x, blockIdx.x - code_blocks, lds);
}

// Joins the splits' partial sums in a fixed order.  The codebook's gradient: 64 neighbouring elements a workgroup, the splits
// dealt to its waves.  Behind its workgroups those of the latents' gradient, whose splits are few: four elements a thread.
struct JoinArgs {
    int d, k, splits, x_splits;
    const float *part, *x_part;
    const void *code;
    float scale;
    void *dcode, *dx;
    long x_size;
    int code_blocks;
};
template <typename E, int JOIN_WAVES>
__global__ __launch_bounds__(64 * JOIN_WAVES) void join_kernel(JoinArgs a) {
    __shared__ float s_acc[JOIN_WAVES][64], s_sum[JOIN_WAVES][64];
    if ((int)blockIdx.x >= a.code_blocks) {
        const long e = (((long)blockIdx.x - a.code_blocks) * (64 * JOIN_WAVES) + threadIdx.x) * 4;
        if (e >= a.x_size) return;
        float x[4] = {};
        if (e + 4 <= a.x_size) {
#pragma unroll 4
            for (int s = 0; s < a.x_splits; ++s) {
                const auto v = *(const typename VecAt<float, 4>::type *)(a.x_part + s * a.x_size + e);
#pragma unroll
                for (int c = 0; c < 4; ++c) x[c] += v[c];
            }
        } else {
            for (int s = 0; s < a.x_splits; ++s)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (e + c < a.x_size) x[c] += a.x_part[s * a.x_size + e + c];
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] *= a.scale;
        put4((E *)a.dx, e, a.x_size, x);
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long size = (long)a.k * a.d, e = (long)blockIdx.x * 64 + lane;
    float acc = 0.f, sum = 0.f;
    if (e < size) {
        const float *p = a.part + e, *ps = a.part + size + e / a.d;
#pragma unroll 8
        for (int s = wave; s < a.splits; s += JOIN_WAVES) {
            acc += p[s * (size + a.k)];
            sum += ps[s * (size + a.k)];
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
        ((E *)a.dcode)[e] = (E)(a.scale * fmaf(-sum, (float)((const E *)a.code)[e], acc));
    }
}

template <typename E>
constexpr int grad_parts() {
    return is_f32<E>() ? 3 : (__is_same(E, f16_t) ? 2 : 1);
}

// Gradient tiles of 64 MT rows by 16 NT columns.  {0, 0}: the small form, while its sixteenfold reading of both operands costs less than
// the longer run through larger tiles (fp32, small and large: 512 x 1024 x 256 14 and 31 us, 2048 x 512 x 256 26 and 30,
// 4096 x 1024 x 64 27 and 21, 4096 x 1024 x 256 81 and 49).
//
// All columns in one tile up to 128, 16-bit types 256: the rows' operand, the large one, is read and cut once.  With fp32's three parts
// 256 columns leave one wave a SIMD and are read from LDS more than the matrix instructions hide: two tiles of 128 (50000 x 512 x 256:
// 290 us in one, 171 so).  128 rows once they fill the chip or the products are large (fp32, 64 and 128 rows: 8192 x 512 x 256 46 and
// 56 us, 32000 x 512 x 256 136 and 109, 8192 x 8192 x 64 201 and 139); the tile of 256 columns later (bf16: 20000 x 2048 x 256 162
// and 167 us, 50000 x 2048 x 256 332 and 343, 8192 x 8192 x 256 290 and 249, 20000 x 8192 x 256 706 and 518; fp16's two parts would
// spill).  `parts` of a code: 3 for fp32,
// 2 for fp16, 1 for bf16.
constexpr int SMALL_ROWS = 4096;
struct Tile {
    int mt, nt;
};
inline Tile grad_tile(int n, int d, int k, int parts) {
    const double work = (double)n * k * d;
    if (n <= SMALL_ROWS && work < 0x1p28) return {0, 0};
    const int nt = d <= 32 ? 2 : (d <= 64 ? 4 : (d <= 128 || parts == 3 ? 8 : 16));
    const bool large = nt == 16 ? parts == 1 && work >= 0x1p34 : n >= 32768 || work >= 0x3p30;
    return {large && k > 1 ? 2 : 1, nt};
}
inline bool small_form(int n, int d, int k) { return grad_tile(n, d, k, 3).mt == 0; }
// Splits of the summed rows of the codebook's gradient.  Small: 512 rows, four stages a wave, and up to there one split does
// without the join's launch.  Else about two workgroups a CU, at least 128 rows each (the partial sums that a split writes
// and the join reads have to stay small beside its rows).
inline int code_splits(int n, int d, int k, int parts) {
    if (small_form(n, d, k)) return ceil_div(n, 512);
    const Tile t = grad_tile(n, d, k, parts);
    const long tiles = (long)ceil_div(k, 64 * t.mt) * ceil_div(d, 16 * t.nt);
    const long want = ceil_div(512, tiles), most = ceil_div(n, 128);
    return (int)(want < most ? want : most);
}
// Splits of the summed codes of the latents' gradient, where row tiles alone leave the chip idle: about two workgroups a CU, and the
// partial sums, written and read again, stay smaller than the share of the logits' gradient that they are made of.
inline int x_splits(int n, int d, int k, int parts) {
    if (small_form(n, d, k)) return 1;
    const Tile t = grad_tile(n, d, k, parts);
    const long tiles = (long)ceil_div(n, 64 * t.mt) * ceil_div(d, 16 * t.nt);
    const long want = 512 / tiles, most = k / std::max(128, 2 * d);
    return (int)std::max(1l, std::min(want, most));
}

template <typename E>
int launch_logits(hipStream_t stream, ProductArgs a) {
    constexpr int P = is_f32<E>() ? 3 : 1;
    using M = std::conditional_t<is_f32<E>(), bf16_t, E>;
    const int stages = ceil_div(a.sum, KT);
    const bool held = stages <= (is_f32<E>() ? 4 : 8);
    // 128 rows a workgroup from 8192 on, where 64 of them occupy the chip (fp32, 64 and 128 rows: 16000 x 256 x 100 19 and 13 us,
    // 26000 x 512 x 256 57 and 50); below, 64, and always as many workgroups to a tile of rows as fill the chip twice, each with its
    // share of the codes.  Many codes of up to two stages, where a workgroup's own start is short: four times, four tiles each at least (bf16, 65536 x 1024 x 64:
    // 73 us twice, 56 four times; 65536 x 512 x 256 34 and 39).
    const int mt = a.rows >= 8192 ? 2 : 1, bn = held ? 64 : 128;
    a.tiles_m = ceil_div(a.rows, 64 * mt);
    const int col_tiles = ceil_div(a.cols, bn);
    a.tiles_n = col_tiles;
    if (held) {
        const int more = stages <= 2 && col_tiles >= 16 ? std::min(ceil_div(1024, a.tiles_m), col_tiles / 4) : 1;
        a.tiles_n = std::min(col_tiles, std::max(ceil_div(512, a.tiles_m), more));
    }
    const long grid = (long)ceil_div(a.tiles_m, 8) * 8 * a.tiles_n;
    GDPSO_REQUIRE(grid_fits(grid, CL_THREADS), "code_logits: too many rows for one call");
#define CL_LOGITS(NS)                                                                                                                        \
    do {                                                                                                                                     \
        if (mt == 2) hipLaunchKernelGGL((logits_kernel<E, P, M, NS, 2>), dim3((unsigned)grid), dim3(CL_THREADS), 0, stream, a);              \
        else hipLaunchKernelGGL((logits_kernel<E, P, M, NS, 1>), dim3((unsigned)grid), dim3(CL_THREADS), 0, stream, a);                      \
    } while (0)
    if (stages == 1) CL_LOGITS(1);
    else if (stages == 2) CL_LOGITS(2);
    else if (stages == 3) CL_LOGITS(3);
    else if (stages == 4) CL_LOGITS(4);
    else if (held) {
        if constexpr (!is_f32<E>()) {
            if (stages == 5) CL_LOGITS(5);
            else if (stages == 6) CL_LOGITS(6);
            else if (stages == 7) CL_LOGITS(7);
            else CL_LOGITS(8);
        }
    } else if (mt == 2) hipLaunchKernelGGL((logits_tile_kernel<E, P, M, 2, 8>), dim3((unsigned)grid), dim3(CL_THREADS), 0, stream, a);
    else hipLaunchKernelGGL((logits_tile_kernel<E, P, M, 1, 8>), dim3((unsigned)grid), dim3(CL_THREADS), 0, stream, a);
#undef CL_LOGITS
    GDPSO_HIP(hipGetLastError());
    return GDPSO_OK;
}

// code.out or x.out null: that gradient is not wanted
template <typename E>
int launch_grads(hipStream_t stream, ProductArgs code, ProductArgs x, Tile t) {
    const bool small = t.mt == 0;
    const int tile_m = small ? 16 : 64 * t.mt, tile_n = 16 * (small ? SMALL_NT : t.nt);
    code.tiles_m = ceil_div(code.rows, tile_m);
    x.tiles_m = ceil_div(x.rows, tile_m);
    code.tiles_n = x.tiles_n = ceil_div(x.cols, tile_n);
    // the larger form deals splits and row tiles to the XCDs in eights
    const long splits = small ? code.splits : (code.splits + 7) / 8 * 8, row_tiles = small ? x.tiles_m : (x.tiles_m + 7) / 8 * 8 * x.splits;
    const long code_blocks = code.out ? splits * code.tiles_m * code.tiles_n : 0;
    const long grid = code_blocks + (x.out ? row_tiles * x.tiles_n : 0);
    GDPSO_REQUIRE(grid_fits(grid, CL_THREADS), "code_logits_grad: too many rows for one call");
    constexpr int P = grad_parts<E>();
#define CL_GRADS(MT, NT) hipLaunchKernelGGL((grads_kernel<E, P, MT, NT>), dim3((unsigned)grid), dim3(CL_THREADS), 0, stream, code, (int)code_blocks, x)
    if (small) {
        hipLaunchKernelGGL((grads_small_kernel<E, P>), dim3((unsigned)grid), dim3(CL_THREADS), 0, stream, code, (int)code_blocks, x);
    } else if (t.mt == 2) {
        if (t.nt == 2) CL_GRADS(2, 2);
        else if (t.nt == 4) CL_GRADS(2, 4);
        else if (t.nt == 8) CL_GRADS(2, 8);
        else if constexpr (P == 1) CL_GRADS(2, 16);
    } else {
        if (t.nt == 2) CL_GRADS(1, 2);
        else if (t.nt == 4) CL_GRADS(1, 4);
        else if (t.nt == 8) CL_GRADS(1, 8);
        else if constexpr (!is_f32<E>()) CL_GRADS(1, 16);
    }
#undef CL_GRADS
    GDPSO_HIP(hipGetLastError());
    return GDPSO_OK;
}

int code_check(const char *what, int n, int d, int k, int dtype, float temperature) {
    using w = std::string;
    GDPSO_REQUIRE(n >= 0 && k > 0 && d > 0, w(what) + ": n >= 0, k > 0 and d > 0 are required");
    GDPSO_REQUIRE(d <= CL_MAX_D, w(what) + ": embedding size above 4096");
    GDPSO_REQUIRE(k <= (1 << 20), w(what) + ": more than 2^20 codes");
    GDPSO_REQUIRE(dtype_ok(dtype), w(what) + ": unknown element type");
    GDPSO_REQUIRE(temperature >= 1e-6f && temperature <= 1e6f, w(what) + ": temperature must lie in [1e-6, 1e6]");
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
    const ProductArgs a = {inputs, codebook, logits, n, k, d, d, d, 0, 0, 1, ceil_div(d, KT) * (long)KT, 1.f / temperature, nullptr};
    GDPSO_WITH_DTYPE(dtype, rc = launch_logits<E>((hipStream_t)stream_, a));
    return rc;
}

namespace gdpso {
namespace {
// Workspace of the gradients: planes of the codebook and of the latents (16-bit types, two parts as fp16 needs them), then the splits'
// partial sums.  The small form has no planes.
struct GradSpace {
    size_t latents, part, x_part, bytes;  // offsets; the codebook's planes come first
};
inline long plane_pitch(long rows) { return (rows + KT - 1) / KT * KT; }
inline GradSpace grad_space(int n, int d, int k, int parts) {
    GradSpace s = {0, 0, 0, 0};
    if (n <= 0) return s;
    if (parts < 3 && !small_form(n, d, k)) {
        s.latents = (size_t)2 * d * plane_pitch(k) * 2;
        s.part = s.latents + (size_t)2 * d * plane_pitch(n) * 2;
    }
    const int splits = code_splits(n, d, k, parts), xs = x_splits(n, d, k, parts);
    s.x_part = s.part + (splits > 1 ? (size_t)splits * k * (d + 1) * sizeof(float) : 0);
    s.bytes = s.x_part + (xs > 1 ? (size_t)xs * n * d * sizeof(float) : 0);
    return s;
}
template <typename E>
int launch_planes(hipStream_t stream, const PlanesArgs &a, bool codes, bool latents) {
    PlanesArgs b = a;
    const int col_tiles = ceil_div(a.cols, 64);
    b.first = codes ? ceil_div(a.rows[0], 64) * col_tiles : 0;
    const long grid = b.first + (latents ? (long)ceil_div(a.rows[1], 64) * col_tiles : 0);
    GDPSO_REQUIRE(grid_fits(grid, CL_THREADS), "code_logits_grad: too many rows for one call");
    hipLaunchKernelGGL((planes_kernel<E, grad_parts<E>()>), dim3((unsigned)grid), dim3(CL_THREADS), 0, stream, b);
    GDPSO_HIP(hipGetLastError());
    return GDPSO_OK;
}
}  // namespace
}  // namespace gdpso

extern "C" size_t gdpso_code_logits_grad_workspace_bytes(int n, int d, int k) {
    if (n <= 0 || d <= 0 || k <= 0) return 0;
    return std::max({grad_space(n, d, k, 1).bytes, grad_space(n, d, k, 2).bytes, grad_space(n, d, k, 3).bytes});  // whatever the type
}

extern "C" int gdpso_code_logits_grad(void *stream_, int n, int d, int k, const float *grad_logits, const void *inputs, const void *codebook, int dtype,
                                      float temperature, void *grad_inputs, void *grad_codebook, void *workspace, size_t workspace_bytes) {
    int rc = code_check("code_logits_grad", n, d, k, dtype, temperature);
    if (rc) return rc;
    GDPSO_REQUIRE(n == 0 || (grad_logits && inputs), "code_logits_grad: null argument");
    GDPSO_REQUIRE(codebook, "code_logits_grad: null argument");
    const int parts = dtype == DT_F32 ? 3 : (dtype == DT_F16 ? 2 : 1);
    const GradSpace space = grad_space(n, d, k, parts);
    const size_t need = gdpso_code_logits_grad_workspace_bytes(n, d, k);
    GDPSO_REQUIRE(need == 0 || workspace, "code_logits_grad: null workspace");
    if (workspace_bytes < need) return fail(GDPSO_ERR_WORKSPACE, "code_logits_grad: workspace too small");
    hipStream_t stream = (hipStream_t)stream_;
    const float scale = 2.f / temperature;
    const int splits = code_splits(n, d, k, parts), xs = x_splits(n, d, k, parts);
    float *const part = (float *)((char *)workspace + space.part), *const x_part = (float *)((char *)workspace + space.x_part);
    if (n > 0 && (grad_inputs || grad_codebook)) {
        const long per = ceil_div(ceil_div(n, splits), KT) * (long)KT;
        ProductArgs code = {grad_logits, inputs, splits > 1 && grad_codebook ? part : grad_codebook, k, d, n, k, d, 0, 0, splits, per, scale, codebook};
        const long x_per = ceil_div(ceil_div(k, xs), KT) * (long)KT;
        ProductArgs x = {grad_logits, codebook, xs > 1 && grad_inputs ? x_part : grad_inputs, n, d, k, k, d, 0, 0, xs, x_per, scale, nullptr};
        if (parts < 3 && !small_form(n, d, k)) {
            const PlanesArgs planes = {{codebook, inputs}, {(bf16_t *)workspace, (bf16_t *)((char *)workspace + space.latents)}, {k, n},
                                       {plane_pitch(k), plane_pitch(n)}, d, 0};
            rc = dtype == DT_BF16 ? launch_planes<bf16_t>(stream, planes, grad_inputs != nullptr, grad_codebook != nullptr)
                                  : launch_planes<f16_t>(stream, planes, grad_inputs != nullptr, grad_codebook != nullptr);
            if (rc) return rc;
            x.n = planes.dst[0];
            x.ld_n = planes.pitch[0];
            code.n = planes.dst[1];
            code.ld_n = planes.pitch[1];
        }
        GDPSO_WITH_DTYPE(dtype, rc = launch_grads<E>(stream, code, x, grad_tile(n, d, k, parts)));
        if (rc) return rc;
    }
    const bool join_code = grad_codebook && splits != 1, join_x = grad_inputs && xs > 1;  // no rows: zeros
    if (join_code || join_x) {
        const int waves = splits > 64 ? 16 : 4;  // many splits of few elements: more waves a workgroup (65536 x 64 x 64: 32 us with 4, 27)
        const long code_blocks = join_code ? ceil_div((long)k * d, 64) : 0, x_size = (long)n * d;
        const long grid = code_blocks + (join_x ? ceil_div(x_size, 64 * 4 * waves) : 0);
        GDPSO_REQUIRE(grid_fits(grid, 64 * waves), "code_logits_grad: too many rows for one call");
        const JoinArgs a = {d, k, splits, xs, part, x_part, codebook, scale, grad_codebook, grad_inputs, x_size, (int)code_blocks};
        if (waves == 16)
            GDPSO_WITH_DTYPE(dtype, hipLaunchKernelGGL((join_kernel<E, 16>), dim3((unsigned)grid), dim3(64 * 16), 0, stream, a));
        else
            GDPSO_WITH_DTYPE(dtype, hipLaunchKernelGGL((join_kernel<E, 4>), dim3((unsigned)grid), dim3(64 * 4), 0, stream, a));
        GDPSO_HIP(hipGetLastError());
    }
    return GDPSO_OK;
}
