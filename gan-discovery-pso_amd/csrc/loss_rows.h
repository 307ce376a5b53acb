// What the row-wise losses (balance.hip, distill.hip) share: rows of logits in registers, reductions over the lanes that
// hold a row, and the scaled exponential of a softmax.
//
// A row belongs to a team of threads: 1 ... 64 lanes of a wave, so that rows of a few columns still fill a wave's
// loads, or a whole workgroup.  Thread `pos` of a team of TEAM holds chunks of 16 bytes, chunk j at column
// (j * TEAM + pos) * VEC, so neighbouring threads read neighbouring memory and a thread keeps the same columns
// in every row.  Chunks are loaded as vectors at element alignment (rows may start anywhere); the chunk that a row's
// end cuts is read and written element by element and filled up with -inf, which adds nothing to a softmax.
#pragma once
#include "common.h"

#include <math.h>

namespace gdpso {

// A launch's work items are counted in 32 bits.
inline bool grid_fits(long blocks, int threads) { return blocks < (1l << 32) / threads; }

template <typename E, int N>
struct VecAt {  // N elements at element alignment
    typedef E type __attribute__((ext_vector_type(N), aligned(sizeof(E))));
};

// Softmax over x / temperature in base 2: exp2(c x - c m), c = log2(e) / temperature.  fmaf(x, c, -c m) rounds once; the
// rounding of c m is the same factor in every term and cancels in the quotient (logarithms use the same shifted values).
// That factor stays near 1 only while c m is moderate: from 2^20 on (masks of a type's lowest value, a small
// temperature) the difference x - m is formed first (m0 = m, m1 = 0), which is exact where it matters, x near m.
struct Shift {
    float c, m0, m1;
    __device__ __forceinline__ Shift(float scale, float m) {
        c = scale;
        if (m == -INFINITY) m = 0.f;  // nothing finite: every term is 0, the sum 0
        const float cm = c * m;
        const bool big = fabsf(cm) > 1048576.f;
        m0 = big ? m : 0.f;
        m1 = big ? 0.f : cm;
    }
    __device__ __forceinline__ float arg(float x) const { return fmaf(x - m0, c, -m1); }  // base-2 logarithm of the term
    __device__ __forceinline__ float exp(float x) const { return __builtin_amdgcn_exp2f(arg(x)); }
};
// The fmaf form's scale: log2(e) / temperature.
inline float log2e_over(float temperature) { return (float)(1.4426950408889634074 / (double)temperature); }

// A value moved between the lanes of a wave by the DPP control CTRL (no LDS traffic).
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// All lanes of every group of TEAM lanes get the group's reduction.  Once 4 (8) lanes agree, a mirrored half row (row) reaches
// the other 4 (8).
template <int TEAM, typename F>
__device__ __forceinline__ float team_reduce(float v, F op) {
    if constexpr (TEAM > 1) v = op(v, dpp<0xB1>(v));   // quad_perm 1,0,3,2
    if constexpr (TEAM > 2) v = op(v, dpp<0x4E>(v));   // quad_perm 2,3,0,1
    if constexpr (TEAM > 4) v = op(v, dpp<0x141>(v));  // row_half_mirror
    if constexpr (TEAM > 8) v = op(v, dpp<0x140>(v));  // row_mirror
    if constexpr (TEAM == 32) v = op(v, __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, v), 0x401f)));  // lane ^ 16
    if constexpr (TEAM == 64) {
        v = op(v, dpp<0x142>(v));  // row_bcast 15: rows 1 and 3 now hold the halves
        v = op(v, dpp<0x143>(v));  // row_bcast 31: row 3 holds all
        v = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
    }
    return v;
}
template <int TEAM>
__device__ __forceinline__ float team_max(float v) {
    return team_reduce<TEAM>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int TEAM>
__device__ __forceinline__ float team_sum(float v) {
    return team_reduce<TEAM>(v, [](float a, float b) { return a + b; });
}

// NCH chunks of a row per thread.  ENDS, for teams of more threads than two chunks have elements: chunks of 16-bit columns begin at
// the row's first multiple of 16 bytes, and the few columns ahead of them and behind the last whole one are held one a thread.  Rows
// of an odd number of columns are off 16 bytes (8192 x 50007 bf16, loss alone: 246 us at element alignment, 227 so; fp32 gains
// nothing), and many chunks that each might be the cut one cost a workgroup's rows twice the registers.
template <typename E, int TEAM, int NCH, bool ENDS = false>
struct RowRegs {
    static constexpr int VEC = vec_of<E>();
    using V = typename VecAt<E, VEC>::type;
    using W = __attribute__((ext_vector_type(4))) unsigned;
    W raw[NCH];
    E single;  // ENDS: the column ahead of the chunks or behind them that this thread holds, if any
    int head;  // ENDS: columns ahead of the chunks

    // Columns of a row ahead of its first multiple of 16 bytes, the column behind its last whole chunk, and thread pos' column among
    // those outside the chunks (e or more: none).
    __device__ __forceinline__ static int head_of(const E *row, int e) { return is_f32<E>() ? 0 : min((int)(-(uintptr_t)row / sizeof(E) % VEC), e); }
    __device__ __forceinline__ static int outside(int head, int e, int pos) { return pos < head ? pos : head + (e - head) / VEC * VEC + pos - head; }
    __device__ __forceinline__ static int column(int j, int pos) { return (j * TEAM + pos) * VEC; }
    __device__ __forceinline__ void load(const E *__restrict__ row, int e, int pos) {
        if constexpr (ENDS) {
            static_assert(TEAM >= 2 * VEC, "a thread for every column outside the chunks");
            constexpr unsigned none = is_f32<E>() ? 0xff800000u : (__is_same(E, bf16_t) ? 0xff80ff80u : 0xfc00fc00u);  // -inf
            head = head_of(row, e);
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                const int c = head + column(j, pos);
                raw[j] = W{none, none, none, none};
                if (c + VEC <= e) raw[j] = __builtin_bit_cast(W, *(const V *)(row + c));
            }
            const int c = outside(head, e, pos);
            single = c < e ? row[c] : (E)-INFINITY;
            return;
        }
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            const int c = column(j, pos);
            V x;
            if (c + VEC <= e) x = *(const V *)(row + c);
            else
#pragma unroll
                for (int v = 0; v < VEC; ++v) x[v] = c + v < e ? row[c + v] : (E)-INFINITY;
            raw[j] = __builtin_bit_cast(W, x);
        }
    }
    __device__ __forceinline__ float at(int j, int v) const {
        if constexpr (is_f32<E>()) {
            const unsigned word = raw[j][v];  // (bit_cast of the element itself would read element 0)
            return __builtin_bit_cast(float, word);
        } else if constexpr (__is_same(E, bf16_t)) return __builtin_bit_cast(float, v & 1 ? raw[j][v >> 1] & 0xffff0000u : raw[j][v >> 1] << 16);
        else return (float)__builtin_bit_cast(f16_t, (unsigned short)(raw[j][v >> 1] >> (v & 1) * 16));
    }
    // Between two passes over the row: keeps the compiler from carrying 16-bit logits in their widened form (twice the
    // registers) from one to the next.
    __device__ __forceinline__ void again() {
        if constexpr (!is_f32<E>())
#pragma unroll
            for (int j = 0; j < NCH; ++j) {
                unsigned a = raw[j][0], b = raw[j][1], c = raw[j][2], d = raw[j][3];
                asm volatile("" : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
                raw[j] = W{a, b, c, d};
            }
    }
    // chunk j lies beyond the row for the whole team: the same for every thread, so a branch skips its arithmetic
    __device__ __forceinline__ static bool beyond(int j, int e) { return j > 0 && j * TEAM * VEC >= e; }
    __device__ __forceinline__ float max(int e) const {
        float m = ENDS ? (float)single : -INFINITY;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            if (beyond(j, e)) continue;
#pragma unroll
            for (int v = 0; v < VEC; ++v) m = fmaxf(m, at(j, v));
        }
        return m;
    }
    __device__ __forceinline__ float sum_exp(const Shift &s, int e) const {
        float l = ENDS ? s.exp((float)single) : 0.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            if (beyond(j, e)) continue;
#pragma unroll
            for (int v = 0; v < VEC; ++v) l += s.exp(at(j, v));
        }
        return l;
    }
    // row[c] = f(logit), past the caches: a long row's gradient is not read again before later rows have pushed it out
    // (8192 x 50007 bf16: 412 us, 408 with `clear` alone so, 401 with both)
    template <typename F>
    __device__ __forceinline__ void map(E *__restrict__ row, int e, int pos, F f) const {
        static_assert(ENDS, "long rows");
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            if (beyond(j, e)) continue;
            const int c = head + column(j, pos);
            V x;
#pragma unroll
            for (int v = 0; v < VEC; ++v) x[v] = (E)f(at(j, v));
            if (c + VEC <= e) __builtin_nontemporal_store(x, (V *)(row + c));
        }
        const int c = outside(head, e, pos);
        if (c < e) row[c] = (E)f((float)single);
    }
    // row[c] = 0
    __device__ __forceinline__ static void clear(E *__restrict__ row, int e, int pos) {
        if constexpr (ENDS) {
            const int head = head_of(row, e);
#pragma unroll 1
            for (int j = 0; j < NCH; ++j) {
                const int c = head + column(j, pos);
                if (c + VEC <= e) __builtin_nontemporal_store(V{}, (V *)(row + c));
            }
            const int c = outside(head, e, pos);
            if (c < e) row[c] = (E)0.f;
            return;
        }
#pragma unroll 1
        for (int j = 0; j < NCH; ++j) {
            const int c = column(j, pos);
            if (c + VEC <= e) __builtin_nontemporal_store(V{}, (V *)(row + c));
            else
#pragma unroll
                for (int v = 0; v < VEC; ++v)
                    if (c + v < e) row[c + v] = (E)0.f;
        }
    }
    // row[c] = f(j, v)
    template <typename F>
    __device__ __forceinline__ static void store(E *__restrict__ row, int e, int pos, F f) {
#pragma unroll
        for (int j = 0; j < NCH; ++j) {
            if (beyond(j, e)) continue;
            const int c = column(j, pos);
            V x;
#pragma unroll
            for (int v = 0; v < VEC; ++v) x[v] = (E)f(j, v);
            if (c + VEC <= e) *(V *)(row + c) = x;
            else
#pragma unroll
                for (int v = 0; v < VEC; ++v)
                    if (c + v < e) row[c + v] = x[v];
        }
    }
};

__device__ __forceinline__ long long load_index(const void *idx, int index_bytes, long long i) {
    return index_bytes == 8 ? ((const long long *)idx)[i] : (long long)((const int *)idx)[i];
}
__device__ __forceinline__ float load_typed(const void *p, int dtype, long long i) {
    if (dtype == DT_F32) return ((const float *)p)[i];
    if (dtype == DT_BF16) return (float)((const bf16_t *)p)[i];
    return (float)((const f16_t *)p)[i];
}
// Bytes of mask[0, n) that are not 0, summed over the calling workgroup of THREADS threads.
template <int THREADS>
__device__ __forceinline__ long long count_kept(const unsigned char *__restrict__ mask, long long n) {
    __shared__ long long s_kept[THREADS / 64];
    using B = typename VecAt<unsigned char, 16>::type;
    int kept = 0;
    long long i = (long long)threadIdx.x * 16;
    for (; i + 16 <= n; i += THREADS * 16) {
        const auto w = __builtin_bit_cast(__attribute__((ext_vector_type(4))) unsigned, *(const B *)(mask + i));
#pragma unroll
        for (int q = 0; q < 4; ++q) kept += __popc((((w[q] & 0x7f7f7f7fu) + 0x7f7f7f7fu) | w[q]) & 0x80808080u);
    }
    for (; i < n && i < n / 16 * 16 + 16; ++i) kept += mask[i] != 0;
    for (int o = 32; o > 0; o >>= 1) kept += __shfl_xor(kept, o, 64);
    if ((threadIdx.x & 63) == 0) s_kept[threadIdx.x >> 6] = kept;
    __syncthreads();
    long long total = 0;
    for (int w = 0; w < THREADS / 64; ++w) total += s_kept[w];
    return total;
}

}  // namespace gdpso
