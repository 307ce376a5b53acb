// Distillation from a teacher's k highest logits (t the temperature, idx their columns):
//
//   q_i = softmax(teacher's logits / t), p_i = softmax(row i / t), loss = t^2 mean_i sum_j q_ij (log q_ij - log p_i[idx_ij])
//   d loss / d s[i,c] = (t / rows) (p[i,c] - sum of q_ij with idx_ij = c)
//
// The work is one softmax over a long row and k corrections, bound by reading the logits and writing the gradient once
// each.  Rows are therefore held in registers between the two: by 1 ... 64 lanes up to 2048 fp32 or 4096 16-bit columns
// (dist_team_kernel), by a workgroup of 256 ... 1024 threads up to 65536 fp32 or 131072 16-bit columns (dist_row_kernel).  Longer
// rows, rows of 16384 columns or more where there are fewer than 128 of them (as workgroups they would leave most CUs idle), and the
// backward pass of all rows that lanes do not hold, are cut into segments: one launch leaves every segment's maximum and sum (the
// backward pass is given them), a second joins them and writes (dist_part_kernel, dist_apply_kernel).  Rows that the teacher may name
// whole go their own way at high temperatures (dist_full_kernel).
//
// The columns that a teacher names are stored a second time, behind the row's plain p; where a row names a column
// twice (a bit per column in LDS finds out, columns folded to 65536 bits), the first of its entries adds the others' weight in
// order and stores for all.  So nothing depends on the order of atomics, and the same call gives the same bits.
//
// Calls with inputs in rotation, half the rows masked (those are only written): 65536 x 512 fp32 from 16 entries 56 us (209 MB, 3.7 TB/s;
// the backward pass's gradient alone 45), 8192 x 50007 bf16 from 64 entries 300 ... 320 us (1.24 GB, 4 TB/s; value alone 155, gradient
// alone 256); a copy of 4 GiB runs at 4.76 TB/s.  12 x 131072 fp16 from 128: kernels of 4.2 + 8.2 us.
//
// Softmax statistics, terms and gradients are fp32 (dist_full_kernel: fp64 sums), the mean over the rows fp64; the gradient is rounded once, to the logits'
// type, when it is stored.
#include "loss_rows.h"

#include <algorithm>

namespace gdpso {
namespace {

constexpr int DIST_MAX_K = GDPSO_DISTILL_MAX_K;
constexpr int TEAM_THREADS = 256;
// Chunks of 16 bytes that the lanes of a wave hold, eight each (127765 x 2101 bf16: 566 us so, 673 by workgroups; fp32 rows of that
// length would be sixteen chunks a lane: 632, 589 by workgroups).
constexpr int TEAM_MAX_CHUNKS = 512;
constexpr int SEG_THREADS = 256, SEG_NCH = 8;  // a segment: at most 8192 fp32 or 16384 16-bit columns
constexpr int BITS = 1 << 16;
constexpr float LN2 = 0.69314718f;

// Where 1 / rows kept comes from: there is no mask, the stats hold it, or every workgroup counts the mask itself.
enum Kept { KEPT_ALL, KEPT_READ, KEPT_COUNT };
// Rows up to which counting costs less than a launch for it, 64 mask bytes a thread (a call with 16384 x 64: 18.6 us, 20.7 with the
// launch; 65536 x 64: 36 and 26).
constexpr int COUNT_ROWS = 16384;

struct DistArgs {
    int n, v, k;
    const void *logits;
    long long row_stride;
    const void *t_logits;
    int t_dtype;
    const void *t_idx;
    int index_bytes;
    const unsigned char *mask;
    float temperature, c;  // c = log2(e) / temperature
    float grad_scale;
    const float *upstream;
    float *stats;            // maximum and sum of every row, written with VALUE, read without
    float *inv_rows;         // 1 / rows kept, last of the stats: written by the kernel that finishes, or ahead of this one
    float inv_all;           // the same where no mask leaves rows out
    Kept kept;
    unsigned *ticket;        // segments: cleared by their first launch, the last workgroup of the second finishes; else null
    float *loss;
    float *row_loss;
    void *grad;
    double *loss_part;       // sums of row losses, one a workgroup (segments: one a row)
    int seg, segs;           // columns a segment, segments a row
    float2 *parts;           // [n][segs] maximum and sum of a segment; null: stats are read
};

__device__ __forceinline__ float inverse(long long rows) { return rows > 0 ? (float)(1. / (double)rows) : 0.f; }
template <int THREADS>
__device__ __forceinline__ float inv_kept(const DistArgs &a) {  // called by the whole workgroup
    if (a.kept == KEPT_COUNT) return inverse(count_kept<THREADS>(a.mask, a.n));
    return a.kept == KEPT_READ ? *a.inv_rows : a.inv_all;
}
__device__ __forceinline__ float grad_factor(const DistArgs &a, float inv) { return (a.upstream ? *a.upstream : a.grad_scale) * a.temperature * inv; }

// The mean over the rows: thread 0's `sum` is workgroup `block` of `blocks`.  One workgroup finishes by itself; with a ticket the last
// one adds all sums up in order; else a launch behind this one does (a ticket's release writes the L2's dirty lines back: with
// thousands of workgroups behind a large gradient it took 70 us, the launch 3).
template <int THREADS>
__device__ __forceinline__ void finish_loss(const DistArgs &a, double sum, int block, int blocks, float inv) {
    __shared__ double s_sum[THREADS / 64];
    __shared__ bool s_last;
    if (threadIdx.x == 0) {
        s_last = false;
        if (blocks == 1) {
            *a.loss = (float)(sum * (double)inv);
            if (a.kept != KEPT_READ) *a.inv_rows = inv;
        } else if (a.ticket) {
            __hip_atomic_store(&a.loss_part[block], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s_last = __hip_atomic_fetch_add(a.ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)blocks - 1;
        } else {
            a.loss_part[block] = sum;
        }
    }
    __syncthreads();
    if (!s_last) return;
    double s = 0.;
    for (int b = threadIdx.x; b < blocks; b += THREADS) s += __hip_atomic_load(&a.loss_part[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < THREADS / 64; ++w) s += s_sum[w];
        *a.loss = (float)(s * (double)inv);
        if (a.kept != KEPT_READ) *a.inv_rows = inv;
    }
}
// Entry j of row i: its column (-1: absent) and logit (-inf where absent).
__device__ __forceinline__ void entry(const DistArgs &a, long long i, int j, int &c, float &t) {
    const long long col = load_index(a.t_idx, a.index_bytes, i * a.k + j);
    const bool in = col >= 0 && col < a.v;
    c = in ? (int)col : -1;
    t = in ? load_typed(a.t_logits, a.t_dtype, i * a.k + j) : -INFINITY;
}
// q (log2 q - log2 p) short of the two sums' logarithms
__device__ __forceinline__ float entry_term(float q, float t_arg, float s_arg) { return q == 0.f ? 0.f : q * (t_arg - s_arg); }
__device__ __forceinline__ float row_loss_of(const DistArgs &a, float terms, float l, float tl) {
    return l == 0.f || tl == 0.f ? 0.f : a.temperature * a.temperature * LN2 * (terms + (log2f(l) - log2f(tl)));
}

// The group of rows that a workgroup takes at u = its index, index + grid ...  Workgroups b, b + 8 ... run on one XCD, and a padded
// batch keeps and leaves out rows in runs, so groups dealt out in order leave some XCDs nothing but masked rows wherever eight groups
// divide a run.  Short rows: the groups of every eight neighbours are dealt to the XCDs starting at another one than the eight before
// (256 columns fp32, every other 32 rows masked: 236 us in order, 163 so).  Rows of whole workgroups: each XCD has its eighth in one
// piece (half masked, 8192 x 50007 bf16: 350 us in order, 354 dealt, 314 in pieces; 53676 x 5001 fp32, where a workgroup is 256
// threads: 435 dealt, 480 in pieces).
inline __host__ __device__ long long dealt_end(long long groups) { return (groups + 7) & ~7ll; }
template <bool PIECES>
__device__ __forceinline__ long long dealt(long long u, long long end) {  // may lie behind the last group
    return PIECES ? (u & 7) * (end >> 3) + (u >> 3) : (u & ~7ll) + ((u + (u >> 3)) & 7);
}

// 1 / rows that the mask keeps
__global__ __launch_bounds__(1024) void dist_kept_kernel(int n, const unsigned char *__restrict__ mask, float *__restrict__ inv_rows) {
    const float inv = inverse(count_kept<1024>(mask, n));
    if (threadIdx.x == 0) *inv_rows = inv;
}

// ------------------------------------------------------------------------------------- rows of lanes
template <typename E, int THREADS, int TEAM, int NCH, bool VALUE, bool GRAD>
__global__ __launch_bounds__(THREADS) void dist_team_kernel(DistArgs a) {
    constexpr int VEC = vec_of<E>(), TEAMS = THREADS / TEAM, WORDS = (TEAM * NCH * VEC + 31) / 32;
    __shared__ unsigned s_bits[GRAD ? TEAMS : 1][GRAD ? WORDS : 1];
    __shared__ double s_loss[VALUE ? THREADS / 64 : 1];
    const int lane = threadIdx.x & 63, pos = threadIdx.x & (TEAM - 1), team = threadIdx.x / TEAM;
    const float inv = inv_kept<THREADS>(a);
    float factor = 0.f;
    if constexpr (GRAD) {
        factor = grad_factor(a, inv);
        for (int w = pos; w < WORDS; w += TEAM) s_bits[team][w] = 0;
    }
    double sum = 0.;
    const long long end = dealt_end((a.n + TEAMS - 1ll) / TEAMS);
    for (long long u = blockIdx.x; u < end; u += gridDim.x) {
        const long long i = dealt<false>(u, end) * TEAMS + team;
        if (i >= a.n) continue;
        const E *row = (const E *)a.logits + i * a.row_stride;
        E *grow = (E *)a.grad + i * a.v;
        if (a.mask && !a.mask[i]) {
            if (VALUE && pos == 0) {
                a.row_loss[i] = 0.f;
                a.stats[2 * i] = 0.f;
                a.stats[2 * i + 1] = 0.f;
            }
            if constexpr (GRAD) RowRegs<E, TEAM, NCH>::clear(grow, a.v, pos);
            continue;
        }
        RowRegs<E, TEAM, NCH> r;
        r.load(row, a.v, pos);
        // the lane's first entry stays in registers; rows with more entries than lanes read theirs again where needed
        int c0 = -1;
        float t0 = -INFINITY, s0 = 0.f;
        if (pos < a.k) entry(a, i, pos, c0, t0);
        if (c0 >= 0) s0 = (float)row[c0];
        const auto each = [&](auto f) {  // f(j, column, teacher's logit, student's logit) for this lane's entries
            if (pos < a.k) f(pos, c0, t0, s0);
            for (int j = pos + TEAM; j < a.k; j += TEAM) {
                int c;
                float t;
                entry(a, i, j, c, t);
                f(j, c, t, c >= 0 ? (float)row[c] : 0.f);
            }
        };
        float m, l;
        if constexpr (VALUE) m = team_max<TEAM>(r.max(a.v));
        else {
            m = a.stats[2 * i];
            l = a.stats[2 * i + 1];
        }
        const Shift s(a.c, m);
        float ex[NCH][VEC];
        float mine = 0.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                ex[j][v] = s.exp(r.at(j, v));
                mine += ex[j][v];
            }
        if constexpr (VALUE) l = team_sum<TEAM>(mine);
        float tm = -INFINITY;
        each([&](int, int, float t, float) { tm = fmaxf(tm, t); });
        const Shift ts(a.c, team_max<TEAM>(tm));
        float tl = 0.f;
        each([&](int, int, float t, float) { tl += ts.exp(t); });
        tl = team_sum<TEAM>(tl);
        const bool empty = l == 0.f || tl == 0.f;
        const float inv_l = empty ? 0.f : 1.f / l, inv_tl = empty ? 0.f : 1.f / tl;
        if constexpr (VALUE) {
            float terms = 0.f;
            each([&](int, int, float t, float x) {
                const float arg = ts.arg(t);
                terms += entry_term(__builtin_amdgcn_exp2f(arg) * inv_tl, arg, s.arg(x));
            });
            terms = team_sum<TEAM>(terms);
            if (pos == 0) {
                const float loss = row_loss_of(a, terms, l, tl);
                a.row_loss[i] = loss;
                a.stats[2 * i] = m;
                a.stats[2 * i + 1] = l;
                sum += loss;
            }
        }
        if constexpr (GRAD) {
            RowRegs<E, TEAM, NCH>::store(grow, a.v, pos, [&](int j, int v) { return empty ? 0.f : factor * (ex[j][v] * inv_l); });
            if (empty) continue;
            bool twice = false;
            each([&](int, int c, float, float) {
                if (c >= 0) twice |= (atomicOr(&s_bits[team][c >> 5], 1u << (c & 31)) >> (c & 31)) & 1;
            });
            __builtin_amdgcn_wave_barrier();
            each([&](int, int c, float, float) {
                if (c >= 0) s_bits[team][c >> 5] = 0;
            });
            __builtin_amdgcn_wave_barrier();
            const unsigned long long team_lanes = (TEAM == 64 ? ~0ull : (1ull << (TEAM & 63)) - 1) << (lane & ~(TEAM - 1));
            const bool repeats = (__ballot(twice) & team_lanes) != 0;
            each([&](int j, int c, float t, float x) {
                if (c < 0) return;
                float q = ts.exp(t) * inv_tl;
                if (repeats) {
                    for (int h = 0; h < a.k; ++h) {
                        if (h == j) continue;
                        int ch;
                        float th;
                        entry(a, i, h, ch, th);
                        if (ch != c) continue;
                        if (h < j) return;  // an entry before this one stores for both
                        q += ts.exp(th) * inv_tl;
                    }
                }
                grow[c] = (E)(factor * (s.exp(x) * inv_l - q));
            });
        }
    }
    if constexpr (VALUE) {
        for (int o = TEAM; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);  // a team's first lane holds its rows' sum
        if (lane == 0) s_loss[threadIdx.x >> 6] = sum;
        __syncthreads();
        if (threadIdx.x == 0)
            for (int w = 1; w < THREADS / 64; ++w) sum += s_loss[w];
        finish_loss<THREADS>(a, sum, blockIdx.x, gridDim.x, inv);
    }
}

// ------------------------------------------------------------------- rows that a teacher may name whole, high temperatures
// Both softmaxes are nearly even there, and loss and gradient are small differences of theirs: the loss is of the order of the
// squared arguments, which t^2 makes up for, and from plain sums it would be off by t^2 2^-22 (8 of 8 columns, t = 1000: 0.2 of 0.45).
// So exponentials near 1 go by their distance to 1, whose sums are as accurate as the arguments, and the loss is a sum in which
// nothing cancels: with delta_j = log q_j - log p_j (p of the column that entry j names),
//
//   sum_j q_j delta_j = sum_j q_j (delta_j - 1 + exp(-delta_j)) + 1 - sum_j p_j        p_j - q_j = q_j (exp(-delta_j) - 1)
//
// Needed where the entries' columns may be the row, 2 k >= v; beside a larger share of other columns the loss is of the order of t^2.
constexpr float FULL_TEMPERATURE = 4.f;  // below, t^2 2^-22 is lost beside the other roundings
// Lanes of a row of v columns; what the lanes of a wave do in common is long (calls of fp32 rows at t = 4, and below:
// 65536 x 100 from 64 132 and 61 us, 179 with a wave a row; 65536 x 512 from 256 649 and 388, 767 with sixteen lanes; 512 x 8 from 8 20 and 17).
inline int full_team(int v) { return v <= 64 ? 8 : (v <= 256 ? 16 : 64); }
constexpr int full_max_v(int team) { return team == 8 ? 64 : (team == 16 ? 256 : 2 * DIST_MAX_K); }

// A sum of exponentials: how many are near 1, and the sum of those ones' distances to 1 and of the others.
struct ExpSum {
    double ones = 0., rest = 0.;
    __device__ __forceinline__ void add(float arg) {  // exp2(arg)
        const bool near = arg > -0.5f;
        ones += near ? 1. : 0.;
        rest += near ? expm1f(arg * LN2) : __builtin_amdgcn_exp2f(arg);
    }
    __device__ __forceinline__ double sum() const { return ones + rest; }
    __device__ __forceinline__ double less(const ExpSum &b) const { return (ones - b.ones) + (rest - b.rest); }
};
__device__ __forceinline__ double exp2_of(float arg) {
    ExpSum one;
    one.add(arg);
    return one.sum();
}
template <int TEAM>
__device__ __forceinline__ double team_sum64(double v) {
    for (int o = TEAM / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
template <int TEAM>
__device__ __forceinline__ ExpSum team_sum64(ExpSum s) {
    s.ones = team_sum64<TEAM>(s.ones);
    s.rest = team_sum64<TEAM>(s.rest);
    return s;
}

template <typename E, int TEAM, bool VALUE, bool GRAD>
__global__ __launch_bounds__(TEAM_THREADS) void dist_full_kernel(DistArgs a) {
    constexpr int TEAMS = TEAM_THREADS / TEAM, WORDS = full_max_v(TEAM) / 32;
    constexpr double LN2_64 = 0.69314718055994531;
    __shared__ unsigned s_bits[GRAD ? TEAMS : 1][GRAD ? WORDS : 1];
    __shared__ double s_loss[VALUE ? TEAM_THREADS / 64 : 1];
    const int lane = threadIdx.x & 63, pos = threadIdx.x & (TEAM - 1), team = threadIdx.x / TEAM;
    const float inv = inv_kept<TEAM_THREADS>(a);
    float factor = 0.f;
    if constexpr (GRAD) {
        factor = grad_factor(a, inv);
        for (int w = pos; w < WORDS; w += TEAM) s_bits[team][w] = 0;
    }
    double sum = 0.;
    for (long long i = (long long)blockIdx.x * TEAMS + team; i < a.n; i += (long long)gridDim.x * TEAMS) {
        const E *row = (const E *)a.logits + i * a.row_stride;
        E *grow = (E *)a.grad + i * a.v;
        if (a.mask && !a.mask[i]) {
            if (VALUE && pos == 0) {
                a.row_loss[i] = 0.f;
                a.stats[2 * i] = 0.f;
                a.stats[2 * i + 1] = 0.f;
            }
            if constexpr (GRAD)
                for (int c = pos; c < a.v; c += TEAM) grow[c] = (E)0.f;
            continue;
        }
        const auto each = [&](auto f) {  // f(j, column, teacher's logit, student's logit) for this lane's entries
            for (int j = pos; j < a.k; j += TEAM) {
                int c;
                float t;
                entry(a, i, j, c, t);
                if (c >= 0) f(j, c, t, (float)row[c]);
            }
        };
        float m = -INFINITY, tm = -INFINITY;
        for (int c = pos; c < a.v; c += TEAM) m = fmaxf(m, (float)row[c]);
        each([&](int, int, float t, float) { tm = fmaxf(tm, t); });
        m = team_max<TEAM>(m);
        const Shift s(a.c, m), ts(a.c, team_max<TEAM>(tm));
        ExpSum l, tl;
        for (int c = pos; c < a.v; c += TEAM) l.add(s.arg((float)row[c]));
        each([&](int, int, float t, float) { tl.add(ts.arg(t)); });
        l = team_sum64<TEAM>(l);
        tl = team_sum64<TEAM>(tl);
        const bool empty = l.sum() == 0. || tl.sum() == 0.;
        const double inv_l = empty ? 0. : 1. / l.sum(), inv_tl = empty ? 0. : 1. / tl.sum();
        const double ratio = empty ? 0. : log1p(l.less(tl) * inv_tl);  // of the two sums, its logarithm
        const auto delta = [&](float t, float x) { return LN2_64 * ((double)ts.arg(t) - (double)s.arg(x)) + ratio; };
        if constexpr (VALUE) {
            double terms = 0.;
            ExpSum named;
            each([&](int, int, float t, float x) {
                const double q = exp2_of(ts.arg(t)) * inv_tl;
                if (q == 0.) return;  // (a NaN is not)
                const double d = delta(t, x);
                terms += q * (d + expm1(-d));
                named.add(s.arg(x));
            });
            terms = team_sum64<TEAM>(terms);
            named = team_sum64<TEAM>(named);
            if (pos == 0) {
                const float loss = empty ? 0.f : (float)((double)a.temperature * a.temperature * (terms + l.less(named) * inv_l));
                a.row_loss[i] = loss;
                a.stats[2 * i] = m;
                a.stats[2 * i + 1] = (float)l.sum();
                sum += loss;
            }
        }
        if constexpr (GRAD) {
            for (int c = pos; c < a.v; c += TEAM) grow[c] = empty ? (E)0.f : (E)(factor * (float)(exp2_of(s.arg((float)row[c])) * inv_l));
            if (empty) continue;
            bool twice = false;
            each([&](int, int c, float, float) { twice |= (atomicOr(&s_bits[team][c >> 5], 1u << (c & 31)) >> (c & 31)) & 1; });
            __builtin_amdgcn_wave_barrier();
            each([&](int, int c, float, float) { s_bits[team][c >> 5] = 0; });
            __builtin_amdgcn_wave_barrier();
            const unsigned long long team_lanes = (TEAM == 64 ? ~0ull : (1ull << (TEAM & 63)) - 1) << (lane & ~(TEAM - 1));
            const bool repeats = (__ballot(twice) & team_lanes) != 0;
            each([&](int j, int c, float t, float x) {
                const double q = exp2_of(ts.arg(t)) * inv_tl;
                double diff = q == 0. ? exp2_of(s.arg(x)) * inv_l : q * expm1(-delta(t, x));
                if (repeats) {
                    for (int h = 0; h < a.k; ++h) {
                        if (h == j) continue;
                        int ch;
                        float th;
                        entry(a, i, h, ch, th);
                        if (ch != c) continue;
                        if (h < j) return;  // an entry before this one stores for both
                        diff -= exp2_of(ts.arg(th)) * inv_tl;
                    }
                }
                grow[c] = (E)(factor * (float)diff);
            });
        }
    }
    if constexpr (VALUE) {
        for (int o = TEAM; o < 64; o <<= 1) sum += __shfl_xor(sum, o, 64);  // a team's first lane holds its rows' sum
        if (lane == 0) s_loss[threadIdx.x >> 6] = sum;
        __syncthreads();
        if (threadIdx.x == 0)
            for (int w = 1; w < TEAM_THREADS / 64; ++w) sum += s_loss[w];
        finish_loss<TEAM_THREADS>(a, sum, blockIdx.x, gridDim.x, inv);
    }
}

// ----------------------------------------------------------------------------------- a workgroup a row or segment
// Two values reduced over the workgroup with one barrier; `slot` has to be free (two barriers ago or never used).
template <int THREADS>
struct PairRed {
    float a[THREADS / 64], b[THREADS / 64];
};
template <int THREADS>
__device__ __forceinline__ void wide_max2(PairRed<THREADS> &slot, float &x, float &y) {
    x = team_max<64>(x);
    y = team_max<64>(y);
    if ((threadIdx.x & 63) == 0) {
        slot.a[threadIdx.x >> 6] = x;
        slot.b[threadIdx.x >> 6] = y;
    }
    __syncthreads();
    x = slot.a[0];
    y = slot.b[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) {
        x = fmaxf(x, slot.a[w]);
        y = fmaxf(y, slot.b[w]);
    }
}
template <int THREADS>
__device__ __forceinline__ void wide_sum2(PairRed<THREADS> &slot, float &x, float &y) {
    x = team_sum<64>(x);
    y = team_sum<64>(y);
    if ((threadIdx.x & 63) == 0) {
        slot.a[threadIdx.x >> 6] = x;
        slot.b[threadIdx.x >> 6] = y;
    }
    __syncthreads();
    x = slot.a[0];
    y = slot.b[0];
#pragma unroll
    for (int w = 1; w < THREADS / 64; ++w) {
        x += slot.a[w];
        y += slot.b[w];
    }
}

// The teacher's entries of one row in LDS, and the columns they name.
struct Entries {
    int c[DIST_MAX_K];
    float t[DIST_MAX_K];
};

template <typename E, int THREADS, int NCH, bool GRAD>
__global__ __launch_bounds__(THREADS, 4) void dist_row_kernel(DistArgs a) {
    __shared__ PairRed<THREADS> s_max, s_sum;
    __shared__ Entries s_e[2];  // by turns: a wave may still read the last row's while the next row's are stored
    __shared__ float s_terms[THREADS / 64];
    __shared__ unsigned s_bits[GRAD ? BITS / 32 : 1];
    __shared__ int s_repeats;
    const int tid = threadIdx.x;
    const float inv = inv_kept<THREADS>(a);
    float factor = 0.f;
    if constexpr (GRAD) {
        factor = grad_factor(a, inv);
        for (int w = tid; w < BITS / 32; w += THREADS) s_bits[w] = 0;
    }
    double sum = 0.;
    int turn = 0;
    const long long end = dealt_end(a.n);
    for (long long u = blockIdx.x; u < end; u += gridDim.x) {
        const long long i = dealt<(THREADS >= 512)>(u, end);
        if (i >= a.n) continue;
        const E *row = (const E *)a.logits + i * a.row_stride;
        E *grow = (E *)a.grad + i * a.v;
        if (a.mask && !a.mask[i]) {
            if (tid == 0) {
                a.row_loss[i] = 0.f;
                a.stats[2 * i] = 0.f;
                a.stats[2 * i + 1] = 0.f;
            }
            if constexpr (GRAD) RowRegs<E, THREADS, NCH, true>::clear(grow, a.v, tid);
            continue;
        }
        RowRegs<E, THREADS, NCH, true> r;
        r.load(row, a.v, tid);
        Entries &ent = s_e[turn];
        turn ^= 1;  // only rows that pass the barriers below take turns
        float tm = -INFINITY;
        for (int j = tid; j < a.k; j += THREADS) {
            int c;
            float t;
            entry(a, i, j, c, t);
            ent.c[j] = c;
            ent.t[j] = t;
            tm = fmaxf(tm, t);
        }
        float m = r.max(a.v);
        wide_max2<THREADS>(s_max, m, tm);
        r.again();
        if (tid == 0) s_repeats = 0;  // read by all before that barrier, set by any behind the next
        const Shift s(a.c, m), ts(a.c, tm);
        float l = r.sum_exp(s, a.v), tl = 0.f;
        for (int j = tid; j < a.k; j += THREADS) tl += ts.exp(ent.t[j]);
        wide_sum2<THREADS>(s_sum, l, tl);
        r.again();
        const bool empty = l == 0.f || tl == 0.f;
        const float inv_l = empty ? 0.f : 1.f / l, inv_tl = empty ? 0.f : 1.f / tl;
        float terms = 0.f;
        for (int j = tid; j < a.k; j += THREADS) {
            const int c = ent.c[j];
            const float arg = ts.arg(ent.t[j]);
            if (c >= 0) terms += entry_term(__builtin_amdgcn_exp2f(arg) * inv_tl, arg, s.arg((float)row[c]));
            if (GRAD && c >= 0) {
                const unsigned bit = 1u << (c & 31);
                if (atomicOr(&s_bits[(c & (BITS - 1)) >> 5], bit) & bit) s_repeats = 1;
            }
        }
        if constexpr (GRAD) r.map(grow, a.v, tid, [&](float x) { return empty ? 0.f : factor * (s.exp(x) * inv_l); });
        if (tid < (a.k + 63) / 64 * 64 || tid < 64) {
            terms = team_sum<64>(terms);
            if ((tid & 63) == 0) s_terms[tid >> 6] = terms;
        }
        __syncthreads();  // the row's plain gradient, the bits and the terms are there
        if (tid == 0) {
            const int waves = std::min(THREADS / 64, (a.k + 63) / 64);
            for (int w = 1; w < waves; ++w) terms += s_terms[w];
            const float loss = row_loss_of(a, terms, l, tl);
            a.row_loss[i] = loss;
            a.stats[2 * i] = m;
            a.stats[2 * i + 1] = l;
            sum += loss;
        }
        if constexpr (GRAD) {
            const bool repeats = s_repeats != 0;
            for (int j = tid; j < a.k; j += THREADS) {
                const int c = ent.c[j];
                if (c < 0) continue;
                s_bits[(c & (BITS - 1)) >> 5] = 0;
                if (empty) continue;
                float q = ts.exp(ent.t[j]) * inv_tl;
                bool first = true;
                if (repeats)
                    for (int h = 0; h < a.k; ++h) {
                        if (ent.c[h] != c || h == j) continue;
                        if (h < j) {
                            first = false;  // an entry before this one stores for both
                            break;
                        }
                        q += ts.exp(ent.t[h]) * inv_tl;
                    }
                if (first) grow[c] = (E)(factor * (s.exp((float)row[c]) * inv_l - q));
            }
        }
    }
    finish_loss<THREADS>(a, sum, blockIdx.x, gridDim.x, inv);
}

// Maximum and sum of a segment; one workgroup more counts the mask.
template <typename E>
__global__ __launch_bounds__(SEG_THREADS) void dist_part_kernel(DistArgs a) {
    __shared__ PairRed<SEG_THREADS> s_max, s_sum;
    const long long i = blockIdx.x / a.segs;
    const int seg = (int)(blockIdx.x - i * a.segs), lo = seg * a.seg, len = std::min(a.seg, a.v - lo);
    if (i == a.n) {
        const float inv = inverse(a.mask ? count_kept<SEG_THREADS>(a.mask, a.n) : a.n);
        if (threadIdx.x == 0) {
            *a.inv_rows = inv;
            *a.ticket = 0;
        }
        return;
    }
    if (a.mask && !a.mask[i]) return;
    RowRegs<E, SEG_THREADS, SEG_NCH, true> r;
    r.load((const E *)a.logits + i * a.row_stride + lo, len, threadIdx.x);
    float m = r.max(len), none = 0.f;
    wide_max2<SEG_THREADS>(s_max, m, none);
    r.again();
    float l = r.sum_exp(Shift(a.c, m), len);
    wide_sum2<SEG_THREADS>(s_sum, l, none);
    if (threadIdx.x == 0) a.parts[blockIdx.x] = make_float2(m, l);
}

// Joins a row's segments (or reads its stats), and writes its loss (the first segment's workgroup) and one segment of its gradient.
template <typename E, bool VALUE, bool GRAD>
__global__ __launch_bounds__(SEG_THREADS) void dist_apply_kernel(DistArgs a) {
    __shared__ PairRed<SEG_THREADS> s_max, s_sum;
    __shared__ Entries ent;
    __shared__ float s_terms[SEG_THREADS / 64];
    __shared__ unsigned s_bits[GRAD ? BITS / 32 : 1];
    __shared__ int s_repeats;
    const int tid = threadIdx.x;
    const long long i = GRAD ? blockIdx.x / a.segs : blockIdx.x;
    const int seg = GRAD ? (int)(blockIdx.x - i * a.segs) : 0, lo = seg * a.seg, len = std::min(a.seg, a.v - lo);
    const E *row = (const E *)a.logits + i * a.row_stride;
    E *grow = (E *)a.grad + i * a.v;
    if (a.mask && !a.mask[i]) {
        if (VALUE && seg == 0) {
            if (tid == 0) {
                a.row_loss[i] = 0.f;
                a.stats[2 * i] = 0.f;
                a.stats[2 * i + 1] = 0.f;
            }
            finish_loss<SEG_THREADS>(a, 0., (int)i, a.n, *a.inv_rows);
        }
        if constexpr (GRAD) RowRegs<E, SEG_THREADS, SEG_NCH, true>::clear(grow + lo, len, tid);
        return;
    }
    RowRegs<E, SEG_THREADS, SEG_NCH, true> r;
    if constexpr (GRAD) r.load(row + lo, len, tid);
    float tm = -INFINITY, m = -INFINITY;
    for (int j = tid; j < a.k; j += SEG_THREADS) {
        int c;
        float t;
        entry(a, i, j, c, t);
        ent.c[j] = c;
        ent.t[j] = t;
        tm = fmaxf(tm, t);
    }
    if constexpr (VALUE)
        for (int p = tid; p < a.segs; p += SEG_THREADS) m = fmaxf(m, a.parts[i * a.segs + p].x);
    else m = a.stats[2 * i];
    if constexpr (GRAD) {
        for (int w = tid; w < BITS / 32; w += SEG_THREADS) s_bits[w] = 0;
        if (tid == 0) s_repeats = 0;
    }
    wide_max2<SEG_THREADS>(s_max, m, tm);
    const Shift s(a.c, m), ts(a.c, tm);
    float tl = 0.f, l = 0.f;
    if constexpr (VALUE)
        for (int p = tid; p < a.segs; p += SEG_THREADS) {
            const float2 part = a.parts[i * a.segs + p];
            // a segment's sum is relative to its own shift: to the row's by the quotient of the two
            const Shift own(a.c, part.x);
            l += part.y == 0.f ? 0.f : part.y * __builtin_amdgcn_exp2f(s.arg(part.x) - own.arg(part.x));
        }
    for (int j = tid; j < a.k; j += SEG_THREADS) tl += ts.exp(ent.t[j]);
    wide_sum2<SEG_THREADS>(s_sum, l, tl);
    if constexpr (!VALUE) l = a.stats[2 * i + 1];
    const bool empty = l == 0.f || tl == 0.f;
    const float inv_l = empty ? 0.f : 1.f / l, inv_tl = empty ? 0.f : 1.f / tl;
    float terms = 0.f;
    for (int j = tid; j < a.k; j += SEG_THREADS) {
        const int c = ent.c[j];
        if (c < 0) continue;
        if (VALUE && seg == 0) {
            const float arg = ts.arg(ent.t[j]);
            terms += entry_term(__builtin_amdgcn_exp2f(arg) * inv_tl, arg, s.arg((float)row[c]));
        }
        if (GRAD && c >= lo && c < lo + len) {
            const unsigned bit = 1u << (c & 31);
            if (atomicOr(&s_bits[(c & (BITS - 1)) >> 5], bit) & bit) s_repeats = 1;
        }
    }
    const float inv = *a.inv_rows, factor = grad_factor(a, inv);
    if constexpr (GRAD) {
        r.map(grow + lo, len, tid, [&](float x) { return empty ? 0.f : factor * (s.exp(x) * inv_l); });
    }
    if (VALUE && seg == 0) {
        terms = team_sum<64>(terms);
        if ((tid & 63) == 0) s_terms[tid >> 6] = terms;
    }
    __syncthreads();  // the segment's plain gradient, the bits and the terms are there
    if (VALUE && seg == 0) {
        float loss = 0.f;
        if (tid == 0) {
            for (int w = 1; w < SEG_THREADS / 64; ++w) terms += s_terms[w];
            loss = row_loss_of(a, terms, l, tl);
            a.row_loss[i] = loss;
            a.stats[2 * i] = m;
            a.stats[2 * i + 1] = l;
        }
        finish_loss<SEG_THREADS>(a, loss, (int)i, a.n, inv);
    }
    if constexpr (GRAD) {
        if (empty) return;
        for (int j = tid; j < a.k; j += SEG_THREADS) {
            const int c = ent.c[j];
            if (c < lo || c >= lo + len) continue;
            float q = ts.exp(ent.t[j]) * inv_tl;
            bool first = true;
            if (s_repeats)
                for (int h = 0; h < a.k; ++h) {
                    if (ent.c[h] != c || h == j) continue;
                    if (h < j) {
                        first = false;
                        break;
                    }
                    q += ts.exp(ent.t[h]) * inv_tl;
                }
            if (first) grow[c] = (E)(factor * (s.exp((float)row[c]) * inv_l - q));
        }
    }
}

// The mean where neither one workgroup nor a ticket could finish it.
__global__ __launch_bounds__(1024) void dist_finish_kernel(DistArgs a, int parts) {
    __shared__ double s_sum[16];
    double s = 0.;
    for (int i = threadIdx.x; i < parts; i += 1024) s += a.loss_part[i];
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6] = s;
    const float inv = a.kept == KEPT_READ ? *a.inv_rows : inverse(a.mask ? count_kept<1024>(a.mask, a.n) : a.n);
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 16; ++w) s += s_sum[w];
        *a.loss = (float)(s * (double)inv);
        *a.inv_rows = inv;
    }
}

int distill_check(const char *what, int n, int v, int k, const void *logits, long long row_stride, int dtype, const void *t_logits, int t_dtype,
                  const void *t_idx, int index_bytes, float temperature) {
    using w = std::string;
    GDPSO_REQUIRE(n >= 0 && v > 0 && k > 0, w(what) + ": n >= 0, v > 0 and k > 0 are required");
    GDPSO_REQUIRE(k <= DIST_MAX_K, w(what) + ": more than 1024 teacher logits a row");
    GDPSO_REQUIRE(dtype_ok(dtype) && dtype_ok(t_dtype), w(what) + ": unknown element type");
    GDPSO_REQUIRE(index_bytes == 4 || index_bytes == 8, w(what) + ": indices are 4 or 8 bytes");
    GDPSO_REQUIRE(temperature >= 1e-6f && temperature <= 1e6f, w(what) + ": temperature must lie in [1e-6, 1e6]");
    GDPSO_REQUIRE(n == 0 || (logits && t_logits && t_idx), w(what) + ": null argument");
    GDPSO_REQUIRE(row_stride >= 0, w(what) + ": negative row stride");
    return GDPSO_OK;
}

// How rows of v columns are held.
enum Way { BY_TEAM, BY_FULL, BY_ROW, BY_SEGMENT };
struct Plan {
    Way way;
    int team, chunks;  // BY_TEAM, BY_FULL: lanes a row; BY_TEAM: chunks a lane
    int threads;       // of a workgroup (BY_ROW: threads a row, chunks a thread in `chunks`)
    int seg, segs;
};
inline bool may_be_full(int v, int k) { return v <= 2ll * k; }
inline Plan plan_rows(int n, int v, int vec, bool full) {
    Plan p = {BY_TEAM, 0, 0, 0, 0, 0};
    const int chunks = ceil_div(v, vec);
    if (full) {
        p.way = BY_FULL;
        p.team = full_team(v);
        p.threads = TEAM_THREADS;
        return p;
    }
    if (chunks <= TEAM_MAX_CHUNKS) {
        p.team = 1;
        while (p.team < chunks && p.team < 64) p.team <<= 1;
        p.chunks = 1;
        while (p.team * p.chunks < chunks) p.chunks <<= 1;
        // Many rows: fewer lanes a row and up to four chunks a lane, so that a wave deals with several rows' teachers at once (65536 x
        // 512 fp32: 75 us with 64 lanes, 67 with 32; 262144 x 256: 434 and 238).  Few rows have to spread over the chip instead.
        if (n >= 8192)
            while (p.team > 16 && p.chunks < 4) p.team >>= 1, p.chunks <<= 1;
        // rows that 1024 threads finish in two rounds are left to one workgroup
        p.threads = p.team <= 8 && n > 2 * (TEAM_THREADS / p.team) && n <= 2 * (1024 / p.team) ? 1024 : TEAM_THREADS;
        return p;
    }
    p.way = BY_ROW;
    if (chunks <= 256 * 8) p.threads = 256, p.chunks = 8;
    else if (chunks <= 512 * 16) p.threads = 512, p.chunks = 16;
    else if (chunks <= 1024 * 16) p.threads = 1024, p.chunks = 16;
    else p.way = BY_SEGMENT;
    // few rows of many columns: as workgroups of a row they would occupy one CU each (50007 bf16 columns, by segments and by rows: 100
    // rows 21 and 32 us, 200 rows 51 and 22)
    if (n < 128 && v >= 16384) p.way = BY_SEGMENT;
    const int most = SEG_THREADS * SEG_NCH * vec, least = SEG_THREADS * vec;
    // about two workgroups a CU, segments of whole rounds of the workgroup's loads
    long seg = ceil_div((long)v * n, 512 * (long)least) * (long)least;
    p.seg = (int)std::min<long>(std::max<long>(seg, least), most);
    p.segs = ceil_div(v, p.seg);
    return p;
}

// Workgroups at most, an odd number of eights, so that a workgroup's later rows fall elsewhere in a padded batch's pattern than its
// first: few rows a workgroup, so that those with masked rows leave their place to others (8192 x 50007 bf16, half masked: 2048
// workgroups 375 us, 8192 351), but a team's teacher entries and LDS are set up once for several (fp32, 262144 x 256, half masked: 4088
// workgroups 163 us, 8184 247).
constexpr int DIST_TEAM_BLOCKS = 4088, DIST_ROW_BLOCKS = 16376;
inline int dist_blocks(const Plan &p, int n) {
    if (p.way == BY_SEGMENT) return n > 0 ? n : 1;
    const long rows = p.way == BY_ROW ? 1 : p.threads / p.team;
    const long want = ((long)n + rows - 1) / rows;
    if (p.way == BY_TEAM && want <= 2) return 1;  // a second round of rows costs less than the launch that joins workgroups
    return (int)(want < 1 ? 1 : std::min<long>(want, p.way == BY_ROW ? DIST_ROW_BLOCKS : DIST_TEAM_BLOCKS));
}
// Workspace: ticket, sums of row losses, segments
constexpr size_t TICKET_BYTES = 16;
inline size_t loss_bytes(const Plan &p, int n) { return ((size_t)dist_blocks(p, n) * sizeof(double) + 15) / 16 * 16; }
inline size_t space_bytes(const Plan &p, int n) {
    return TICKET_BYTES + loss_bytes(p, n) + (p.way == BY_SEGMENT ? (size_t)n * p.segs * sizeof(float2) : 0);
}

template <typename E, bool VALUE, bool GRAD>
int launch_team(hipStream_t stream, const DistArgs &a, const Plan &p) {
    const dim3 grid(dist_blocks(p, a.n));
#define DIST_TEAM(N, T, C) hipLaunchKernelGGL((dist_team_kernel<E, N, T, C, VALUE, GRAD>), grid, dim3(N), 0, stream, a)
    if (p.threads == 1024) {
        if (p.team == 1) DIST_TEAM(1024, 1, 1);
        else if (p.team == 2) DIST_TEAM(1024, 2, 1);
        else if (p.team == 4) DIST_TEAM(1024, 4, 1);
        else DIST_TEAM(1024, 8, 1);
    } else {
        switch (p.team * 32 + p.chunks) {
            case 1 * 32 + 1: DIST_TEAM(256, 1, 1); break;
            case 2 * 32 + 1: DIST_TEAM(256, 2, 1); break;
            case 4 * 32 + 1: DIST_TEAM(256, 4, 1); break;
            case 8 * 32 + 1: DIST_TEAM(256, 8, 1); break;
            case 16 * 32 + 1: DIST_TEAM(256, 16, 1); break;
            case 32 * 32 + 1: DIST_TEAM(256, 32, 1); break;
            case 64 * 32 + 1: DIST_TEAM(256, 64, 1); break;
            case 64 * 32 + 2: DIST_TEAM(256, 64, 2); break;
            case 16 * 32 + 2: DIST_TEAM(256, 16, 2); break;
            case 16 * 32 + 4: DIST_TEAM(256, 16, 4); break;
            case 32 * 32 + 4: DIST_TEAM(256, 32, 4); break;
            case 64 * 32 + 4: DIST_TEAM(256, 64, 4); break;
            case 64 * 32 + 8: DIST_TEAM(256, 64, 8); break;
            default: break;
        }
    }
#undef DIST_TEAM
    GDPSO_HIP(hipGetLastError());
    return GDPSO_OK;
}

template <typename E, bool VALUE, bool GRAD>
int launch_distill(hipStream_t stream, const DistArgs &a, const Plan &p) {
    if (p.way == BY_TEAM) return launch_team<E, VALUE, GRAD>(stream, a, p);
    if (p.way == BY_FULL) {
        const dim3 grid(dist_blocks(p, a.n));
        if (p.team == 8) hipLaunchKernelGGL((dist_full_kernel<E, 8, VALUE, GRAD>), grid, dim3(TEAM_THREADS), 0, stream, a);
        else if (p.team == 16) hipLaunchKernelGGL((dist_full_kernel<E, 16, VALUE, GRAD>), grid, dim3(TEAM_THREADS), 0, stream, a);
        else hipLaunchKernelGGL((dist_full_kernel<E, 64, VALUE, GRAD>), grid, dim3(TEAM_THREADS), 0, stream, a);
        GDPSO_HIP(hipGetLastError());
        return GDPSO_OK;
    }
    if (VALUE && p.way == BY_ROW) {
        const dim3 grid(dist_blocks(p, a.n));
        if (p.threads == 256) hipLaunchKernelGGL((dist_row_kernel<E, 256, 8, GRAD>), grid, dim3(256), 0, stream, a);
        else if (p.threads == 512) hipLaunchKernelGGL((dist_row_kernel<E, 512, 16, GRAD>), grid, dim3(512), 0, stream, a);
        else hipLaunchKernelGGL((dist_row_kernel<E, 1024, 16, GRAD>), grid, dim3(1024), 0, stream, a);
    } else {
        const long blocks = (long)a.n * a.segs;
        GDPSO_REQUIRE(grid_fits(blocks + 1, SEG_THREADS), "distill: too many rows for one call");
        if (VALUE) hipLaunchKernelGGL((dist_part_kernel<E>), dim3((unsigned)blocks + 1), dim3(SEG_THREADS), 0, stream, a);
        hipLaunchKernelGGL((dist_apply_kernel<E, VALUE, GRAD>), dim3((unsigned)(GRAD ? blocks : a.n)), dim3(SEG_THREADS), 0, stream, a);
    }
    GDPSO_HIP(hipGetLastError());
    return GDPSO_OK;
}

}  // namespace
}  // namespace gdpso

using namespace gdpso;

extern "C" size_t gdpso_distill_workspace_bytes(int n, int v, int k) {
    if (n < 0 || v <= 0 || k <= 0) return 0;
    const size_t size = std::max(space_bytes(plan_rows(n, v, 4, false), n), space_bytes(plan_rows(n, v, 8, false), n));
    return may_be_full(v, k) ? std::max(size, space_bytes(plan_rows(n, v, 4, true), n)) : size;  // whatever type and temperature
}

extern "C" int gdpso_distill(void *stream_, int n, int v, int k, const void *logits, long long row_stride, int dtype, const void *t_logits, int t_dtype,
                             const void *t_indices, int index_bytes, const unsigned char *mask, float temperature, float grad_scale, float *loss,
                             float *row_loss, float *row_stats, void *grad, void *workspace, size_t workspace_bytes) {
    int rc = distill_check("distill", n, v, k, logits, row_stride, dtype, t_logits, t_dtype, t_indices, index_bytes, temperature);
    if (rc) return rc;
    GDPSO_REQUIRE(loss && row_stats && workspace && (n == 0 || row_loss), "distill: null argument");
    if (workspace_bytes < gdpso_distill_workspace_bytes(n, v, k)) return fail(GDPSO_ERR_WORKSPACE, "distill: workspace too small");
    hipStream_t stream = (hipStream_t)stream_;
    float *inv_rows = row_stats + 2 * (size_t)n;
    const Plan p = plan_rows(n, v, 16 / (int)dtype_size(dtype), temperature >= FULL_TEMPERATURE && may_be_full(v, k));
    unsigned *ticket = (unsigned *)workspace;
    double *loss_part = (double *)((char *)workspace + TICKET_BYTES);
    float2 *parts = (float2 *)((char *)loss_part + loss_bytes(p, n));
    const bool one = dist_blocks(p, n) == 1;
    // the kept rows ahead of a gradient: by the workgroups themselves, by the segments' first launch, or by a launch of its own
    // (no rows: neither runs, and the finishing launch counts)
    const bool ahead = mask && n > COUNT_ROWS && p.way != BY_SEGMENT && (grad || one);
    const Kept kept = (p.way == BY_SEGMENT && n > 0) || ahead ? KEPT_READ : (mask && (grad || one) ? KEPT_COUNT : KEPT_ALL);
    const DistArgs a = {n, v, k, logits, row_stride, t_logits, t_dtype, t_indices, index_bytes, mask, temperature, log2e_over(temperature), grad_scale,
                        nullptr, row_stats, inv_rows, n > 0 ? (float)(1. / n) : 0.f, kept, p.way == BY_SEGMENT ? ticket : nullptr, loss, row_loss,
                        grad, loss_part, p.seg, p.segs, parts};
    if (n > 0) {
        if (ahead) hipLaunchKernelGGL(dist_kept_kernel, dim3(1), dim3(1024), 0, stream, n, mask, inv_rows);
        if (grad)
            GDPSO_WITH_DTYPE(dtype, rc = (launch_distill<E, true, true>(stream, a, p)));
        else
            GDPSO_WITH_DTYPE(dtype, rc = (launch_distill<E, true, false>(stream, a, p)));
        if (rc) return rc;
    }
    if (n == 0 || (!one && !a.ticket)) hipLaunchKernelGGL(dist_finish_kernel, dim3(1), dim3(1024), 0, stream, a, n > 0 ? dist_blocks(p, n) : 0);
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
    const Plan p = plan_rows(n, v, 16 / (int)dtype_size(dtype), temperature >= FULL_TEMPERATURE && may_be_full(v, k));
    const DistArgs a = {n, v, k, logits, row_stride, t_logits, t_dtype, t_indices, index_bytes, mask, temperature, log2e_over(temperature), 0.f, upstream,
                        (float *)row_stats, (float *)row_stats + 2 * (size_t)n, 0.f, KEPT_READ, nullptr, nullptr, nullptr, grad, nullptr, p.seg, p.segs,
                        nullptr};
    GDPSO_WITH_DTYPE(dtype, rc = (launch_distill<E, false, true>((hipStream_t)stream_, a, p)));
    return rc;
}
