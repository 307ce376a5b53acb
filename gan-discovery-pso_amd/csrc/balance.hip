// Balance loss of a choice among e codes (experts, classes) and the counts it rests on:
//
//   p_i = softmax(row i), P[c] = mean of p over the kept rows, f[c] = choices of c / all counted choices
//   loss = e sum_c f[c] P[c]            d loss / d s[i,c] = (e / rows) p[i,c] (f[c] - sum_j f[j] p[i,j])
//
// One pass over the logits: a row is read once into the registers of its team of threads, its softmax is finished
// there, added to the team's running column sums and, for the gradient, multiplied out and stored.  f does not depend on the
// logits, so the choices are counted first and value and gradient need one read and one write of [n, e] together.  The
// pass is bound by memory (inputs in rotation: 50001 x 1001 fp32 without a gradient 41 us, 4.9 TB/s; 131072 x 64 bf16 with one 14 us,
// 2.3 TB/s, the backward pass's gradient alone 11); the counting and the join of the column sums are 5 to 9 us each beside it.
// Rows of more than 2048 columns, a workgroup each, whose threads hold 32 values whatever the row's length: 20000 x 5000 fp32 with a
// gradient 267 us (800 MB, 3.0 TB/s), without 141 (2.8 TB/s), and a join of 16.
//
// Sums are fp32 within a workgroup's rows, fp64 across workgroups, in an order that n, e and the type fix: the same call
// gives the same bits.  The gradient is rounded once, to the logits' type, when it is stored.
#include "loss_rows.h"

#include <algorithm>

namespace gdpso {
namespace {

constexpr int BAL_MAX_E = GDPSO_BALANCE_MAX_E;
constexpr int TEAM_THREADS = 256;
constexpr int TEAM_MAX_E = 2048;  // columns a wave holds: 32 values a lane, beside 32 column sums and 32 f
constexpr int WIDE_THREADS = 512; // rows of up to 16384 columns: 32 values a thread
constexpr int HIST_THREADS = 1024;
constexpr int JOIN_COLS = 16, JOIN_GROUPS = 64;
constexpr int HIST_MAX = 64;
// Choices that every workgroup of the gradient counts for itself, 16 a thread (a call with 4096 choices: 17.8 us, 19.9 with a launch
// that counts).
constexpr int OWN_CHOICES = 4096;

// Counting workgroups: eight choices a thread; the partial counts are read again by every workgroup of the gradient, so there
// are at most 64 of them.
inline int hist_blocks(long long choices, int threads) {
    const long long h = (choices + threads * 8 - 1) / (threads * 8);
    return h < 1 ? 1 : (h > HIST_MAX ? HIST_MAX : (int)h);
}

struct Choices {
    const void *idx;
    int index_bytes;
    const unsigned char *mask;
    int n, k, e;
    int blocks;
    unsigned *part;  // [blocks][e + 2]: choices of every code, rows kept, choices counted
};
inline __host__ __device__ int hist_copies(int e) { return e <= 256 ? 8 : 1; }

// Counts of one of `blocks` shares of the choices into s_hist[0, e) and s_total (rows kept, choices counted).  Copies by
// lane keep the lanes of a wave off each other's counters where there are few codes.
__device__ void count_choices(const Choices &a, int block, int blocks, unsigned *s_hist, unsigned *s_total, int threads) {
    const int copies = hist_copies(a.e);
    for (int c = threadIdx.x; c < copies * a.e; c += threads) s_hist[c] = 0;
    if (threadIdx.x < 2) s_total[threadIdx.x] = 0;
    __syncthreads();
    unsigned *mine = s_hist + (copies > 1 ? (threadIdx.x & 7) * a.e : 0);
    unsigned rows = 0, counted = 0;
    const long long step = (long long)blocks * threads, first = (long long)block * threads + threadIdx.x;
    if (a.mask) {
#pragma unroll 4
        for (long long i = first; i < a.n; i += step) {
            const bool keep = a.mask[i] != 0;
            rows += keep;
#pragma unroll 2
            for (int j = 0; j < a.k; ++j) {
                const long long c = load_index(a.idx, a.index_bytes, i * a.k + j);
                if (keep && c >= 0 && c < a.e) {
                    ++counted;
                    atomicAdd(&mine[c], 1u);
                }
            }
        }
    } else {
        const long long total = (long long)a.n * a.k;
#pragma unroll 4
        for (long long i = first; i < total; i += step) {
            const long long c = load_index(a.idx, a.index_bytes, i);
            if (c >= 0 && c < a.e) {
                ++counted;
                atomicAdd(&mine[c], 1u);
            }
        }
        if (block == 0 && threadIdx.x == 0) rows = a.n;
    }
    for (int o = 32; o > 0; o >>= 1) {
        rows += __shfl_xor(rows, o, 64);
        counted += __shfl_xor(counted, o, 64);
    }
    if ((threadIdx.x & 63) == 0) {
        atomicAdd(&s_total[0], rows);
        atomicAdd(&s_total[1], counted);
    }
    __syncthreads();
    if (copies > 1) {
        for (int c = threadIdx.x; c < a.e; c += threads) {
            unsigned s = s_hist[c];
            for (int r = 1; r < copies; ++r) s += s_hist[r * a.e + c];
            s_hist[c] = s;
        }
        __syncthreads();
    }
}
__device__ __forceinline__ void write_counts(const Choices &a, int block, const unsigned *s_hist, const unsigned *s_total, int threads) {
    unsigned *out = a.part + (size_t)block * (a.e + 2);
    for (int c = threadIdx.x; c < a.e; c += threads) out[c] = s_hist[c];
    if (threadIdx.x < 2) out[a.e + threadIdx.x] = s_total[threadIdx.x];
}

__global__ __launch_bounds__(HIST_THREADS) void bal_count_kernel(Choices a) {
    extern __shared__ unsigned s_hist[];
    __shared__ unsigned s_total[2];
    count_choices(a, blockIdx.x, a.blocks, s_hist, s_total, HIST_THREADS);
    write_counts(a, blockIdx.x, s_hist, s_total, HIST_THREADS);
}

struct BalArgs {
    int n, e;
    const void *logits;
    long long row_stride;
    const unsigned char *mask;
    int row_blocks;
    float *col_part;            // [row_blocks][e] column sums of p
    const unsigned *count_part; // [count_blocks][e + 2]
    int count_blocks;
    const long long *counts, *totals;  // or the finished counts [e] and totals [2]
    float grad_scale;
    const float *upstream;
    void *grad;
    unsigned *ticket;           // cleared here for the join
    bool own_counts;
};

// Sum of a column of the partial counts, several loads under way at a time.
__device__ __forceinline__ unsigned sum_counts(const unsigned *__restrict__ part, int blocks, int stride) {
    unsigned s = 0;
#pragma unroll 16
    for (int h = 0; h < blocks; ++h) s += part[(size_t)h * stride];
    return s;
}
// f into LDS and the gradient's factor grad_scale * e / rows (0 when no row is kept).
__device__ __forceinline__ float shares(const BalArgs &a, float *s_f, int threads) {
    __shared__ long long s_total[2];
    if (threadIdx.x < 2) s_total[threadIdx.x] = a.counts ? a.totals[threadIdx.x] : sum_counts(a.count_part + a.e + threadIdx.x, a.count_blocks, a.e + 2);
    for (int c = threadIdx.x; c < a.e; c += threads) s_f[c] = a.counts ? (float)a.counts[c] : (float)sum_counts(a.count_part + c, a.count_blocks, a.e + 2);
    __syncthreads();
    const long long rows = s_total[0], counted = s_total[1];
    const float inv = counted > 0 ? (float)(1. / (double)counted) : 0.f;
    for (int c = threadIdx.x; c < a.e; c += threads) s_f[c] *= inv;
    __syncthreads();
    const float g = a.upstream ? *a.upstream : a.grad_scale;
    return rows > 0 ? g * (float)a.e / (float)rows : 0.f;
}

// Rows of at most TEAM * NCH * VEC columns, TEAM lanes a row.
template <typename E, int TEAM, int NCH, bool SUMS, bool GRAD>
__global__ __launch_bounds__(TEAM_THREADS) void bal_team_kernel(BalArgs a, Choices ch) {
    constexpr int VEC = vec_of<E>(), TEAMS = TEAM_THREADS / TEAM;
    extern __shared__ float s_mem[];
    __shared__ unsigned s_total[SUMS ? 2 : 1];
    if (SUMS && !GRAD && (int)blockIdx.x >= a.row_blocks) {  // without a gradient nothing waits for the counts: they ride along
        count_choices(ch, blockIdx.x - a.row_blocks, ch.blocks, (unsigned *)s_mem, s_total, TEAM_THREADS);
        write_counts(ch, blockIdx.x - a.row_blocks, (unsigned *)s_mem, s_total, TEAM_THREADS);
        return;
    }
    const int pos = threadIdx.x & (TEAM - 1), team = threadIdx.x / TEAM;
    float f[NCH][VEC], acc[NCH][VEC];
    float factor = 0.f;
    if constexpr (GRAD) {
        if (SUMS && a.own_counts) {  // few choices: every workgroup counts them all, which costs less than a launch ahead of this one
            unsigned *s_hist = (unsigned *)s_mem;
            count_choices(ch, 0, 1, s_hist, s_total, TEAM_THREADS);
            if (blockIdx.x == 0) write_counts(ch, 0, s_hist, s_total, TEAM_THREADS);
            __syncthreads();  // from here on the counters' memory holds f
            const float inv = s_total[1] > 0 ? (float)(1. / (double)s_total[1]) : 0.f;
            for (int c = threadIdx.x; c < a.e; c += TEAM_THREADS) s_mem[c] = (float)s_hist[c] * inv;
            factor = s_total[0] > 0 ? a.grad_scale * (float)a.e / (float)s_total[0] : 0.f;
            __syncthreads();
        } else {
            factor = shares(a, s_mem, TEAM_THREADS);
        }
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const int c = RowRegs<E, TEAM, NCH>::column(j, pos) + v;
                f[j][v] = c < a.e ? s_mem[c] : 0.f;
            }
        if (SUMS) __syncthreads();
    }
    if constexpr (SUMS) {
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int v = 0; v < VEC; ++v) acc[j][v] = 0.f;
        if (blockIdx.x == 0 && threadIdx.x == 0) *a.ticket = 0;
    }
    const E *logits = (const E *)a.logits;
    E *grad = (E *)a.grad;
    const float c2 = 1.44269504f;
    for (long long i = (long long)blockIdx.x * TEAMS + team; i < a.n; i += (long long)a.row_blocks * TEAMS) {
        RowRegs<E, TEAM, NCH> row;
        row.load(logits + i * a.row_stride, a.e, pos);
        const bool keep = !a.mask || a.mask[i] != 0;
        const Shift s(c2, team_max<TEAM>(row.max(a.e)));
        float ex[NCH][VEC], l = 0.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                ex[j][v] = s.exp(row.at(j, v));
                l += ex[j][v];
            }
        l = team_sum<TEAM>(l);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                ex[j][v] = keep ? ex[j][v] * inv : 0.f;
                if constexpr (SUMS) acc[j][v] += ex[j][v];
                if constexpr (GRAD) dot = fmaf(ex[j][v], f[j][v], dot);
            }
        if constexpr (GRAD) {
            dot = team_sum<TEAM>(dot);
            RowRegs<E, TEAM, NCH>::store(grad + i * a.e, a.e, pos, [&](int j, int v) {
                return keep ? factor * ex[j][v] * (f[j][v] - dot) : 0.f;
            });
        }
    }
    if constexpr (SUMS) {
        // the wave's teams, then the workgroup's waves, in order
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int v = 0; v < VEC; ++v)
#pragma unroll
                for (int o = TEAM; o < 64; o <<= 1) acc[j][v] += __shfl_xor(acc[j][v], o, 64);
        const int lane = threadIdx.x & 63;
        for (int w = 0; w < TEAM_THREADS / 64; ++w) {
            if ((int)(threadIdx.x >> 6) == w && lane < TEAM) {
#pragma unroll
                for (int j = 0; j < NCH; ++j)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        const int c = RowRegs<E, TEAM, NCH>::column(j, pos) + v;
                        if (c < a.e) s_mem[c] = w == 0 ? acc[j][v] : s_mem[c] + acc[j][v];
                    }
            }
            __syncthreads();
        }
        float *out = a.col_part + (size_t)blockIdx.x * a.e;
        for (int c = threadIdx.x; c < a.e; c += TEAM_THREADS) out[c] = s_mem[c];
    }
}

__device__ __forceinline__ float wide_reduce(float v, float *s_red, bool is_max) {
    v = is_max ? team_max<64>(v) : team_sum<64>(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = s_red[0];
    for (int w = 1; w < WIDE_THREADS / 64; ++w) v = is_max ? fmaxf(v, s_red[w]) : v + s_red[w];
    return v;
}

// Rows of up to 16384 columns, a workgroup a row.
template <typename E, bool SUMS, bool GRAD>
__global__ __launch_bounds__(WIDE_THREADS) void bal_wide_kernel(BalArgs a) {
    constexpr int VEC = vec_of<E>(), NCH = BAL_MAX_E / (WIDE_THREADS * VEC);
    extern __shared__ float s_f[];
    __shared__ float s_red[WIDE_THREADS / 64];
    const int pos = threadIdx.x;
    float acc[NCH][VEC];
    float factor = 0.f;
    if constexpr (GRAD) factor = shares(a, s_f, WIDE_THREADS);
    if constexpr (SUMS) {
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int v = 0; v < VEC; ++v) acc[j][v] = 0.f;
        if (blockIdx.x == 0 && threadIdx.x == 0) *a.ticket = 0;
    }
    const E *logits = (const E *)a.logits;
    E *grad = (E *)a.grad;
    for (long long i = blockIdx.x; i < a.n; i += a.row_blocks) {
        RowRegs<E, WIDE_THREADS, NCH> row;
        row.load(logits + i * a.row_stride, a.e, pos);
        const bool keep = !a.mask || a.mask[i] != 0;
        const Shift s(1.44269504f, wide_reduce(row.max(a.e), s_red, true));
        float ex[NCH][VEC], l = 0.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                ex[j][v] = s.exp(row.at(j, v));
                l += ex[j][v];
            }
        l = wide_reduce(l, s_red, false);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        float dot = 0.f;
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const int c = RowRegs<E, WIDE_THREADS, NCH>::column(j, pos) + v;
                ex[j][v] = keep ? ex[j][v] * inv : 0.f;
                if constexpr (SUMS) acc[j][v] += ex[j][v];
                if constexpr (GRAD) dot = fmaf(ex[j][v], c < a.e ? s_f[c] : 0.f, dot);
            }
        if constexpr (GRAD) {
            dot = wide_reduce(dot, s_red, false);
            RowRegs<E, WIDE_THREADS, NCH>::store(grad + i * a.e, a.e, pos, [&](int j, int v) {
                const int c = RowRegs<E, WIDE_THREADS, NCH>::column(j, pos) + v;
                return keep ? factor * ex[j][v] * ((c < a.e ? s_f[c] : 0.f) - dot) : 0.f;
            });
        }
    }
    if constexpr (SUMS) {
        float *out = a.col_part + (size_t)blockIdx.x * a.e;
#pragma unroll
        for (int j = 0; j < NCH; ++j)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const int c = RowRegs<E, WIDE_THREADS, NCH>::column(j, pos) + v;
                if (c < a.e) out[c] = acc[j][v];
            }
    }
}

// Joins column sums and counts: sixteen columns a workgroup, the partial sums dealt to 64 groups of threads; the last
// workgroup to finish adds the workgroups' shares of the loss up in order.
__global__ __launch_bounds__(JOIN_COLS *JOIN_GROUPS) void bal_join_kernel(int e, int row_blocks, const float *__restrict__ col_part, int count_blocks,
                                                                         const unsigned *__restrict__ count_part, float *__restrict__ mean_prob,
                                                                         long long *__restrict__ counts, long long *__restrict__ totals, double *dots,
                                                                         unsigned *ticket,
                                                                         float *__restrict__ loss) {
    __shared__ double s_col[JOIN_COLS * JOIN_GROUPS / 64][JOIN_COLS];
    __shared__ unsigned s_cnt[JOIN_COLS * JOIN_GROUPS / 64][JOIN_COLS];
    __shared__ long long s_total[2];
    __shared__ bool s_last;
    const int col = threadIdx.x % JOIN_COLS, grp = threadIdx.x / JOIN_COLS, wave = threadIdx.x >> 6;
    const int c = blockIdx.x * JOIN_COLS + col;
    double s = 0.;
    unsigned cnt = 0;
    if (c < e) {
        if (grp < count_blocks) cnt = count_part[(size_t)grp * (e + 2) + c];
#pragma unroll 8
        for (int g = grp; g < row_blocks; g += JOIN_GROUPS) s += (double)col_part[(size_t)g * e + c];
    }
    if (wave == 0) {
        const int lane = threadIdx.x;
        long long rows = 0, counted = 0;
        if (lane < count_blocks) {
            rows = count_part[(size_t)lane * (e + 2) + e];
            counted = count_part[(size_t)lane * (e + 2) + e + 1];
        }
        for (int o = 32; o > 0; o >>= 1) {
            rows += __shfl_xor(rows, o, 64);
            counted += __shfl_xor(counted, o, 64);
        }
        if (lane == 0) {
            s_total[0] = rows;
            s_total[1] = counted;
        }
    }
    // a wave's four groups, then the waves, in order
    for (int o = JOIN_COLS; o < 64; o <<= 1) {
        s += __shfl_xor(s, o, 64);
        cnt += __shfl_xor(cnt, o, 64);
    }
    if ((threadIdx.x & 63) < JOIN_COLS) {
        s_col[wave][col] = s;
        s_cnt[wave][col] = cnt;
    }
    __syncthreads();
    double dot = 0.;
    if (threadIdx.x < JOIN_COLS) {
        long long total = 0;
        s = 0.;
#pragma unroll
        for (int w = 0; w < JOIN_COLS * JOIN_GROUPS / 64; ++w) {
            s += s_col[w][col];
            total += s_cnt[w][col];
        }
        if (c < e) {
            const double mean = s_total[0] > 0 ? s / (double)s_total[0] : 0.;
            mean_prob[c] = (float)mean;
            counts[c] = total;
            dot = s_total[1] > 0 ? mean * ((double)total / (double)s_total[1]) : 0.;
        }
        for (int o = JOIN_COLS / 2; o > 0; o >>= 1) dot += __shfl_xor(dot, o, 64);
    }
    if (threadIdx.x == 0) {
        if (blockIdx.x == 0) {
            totals[0] = s_total[0];
            totals[1] = s_total[1];
        }
        if (gridDim.x == 1) {
            *loss = (float)(dot * e);
            s_last = false;
        } else {
            __hip_atomic_store(&dots[blockIdx.x], dot, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s_last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == gridDim.x - 1;
        }
    }
    __syncthreads();
    if (s_last && threadIdx.x < 64) {
        double t = 0.;
        for (unsigned b = threadIdx.x; b < gridDim.x; b += 64) t += __hip_atomic_load(&dots[b], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        for (int o = 32; o > 0; o >>= 1) t += __shfl_xor(t, o, 64);
        if (threadIdx.x == 0) *loss = (float)(t * e);
    }
}

// How a row of e columns is held: lanes a row and chunks a lane (0 lanes: a workgroup a row).
struct Hold {
    int team, chunks;
};
inline Hold hold_row(int e, int vec) {
    if (e > TEAM_MAX_E) return {0, 0};
    const int chunks = ceil_div(e, vec);
    int team = 1;
    while (team < chunks && team < 64) team <<= 1;
    int per = 1;
    while (team * per < chunks) per <<= 1;
    return {team, per};
}
// Workgroups over the rows: four a CU fill the chip's loads, and every one leaves a row of column sums to join.
inline int row_blocks(int n, int e, int dtype) {
    const Hold h = hold_row(e, 16 / (int)dtype_size(dtype));
    const long per = h.team ? TEAM_THREADS / h.team : 1;
    const long want = (n + per - 1) / per;
    const long most = h.team ? 1024 : 512;
    return (int)(want < 1 ? 1 : (want < most ? want : most));
}

struct BalSpace {
    float *col_part;
    unsigned *count_part;
    double *dots;
    unsigned *ticket;
    size_t bytes;
};
inline BalSpace balance_space(void *ws, int e) {
    // sized for the most workgroups any n and type may take, so that the size asked for depends on nothing else
    char *p = (char *)ws;
    BalSpace s;
    size_t off = 0;
    const auto take = [&](size_t bytes) {
        char *q = p + off;
        off += (bytes + 255) / 256 * 256;
        return q;
    };
    s.dots = (double *)take((size_t)ceil_div(e, JOIN_COLS) * sizeof(double));
    s.ticket = (unsigned *)take(sizeof(unsigned));
    s.count_part = (unsigned *)take((size_t)HIST_MAX * (e + 2) * sizeof(unsigned));
    s.col_part = (float *)take(0);
    s.bytes = off;
    return s;
}

int balance_check(const char *what, int n, int e, const void *logits, long long row_stride, int dtype) {
    using w = std::string;
    GDPSO_REQUIRE(n >= 0 && e > 0, w(what) + ": n >= 0 and e > 0 are required");
    GDPSO_REQUIRE(e <= BAL_MAX_E, w(what) + ": more than 16384 experts");
    GDPSO_REQUIRE(dtype_ok(dtype), w(what) + ": unknown element type");
    GDPSO_REQUIRE(n == 0 || logits, w(what) + ": null argument");
    GDPSO_REQUIRE(row_stride >= 0, w(what) + ": negative row stride");
    return GDPSO_OK;
}

template <typename E, bool SUMS, bool GRAD>
int launch_rows(hipStream_t stream, const BalArgs &a, const Choices &ch) {
    const Hold h = hold_row(a.e, vec_of<E>());
    const bool ride = SUMS && !GRAD && h.team;
    const dim3 grid(a.row_blocks + (ride ? ch.blocks : 0));
    // f, or the column sums of a workgroup, or the counters of one that counts
    const size_t lds = std::max((size_t)a.e, ride || a.own_counts ? (size_t)a.e * hist_copies(a.e) : 0) * sizeof(float);
#define BAL_TEAM(T, C) hipLaunchKernelGGL((bal_team_kernel<E, T, C, SUMS, GRAD>), grid, dim3(TEAM_THREADS), lds, stream, a, ch)
    switch (h.team * 16 + h.chunks) {
        case 1 * 16 + 1: BAL_TEAM(1, 1); break;
        case 2 * 16 + 1: BAL_TEAM(2, 1); break;
        case 4 * 16 + 1: BAL_TEAM(4, 1); break;
        case 8 * 16 + 1: BAL_TEAM(8, 1); break;
        case 16 * 16 + 1: BAL_TEAM(16, 1); break;
        case 32 * 16 + 1: BAL_TEAM(32, 1); break;
        case 64 * 16 + 1: BAL_TEAM(64, 1); break;
        case 64 * 16 + 2: BAL_TEAM(64, 2); break;
        case 64 * 16 + 4: BAL_TEAM(64, 4); break;
        case 64 * 16 + 8:
            if constexpr (is_f32<E>()) BAL_TEAM(64, 8);
            break;
        default: hipLaunchKernelGGL((bal_wide_kernel<E, SUMS, GRAD>), grid, dim3(WIDE_THREADS), GRAD ? lds : 0, stream, a); break;
    }
#undef BAL_TEAM
    GDPSO_HIP(hipGetLastError());
    return GDPSO_OK;
}

}  // namespace
}  // namespace gdpso

using namespace gdpso;

extern "C" size_t gdpso_balance_workspace_bytes(int n, int e) {
    if (n < 0 || e <= 0 || e > BAL_MAX_E) return 0;
    const int f32 = row_blocks(n, e, DT_F32), half = row_blocks(n, e, DT_BF16);
    return balance_space(nullptr, e).bytes + (size_t)(f32 > half ? f32 : half) * e * sizeof(float);
}

extern "C" int gdpso_balance(void *stream_, int n, int e, int k, const void *logits, long long row_stride, int dtype, const void *indices,
                             int index_bytes, const unsigned char *mask, float grad_scale, float *loss, long long *counts, long long *totals,
                             float *mean_prob, void *grad, void *workspace, size_t workspace_bytes) {
    int rc = balance_check("balance", n, e, logits, row_stride, dtype);
    if (rc) return rc;
    GDPSO_REQUIRE(k > 0, "balance: k > 0 is required");
    GDPSO_REQUIRE((long long)n * k < (1ll << 32), "balance: 2^32 choices or more in one call");
    GDPSO_REQUIRE(index_bytes == 4 || index_bytes == 8, "balance: indices are 4 or 8 bytes");
    GDPSO_REQUIRE((n == 0 || indices) && loss && counts && totals && mean_prob && workspace, "balance: null argument");
    if (workspace_bytes < gdpso_balance_workspace_bytes(n, e)) return fail(GDPSO_ERR_WORKSPACE, "balance: workspace too small");
    hipStream_t stream = (hipStream_t)stream_;
    const BalSpace ws = balance_space(workspace, e);
    const bool own = grad && e <= TEAM_MAX_E && (long long)n * k <= OWN_CHOICES;
    const bool apart = !own && (grad || e > TEAM_MAX_E);  // the counting as a launch of its own
    const int hb = own ? 1 : hist_blocks((long long)n * k, apart ? HIST_THREADS : TEAM_THREADS);
    const Choices ch = {indices, index_bytes, mask, n, k, e, hb, ws.count_part};
    BalArgs a = {n, e, logits, row_stride, mask, row_blocks(n, e, dtype), ws.col_part, ws.count_part, hb, nullptr, nullptr, grad_scale, nullptr,
                 grad, ws.ticket, own};
    if (apart) {
        hipLaunchKernelGGL(bal_count_kernel, dim3(hb), dim3(HIST_THREADS), (size_t)e * hist_copies(e) * sizeof(unsigned), stream, ch);
        GDPSO_HIP(hipGetLastError());
    }
    if (grad)
        GDPSO_WITH_DTYPE(dtype, rc = (launch_rows<E, true, true>(stream, a, ch)));
    else
        GDPSO_WITH_DTYPE(dtype, rc = (launch_rows<E, true, false>(stream, a, ch)));
    if (rc) return rc;
    hipLaunchKernelGGL(bal_join_kernel, dim3(ceil_div(e, JOIN_COLS)), dim3(JOIN_COLS * JOIN_GROUPS), 0, stream, e, a.row_blocks, ws.col_part, hb,
                       ws.count_part, mean_prob, counts, totals, ws.dots, ws.ticket, loss);
    GDPSO_HIP(hipGetLastError());
    return GDPSO_OK;
}

extern "C" int gdpso_balance_grad(void *stream_, int n, int e, const void *logits, long long row_stride, int dtype, const unsigned char *mask,
                                  const long long *counts, const long long *totals, const float *upstream, void *grad) {
    int rc = balance_check("balance_grad", n, e, logits, row_stride, dtype);
    if (rc) return rc;
    GDPSO_REQUIRE(n == 0 || (counts && totals && upstream && grad), "balance_grad: null argument");
    if (n == 0) return GDPSO_OK;
    const BalArgs a = {n, e, logits, row_stride, mask, row_blocks(n, e, dtype), nullptr, nullptr, 0, counts, totals, 0.f, upstream,
                       grad, nullptr, false};
    GDPSO_WITH_DTYPE(dtype, rc = (launch_rows<E, false, true>((hipStream_t)stream_, a, Choices{})));
    return rc;
}
