// Gradient of LayerNorm for gfx950: dx, dgamma and dbeta from dy, x and the forward pass's mean and rstd; fp32 /
// binary16 / bfloat16 storage, fp32 arithmetic and fp32 dgamma / dbeta.
//
// Per row, with xh = (x - mean) rstd, g = dy gamma, N columns and D = N or N - 1 (the variance's divisor):
//   dx = rstd (g - sum(g) / N - xh sum(g xh) / D) [+ dres],
// and over the rows  dgamma = sum dy xh,  dbeta = sum dy.
//
// Bound: memory - dy and x (and dres) read once, dx written once.  Both directions of sums are taken in the one pass: a
// wavefront or workgroup walks over rows, keeps its columns' share of dgamma and dbeta in registers, and writes one
// fp32 partial row per workgroup into the caller's workspace at its end; a second launch sums the partial rows in a
// fixed order, so results are the same bits from call to call.  The next row's loads are issued before the present
// row's arithmetic.
#include "ko_internal.h"

#include "row_reduce.h"

namespace ko {
namespace {

template <int IO>
struct Args {
    typedef typename Io<IO>::elem Elem;
    const Elem *dy;
    const Elem *x;
    const float *mean;
    const float *rstd;
    const Elem *gamma;
    const Elem *dres;
    Elem *dx;
    float *dgamma;
    float *dbeta;
    int64_t rows;
    int cols;
    float inv_n, inv_d;
    float *partial;  // [workgroups][2][cols], or null: dgamma and dbeta are left to the column kernel
    hipStream_t stream;
};

// One row's (or one lane group's) loads.
template <int IO, int VPL, bool RES>
struct RowLoads {
    typename Io<IO>::raw dy[VPL], x[VPL], res[RES ? VPL : 1];
    float mean, rstd;
};

// Where a workgroup's column sums go: its partial row, or the results themselves when it is the only one.
__device__ __forceinline__ void put_column_sums(float *partial, float *dgamma, float *dbeta, int cols, int column, float sum_g,
                                                float sum_b) {
    if (gridDim.x == 1) {
        if (dgamma) dgamma[column] = sum_g;
        if (dbeta) dbeta[column] = sum_b;
    } else {
        float *mine = partial + static_cast<int64_t>(blockIdx.x) * 2 * cols;
        mine[column] = sum_g;
        mine[cols + column] = sum_b;
    }
}

// ---- a row in the registers of a group of LPR lanes, WAVES wavefronts per workgroup
constexpr int kWaves = 4;
template <int IO, int LPR, int VPL, bool RES>
__global__ __launch_bounds__(64 * kWaves) void layernorm_backward_wave_kernel(Args<IO> a) {
    constexpr int E = Io<IO>::E;
    constexpr int RPW = 64 / LPR;
    typedef typename Io<IO>::elem Elem;
    extern __shared__ float column_sums[];  // [2][cols]
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sub = lane / LPR;
    const int l = lane % LPR;
    const int cols = a.cols;
    const int nvec = cols / E;
    const bool whole_lines = rows_are_whole_lines<IO>(cols);

    typename Io<IO>::raw gamma[VPL];
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
        gamma[k] = typename Io<IO>::raw{};
        if (a.gamma && l + k * LPR < nvec) gamma[k] = Io<IO>::template load_raw<false>(a.gamma + E * (l + k * LPR));
    }
    float acc_g[VPL][E], acc_b[VPL][E];
#pragma unroll
    for (int k = 0; k < VPL; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) acc_g[k][e] = acc_b[k][e] = 0.0f;

    const uint32_t sub_off = static_cast<uint32_t>(sub) * static_cast<uint32_t>(cols) * sizeof(Elem);
    auto fetch = [&](RowLoads<IO, VPL, RES> &r, int64_t row0) {
        const int64_t row = row0 + sub;
        const bool ok = row < a.rows;
        const Elem *dy = a.dy + row0 * cols, *x = a.x + row0 * cols;
        const Elem *res = RES ? a.dres + row0 * cols : nullptr;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int j = l + k * LPR;
            r.dy[k] = r.x[k] = typename Io<IO>::raw{};
            if constexpr (RES) r.res[k] = typename Io<IO>::raw{};
            if (ok && j < nvec) {
                const uint32_t at = sub_off + Io<IO>::kBytes * j;
                r.dy[k] = Io<IO>::template load_raw<true>(byte_offset(dy, at));
                r.x[k] = Io<IO>::template load_raw<true>(byte_offset(x, at));
                if constexpr (RES) r.res[k] = Io<IO>::template load_raw<true>(byte_offset(res, at));
            }
        }
        r.mean = ok ? a.mean[row] : 0.0f;
        r.rstd = ok ? a.rstd[row] : 0.0f;
    };

    const int64_t stride = static_cast<int64_t>(gridDim.x) * kWaves * RPW;
    int64_t row0 = (static_cast<int64_t>(blockIdx.x) * kWaves + wv) * RPW;
    RowLoads<IO, VPL, RES> cur;
    fetch(cur, row0);
    for (; row0 < a.rows; row0 += stride) {
        RowLoads<IO, VPL, RES> next;
        fetch(next, row0 + stride);
        float xh[VPL][E], g[VPL][E];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            float w[E];
            Io<IO>::unpack(cur.x[k], xh[k]);
            Io<IO>::unpack(cur.dy[k], g[k]);
            Io<IO>::unpack(gamma[k], w);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                xh[k][e] = (xh[k][e] - cur.mean) * cur.rstd;
                acc_g[k][e] = __builtin_fmaf(g[k][e], xh[k][e], acc_g[k][e]);
                acc_b[k][e] += g[k][e];
                if (a.gamma) g[k][e] *= w[e];
                s1 += g[k][e];
                s2 = __builtin_fmaf(g[k][e], xh[k][e], s2);
            }
        }
        s1 = wave::allreduce<LPR, wave::Sum>(s1) * a.inv_n;
        s2 = wave::allreduce<LPR, wave::Sum>(s2) * a.inv_d;
        Elem *dst0 = a.dx + row0 * cols;
        const bool ok = row0 + sub < a.rows;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int j = l + k * LPR;
            if (ok && j < nvec) {
                float o[E], res[E];
                if constexpr (RES) Io<IO>::unpack(cur.res[k], res);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    o[e] = cur.rstd * __builtin_fmaf(-xh[k][e], s2, g[k][e] - s1);
                    if constexpr (RES) o[e] += res[e];
                }
                store_row_vec<IO>(whole_lines, dst0, sub_off + Io<IO>::kBytes * j, o);
            }
        }
        cur = next;
    }
    if (!a.partial && !(gridDim.x == 1 && (a.dgamma || a.dbeta))) return;

    // the lane groups' sums, then the wavefronts' in wave order
#pragma unroll
    for (int k = 0; k < VPL; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) {
#pragma unroll
            for (int step = LPR; step < 64; step <<= 1) {
                acc_g[k][e] += __shfl_xor(acc_g[k][e], step, 64);
                acc_b[k][e] += __shfl_xor(acc_b[k][e], step, 64);
            }
        }
    for (int w = 0; w < kWaves; ++w) {
        if (w == wv && sub == 0) {
#pragma unroll
            for (int k = 0; k < VPL; ++k) {
                const int j = l + k * LPR;
                if (j < nvec) {
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        float *at = column_sums + E * j + e;
                        at[0] = w == 0 ? acc_g[k][e] : at[0] + acc_g[k][e];
                        at[cols] = w == 0 ? acc_b[k][e] : at[cols] + acc_b[k][e];
                    }
                }
            }
        }
        __syncthreads();
    }
    for (int c = threadIdx.x; c < cols; c += 64 * kWaves)
        put_column_sums(a.partial, a.dgamma, a.dbeta, cols, c, column_sums[c], column_sums[cols + c]);
}

// ---- a row in the registers of a workgroup.  AHEAD: the next row's loads are issued before this row's arithmetic
// (up to 512 threads; a 1024-thread workgroup has 128 registers per thread, which the sums and one row fill - it also
// converts what it loaded once for the sums and once more for dx).
template <int IO, int THREADS, int VPL, bool RES, bool AHEAD>
__global__ __launch_bounds__(THREADS) void layernorm_backward_block_kernel(Args<IO> a) {
    constexpr int E = Io<IO>::E;
    typedef typename Io<IO>::elem Elem;
    __shared__ float slots[2][THREADS / 64][2];
    const int cols = a.cols;
    const int nvec = cols / E;
    const bool whole_lines = rows_are_whole_lines<IO>(cols);

    typename Io<IO>::raw gamma[VPL];
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
        const int j = threadIdx.x + k * THREADS;
        gamma[k] = typename Io<IO>::raw{};
        if (a.gamma && j < nvec) gamma[k] = Io<IO>::template load_raw<false>(a.gamma + E * j);
    }
    float acc_g[VPL][E], acc_b[VPL][E];
#pragma unroll
    for (int k = 0; k < VPL; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) acc_g[k][e] = acc_b[k][e] = 0.0f;

    auto fetch = [&](RowLoads<IO, VPL, RES> &r, int64_t row) {
        const bool ok = row < a.rows;
        const Elem *dy = a.dy + row * cols, *x = a.x + row * cols;
        const Elem *res = RES ? a.dres + row * cols : nullptr;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int j = threadIdx.x + k * THREADS;
            r.dy[k] = r.x[k] = typename Io<IO>::raw{};
            if constexpr (RES) r.res[k] = typename Io<IO>::raw{};
            if (ok && j < nvec) {
                const uint32_t at = Io<IO>::kBytes * j;
                r.dy[k] = Io<IO>::template load_raw<true>(byte_offset(dy, at));
                r.x[k] = Io<IO>::template load_raw<true>(byte_offset(x, at));
                if constexpr (RES) r.res[k] = Io<IO>::template load_raw<true>(byte_offset(res, at));
            }
        }
        r.mean = ok ? a.mean[row] : 0.0f;
        r.rstd = ok ? a.rstd[row] : 0.0f;
    };

    int64_t row = blockIdx.x;
    int turn = 0;
    RowLoads<IO, VPL, RES> cur;
    if constexpr (AHEAD) fetch(cur, row);
    for (; row < a.rows; row += gridDim.x, turn ^= 1) {
        RowLoads<IO, VPL, RES> next;
        if constexpr (AHEAD) fetch(next, row + gridDim.x);
        else fetch(cur, row);
        float xh[AHEAD ? VPL : 1][E], g[AHEAD ? VPL : 1][E];
        auto convert = [&](int k, float (&xk)[E], float (&gk)[E]) {
            Io<IO>::unpack(cur.x[k], xk);
            Io<IO>::unpack(cur.dy[k], gk);
#pragma unroll
            for (int e = 0; e < E; ++e) xk[e] = (xk[e] - cur.mean) * cur.rstd;
        };
        auto times_gamma = [&](int k, float (&gk)[E]) {
            if (!a.gamma) return;
            float w[E];
            Io<IO>::unpack(gamma[k], w);
#pragma unroll
            for (int e = 0; e < E; ++e) gk[e] *= w[e];
        };
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            float(&xk)[E] = xh[AHEAD ? k : 0], (&gk)[E] = g[AHEAD ? k : 0];
            convert(k, xk, gk);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                acc_g[k][e] = __builtin_fmaf(gk[e], xk[e], acc_g[k][e]);
                acc_b[k][e] += gk[e];
            }
            times_gamma(k, gk);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                s[0] += gk[e];
                s[1] = __builtin_fmaf(gk[e], xk[e], s[1]);
            }
        }
        block_sum<THREADS / 64, 2>(s, slots[turn]);
        const float s1 = s[0] * a.inv_n, s2 = s[1] * a.inv_d;
        Elem *dst = a.dx + row * cols;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int j = threadIdx.x + k * THREADS;
            if (j < nvec) {
                float o[E], res[E];
                float(&xk)[E] = xh[AHEAD ? k : 0], (&gk)[E] = g[AHEAD ? k : 0];
                if constexpr (!AHEAD) {
                    convert_again<IO>(cur.x[k]);
                    convert_again<IO>(cur.dy[k]);
                    convert(k, xk, gk);
                    times_gamma(k, gk);
                }
                if constexpr (RES) Io<IO>::unpack(cur.res[k], res);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    o[e] = cur.rstd * __builtin_fmaf(-xk[e], s2, gk[e] - s1);
                    if constexpr (RES) o[e] += res[e];
                }
                store_row_vec<IO>(whole_lines, dst, Io<IO>::kBytes * j, o);
            }
        }
        if constexpr (AHEAD) cur = next;
    }
    if (!a.partial && !(gridDim.x == 1 && (a.dgamma || a.dbeta))) return;
#pragma unroll
    for (int k = 0; k < VPL; ++k) {
        const int j = threadIdx.x + k * THREADS;
        if (j < nvec) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                put_column_sums(a.partial, a.dgamma, a.dbeta, cols, E * j + e, acc_g[k][e], acc_b[k][e]);
        }
    }
}

// ---- rows of any length: the sums first, then a second read; no share of dgamma and dbeta (the column kernel's)
template <int IO, int THREADS>
__global__ __launch_bounds__(THREADS) void layernorm_backward_reread_kernel(Args<IO> a) {
    constexpr int E = Io<IO>::E;
    constexpr int UNROLL = E == 1 ? 4 : 2;
    typedef typename Io<IO>::elem Elem;
    __shared__ float slots[2][THREADS / 64][2];
    const int cols = a.cols;
    const int nvec = cols / E;
    const bool whole_lines = rows_are_whole_lines<IO>(cols);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, turn ^= 1) {
        const Elem *dy = a.dy + row * cols, *x = a.x + row * cols;
        const float mean = a.mean[row], rstd = a.rstd[row];
        auto sweep = [&](auto use) {
            for (int j0 = threadIdx.x; j0 < nvec; j0 += THREADS * UNROLL) {
                typename Io<IO>::raw rd[UNROLL], rx[UNROLL], rg[UNROLL];
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    const int64_t j = j0 + u * THREADS;
                    rd[u] = rx[u] = rg[u] = typename Io<IO>::raw{};
                    if (j < nvec) {
                        rd[u] = Io<IO>::template load_raw<false>(dy + E * j);
                        rx[u] = Io<IO>::template load_raw<false>(x + E * j);
                        if (a.gamma) rg[u] = Io<IO>::template load_raw<false>(a.gamma + E * j);
                    }
                }
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    float g[E], xh[E], w[E];
                    Io<IO>::unpack(rd[u], g);
                    Io<IO>::unpack(rx[u], xh);
                    Io<IO>::unpack(rg[u], w);
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        xh[e] = (xh[e] - mean) * rstd;
                        if (a.gamma) g[e] *= w[e];
                    }
                    use(j0 + u * THREADS, g, xh);
                }
            }
        };
        float s[2] = {0.0f, 0.0f};
        sweep([&](int, float (&g)[E], float (&xh)[E]) {  // (vectors past the end hold g = 0)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                s[0] += g[e];
                s[1] = __builtin_fmaf(g[e], xh[e], s[1]);
            }
        });
        block_sum<THREADS / 64, 2>(s, slots[turn]);
        const float s1 = s[0] * a.inv_n, s2 = s[1] * a.inv_d;
        Elem *dst = a.dx + row * cols;
        sweep([&](int j, float (&g)[E], float (&xh)[E]) {
            if (j >= nvec) return;
            float res[E];
            if (a.dres) Io<IO>::template load<true>(a.dres + row * cols + static_cast<int64_t>(E) * j, res);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                g[e] = rstd * __builtin_fmaf(-xh[e], s2, g[e] - s1);
                if (a.dres) g[e] += res[e];
            }
            store_row_vec<IO>(whole_lines, dst, Io<IO>::kBytes * static_cast<uint32_t>(j), g);
        });
    }
}

// ---- dgamma and dbeta alone: workgroup (strip, split) sums 64 columns over every gridDim.y-th group of four rows
template <int IO>
__global__ __launch_bounds__(256) void layernorm_backward_columns_kernel(Args<IO> a) {
    __shared__ float sums[2][4][64];
    const int lane = threadIdx.x & 63;
    const int slice = threadIdx.x >> 6;
    const int c = static_cast<int>(blockIdx.x) * 64 + lane;
    float sg = 0.0f, sb = 0.0f;
    if (c < a.cols) {
        constexpr int UNROLL = 4;
        const int64_t step = int64_t{4} * gridDim.y;
        for (int64_t row0 = int64_t{4} * blockIdx.y + slice; row0 < a.rows; row0 += step * UNROLL) {
            float d[UNROLL], xh[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int64_t row = row0 + u * step;
                d[u] = xh[u] = 0.0f;
                if (row < a.rows) {
                    d[u] = Io<IO>::scalar(a.dy + row * a.cols + c);
                    xh[u] = (Io<IO>::scalar(a.x + row * a.cols + c) - a.mean[row]) * a.rstd[row];
                }
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                sg = __builtin_fmaf(d[u], xh[u], sg);
                sb += d[u];
            }
        }
    }
    sums[0][slice][lane] = sg;
    sums[1][slice][lane] = sb;
    __syncthreads();
    if (slice != 0 || c >= a.cols) return;
    sg = (sums[0][0][lane] + sums[0][1][lane]) + (sums[0][2][lane] + sums[0][3][lane]);
    sb = (sums[1][0][lane] + sums[1][1][lane]) + (sums[1][2][lane] + sums[1][3][lane]);
    if (gridDim.y == 1) {
        if (a.dgamma) a.dgamma[c] = sg;
        if (a.dbeta) a.dbeta[c] = sb;
    } else {
        float *mine = a.partial + static_cast<int64_t>(blockIdx.y) * 2 * a.cols;
        mine[c] = sg;
        mine[a.cols + c] = sb;
    }
}

// ---- the sum of the partial rows: a workgroup takes 16 columns of [dgamma, dbeta], 64 threads each
__global__ __launch_bounds__(1024) void layernorm_backward_reduce_kernel(const float *__restrict__ partial, int groups,
                                                                         int cols, float *__restrict__ dgamma,
                                                                         float *__restrict__ dbeta) {
    __shared__ float sums[64][17];
    const int lane = threadIdx.x & 15;
    const int slice = threadIdx.x >> 4;
    const int64_t width = int64_t{2} * cols;
    const int64_t c = int64_t{16} * blockIdx.x + lane;
    float s = 0.0f;
    if (c < width) {
        for (int p = slice; p < groups; p += 64) s += partial[p * width + c];
    }
    sums[slice][lane] = s;
    __syncthreads();
    // a wavefront folds four columns' 64 slices, lane by lane; then its lanes
    const int wv = threadIdx.x >> 6;
    s = wave::allreduce<64, wave::Sum>(sums[threadIdx.x & 63][wv]);
    const int64_t out = int64_t{16} * blockIdx.x + wv;
    if ((threadIdx.x & 63) == 0 && out < width) {
        if (out < cols) {
            if (dgamma) dgamma[out] = s;
        } else if (dbeta) {
            dbeta[out - cols] = s;
        }
    }
}

__global__ __launch_bounds__(256) void layernorm_backward_zero_kernel(float *dgamma, float *dbeta, int cols) {
    for (int c = blockIdx.x * 256 + threadIdx.x; c < cols; c += gridDim.x * 256) {
        if (dgamma) dgamma[c] = 0.0f;
        if (dbeta) dbeta[c] = 0.0f;
    }
}

// ---------------------------------------------------------------------------------------------------- dispatch
// Workgroups that walk over the rows, at most: a function of the sizes alone, so that the workspace can be sized
// without a device.
int64_t max_groups(int64_t rows, int64_t cols) {
    const int64_t most = cols <= 2048 ? 768 : 512;
    return rows < most ? rows : most;
}

// `batches` of rows over at most `most` workgroups, as evenly as whole trips allow.
int64_t even_grid(int64_t batches, int64_t most) {
    if (batches <= most) return batches;
    const int64_t trips = (batches + most - 1) / most;
    return (batches + trips - 1) / trips;
}

template <int IO>
int launch_reduce(const Args<IO> &a, int64_t groups) {
    const unsigned grid = static_cast<unsigned>((int64_t{2} * a.cols + 15) / 16);
    layernorm_backward_reduce_kernel<<<dim3(grid), dim3(1024), 0, a.stream>>>(a.partial, static_cast<int>(groups), a.cols,
                                                                             a.dgamma, a.dbeta);
    KO_CHECK_LAUNCH();
    return KO_OK;
}

// dgamma and dbeta by a pass of their own: for rows too long to keep column sums in registers, and without a workspace.
template <int IO>
int launch_columns(const Args<IO> &a) {
    if (!a.dgamma && !a.dbeta) return KO_OK;
    const int64_t strips = (a.cols + 63) / 64;
    int64_t splits = 1;
    if (a.partial) {
        splits = 2048 / strips;
        if (splits > (a.rows + 15) / 16) splits = (a.rows + 15) / 16;
        if (splits > max_groups(a.rows, a.cols)) splits = max_groups(a.rows, a.cols);
        if (splits < 1) splits = 1;
    }
    layernorm_backward_columns_kernel<IO><<<dim3(static_cast<unsigned>(strips), static_cast<unsigned>(splits)), dim3(256), 0,
                                            a.stream>>>(a);
    KO_CHECK_LAUNCH();
    return splits > 1 ? launch_reduce(a, splits) : KO_OK;
}

// Who sums dgamma and dbeta next to a launch of `grid` row-walking workgroups: the workgroups themselves, through the
// workspace; without one the column kernel, ahead of them (dx may overwrite dy or x).
template <int IO>
int columns_first(const Args<IO> &a, int64_t grid) {
    return grid > 1 && !a.partial ? launch_columns(a) : KO_OK;
}
template <int IO>
int reduce_last(const Args<IO> &a, int64_t grid) {
    return grid > 1 && a.partial ? launch_reduce(a, grid) : KO_OK;
}

template <int IO, int LPR, int VPL>
int launch_wave(const Args<IO> &a) {
    constexpr int64_t kRows = kWaves * (64 / LPR);
    const int64_t grid = even_grid((a.rows + kRows - 1) / kRows, max_groups(a.rows, a.cols));
    if (const int st = columns_first(a, grid); st != KO_OK) return st;
    const size_t lds = static_cast<size_t>(2) * a.cols * sizeof(float);
    const dim3 g(static_cast<unsigned>(grid)), b(64 * kWaves);
    if (a.dres) layernorm_backward_wave_kernel<IO, LPR, VPL, true><<<g, b, lds, a.stream>>>(a);
    else layernorm_backward_wave_kernel<IO, LPR, VPL, false><<<g, b, lds, a.stream>>>(a);
    KO_CHECK_LAUNCH();
    return reduce_last(a, grid);
}

template <int IO, int THREADS, int VPL>
int launch_block(const Args<IO> &a) {
    constexpr bool kAhead = THREADS < 1024;
    const int64_t grid = even_grid(a.rows, max_groups(a.rows, a.cols));
    if (const int st = columns_first(a, grid); st != KO_OK) return st;
    const dim3 g(static_cast<unsigned>(grid)), b(THREADS);
    if (a.dres) layernorm_backward_block_kernel<IO, THREADS, VPL, true, kAhead><<<g, b, 0, a.stream>>>(a);
    else layernorm_backward_block_kernel<IO, THREADS, VPL, false, kAhead><<<g, b, 0, a.stream>>>(a);
    KO_CHECK_LAUNCH();
    return reduce_last(a, grid);
}

template <int IO>
int launch_long(const Args<IO> &a) {
    if (const int st = launch_columns(a); st != KO_OK) return st;  // (dx may overwrite dy or x)
    const int64_t grid = a.rows > 0x7fffffff ? 0x7fffffff : a.rows;
    layernorm_backward_reread_kernel<IO, 1024><<<dim3(static_cast<unsigned>(grid)), dim3(1024), 0, a.stream>>>(a);
    KO_CHECK_LAUNCH();
    return KO_OK;
}

template <int IO>
int dispatch(const Args<IO> &a) {
    constexpr int E = Io<IO>::E;
    const int nvec = a.cols / E;
    if constexpr (E == 1) {
        if (nvec <= 16) return launch_wave<IO, 16, 1>(a);
        if (nvec <= 64) return launch_wave<IO, 64, 1>(a);
        if (nvec <= 128) return launch_wave<IO, 64, 2>(a);
        if (nvec <= 256) return launch_wave<IO, 64, 4>(a);
        if (nvec <= 512) return launch_wave<IO, 64, 8>(a);
        if (nvec <= 1024) return launch_wave<IO, 64, 16>(a);
        if (nvec <= 2048) return launch_block<IO, 512, 4>(a);
        if (nvec <= 4096) return launch_block<IO, 512, 8>(a);
        if (nvec <= 8192) return launch_block<IO, 1024, 8>(a);
    } else {
        int lpr = 0, vpl = 0;
        if (choose_row_group(nvec, 4, &lpr, &vpl)) {
#define KO_WAVE(L, V) if (lpr == L && vpl == V) return launch_wave<IO, L, V>(a)
            KO_WAVE(8, 1); KO_WAVE(8, 2); KO_WAVE(8, 3);
            KO_WAVE(16, 1); KO_WAVE(16, 2); KO_WAVE(16, 3);
            KO_WAVE(32, 1); KO_WAVE(32, 2); KO_WAVE(32, 3);
            KO_WAVE(64, 1); KO_WAVE(64, 2); KO_WAVE(64, 3); KO_WAVE(64, 4);
#undef KO_WAVE
        }
        if (nvec <= 512) return launch_block<IO, 256, 2>(a);
        if (nvec <= 1024) return launch_block<IO, 512, 2>(a);
        if (nvec <= 2048) return launch_block<IO, 1024, 2>(a);
        if constexpr (E == 4) {
            if (nvec <= 4096) return launch_block<IO, 1024, 4>(a);
        }
    }
    return launch_long(a);
}

size_t workspace_bytes(int64_t rows, int64_t cols) {
    if (rows <= 1 || cols <= 0 || cols > (1 << 30)) return 0;
    return static_cast<size_t>(max_groups(rows, cols)) * 2 * static_cast<size_t>(cols) * sizeof(float);
}

template <int IO>
int entry(const void *dy, const void *x, const float *mean, const float *rstd, const void *gamma, const void *dres, void *dx,
          float *dgamma, float *dbeta, int64_t rows, int64_t cols, int unbiased, void *workspace, size_t bytes,
          ko_stream_t stream) {
    typedef typename Io<IO>::elem Elem;
    if (rows < 0 || cols <= 0)
        return fail(KO_ERR_INVALID_ARGUMENT, "layernorm_backward: rows=%lld cols=%lld", (long long)rows, (long long)cols);
    if (cols > (1 << 30)) return fail(KO_ERR_UNSUPPORTED_SHAPE, "layernorm_backward: cols=%lld too large", (long long)cols);
    if (rows > 0 && (!dy || !x || !mean || !rstd || !dx))
        return fail(KO_ERR_INVALID_ARGUMENT, "layernorm_backward: null dy/in/mean/rstd/dx pointer");
    const uintptr_t rows_at = reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(x) |
                              reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(gamma) |
                              reinterpret_cast<uintptr_t>(dres);
    if (rows_at & (sizeof(Elem) - 1))
        return fail(KO_ERR_INVALID_ARGUMENT, "layernorm_backward: dy/in/gamma/dres/dx must be aligned to their element type");
    if ((reinterpret_cast<uintptr_t>(mean) | reinterpret_cast<uintptr_t>(rstd) | reinterpret_cast<uintptr_t>(dgamma) |
         reinterpret_cast<uintptr_t>(dbeta)) & 3)
        return fail(KO_ERR_INVALID_ARGUMENT, "layernorm_backward: mean/rstd/dgamma/dbeta must be 4-byte aligned");
    if (workspace && bytes < workspace_bytes(rows, cols))
        return fail(KO_ERR_INVALID_ARGUMENT, "layernorm_backward: workspace of %zu bytes, %zu needed", bytes, workspace_bytes(rows, cols));
    if (reinterpret_cast<uintptr_t>(workspace) & 15)
        return fail(KO_ERR_INVALID_ARGUMENT, "layernorm_backward: workspace must be 16-byte aligned");
    if (rows == 0) {  // the sum over no rows
        if (!dgamma && !dbeta) return KO_OK;
        int64_t grid = (cols + 255) / 256;
        if (grid > 1024) grid = 1024;
        layernorm_backward_zero_kernel<<<dim3(static_cast<unsigned>(grid)), dim3(256), 0, as_stream(stream)>>>(
            dgamma, dbeta, static_cast<int>(cols));
        KO_CHECK_LAUNCH();
        return KO_OK;
    }
    const float inv_n = 1.0f / static_cast<float>(cols);
    const float inv_d = unbiased ? 1.0f / static_cast<float>(cols - 1) : inv_n;
    float *partial = (dgamma || dbeta) ? static_cast<float *>(workspace) : nullptr;
    auto run = [&](auto kind) {
        constexpr int KIND = decltype(kind)::value;
        const Args<KIND> a{static_cast<const Elem *>(dy), static_cast<const Elem *>(x), mean, rstd,
                           static_cast<const Elem *>(gamma), static_cast<const Elem *>(dres), static_cast<Elem *>(dx), dgamma,
                           dbeta, rows, static_cast<int>(cols), inv_n, inv_d, partial, as_stream(stream)};
        return dispatch<KIND>(a);
    };
    // rows that do not start on 16-byte boundaries are walked element by element
    if (cols % Io<IO>::E != 0 || (rows_at & 15) != 0) return run(std::integral_constant<int, io_by_element(IO)>{});
    return run(std::integral_constant<int, IO>{});
}

}  // namespace
}  // namespace ko

KO_EXPORT size_t ko_layernorm_backward_workspace_bytes(int64_t rows, int64_t cols) { return ko::workspace_bytes(rows, cols); }

KO_EXPORT int ko_layernorm_backward_f32(const float *dy, const float *in, const float *mean, const float *rstd,
                                        const float *gamma, const float *dres, float *dx, float *dgamma, float *dbeta,
                                        int64_t rows, int64_t cols, int unbiased, void *workspace, size_t workspace_bytes,
                                        ko_stream_t stream) {
    return ko::entry<ko::IO_F32>(dy, in, mean, rstd, gamma, dres, dx, dgamma, dbeta, rows, cols, unbiased, workspace,
                                 workspace_bytes, stream);
}

KO_EXPORT int ko_layernorm_backward_16(const void *dy, const void *in, const float *mean, const float *rstd, const void *gamma,
                                       const void *dres, void *dx, float *dgamma, float *dbeta, int64_t rows, int64_t cols,
                                       int unbiased, int dtype, void *workspace, size_t workspace_bytes, ko_stream_t stream) {
    if (dtype == KO_F16)
        return ko::entry<ko::IO_F16>(dy, in, mean, rstd, gamma, dres, dx, dgamma, dbeta, rows, cols, unbiased, workspace,
                                     workspace_bytes, stream);
    if (dtype == KO_BF16)
        return ko::entry<ko::IO_BF16>(dy, in, mean, rstd, gamma, dres, dx, dgamma, dbeta, rows, cols, unbiased, workspace,
                                      workspace_bytes, stream);
    return ko::fail(KO_ERR_INVALID_ARGUMENT, "layernorm_backward: dtype=%d is neither KO_F16 nor KO_BF16", dtype);
}
