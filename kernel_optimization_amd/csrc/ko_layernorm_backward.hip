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
    float *partial;  // [row workgroups][2][cols], or null: dgamma and dbeta are left to others
    hipStream_t stream;
    int row_groups;  // workgroups of the launch that walk over rows
};

// dgamma and dbeta of a strip of COLUMNS columns alone, by a workgroup: THREADS / COLUMNS slices of the rows from `first` on, every
// `step`-th row, side by side, then folded in order.  The sums come back in the first COLUMNS threads.  Sum: what eight rows'
// sums in 32 bits are added up in; without a workspace a thread goes through a quarter of all rows, and 196608 additions in 32 bits
// of terms of one sign were off by 190 half steps.
template <int IO, int THREADS, int COLUMNS, class Sum>
__device__ __forceinline__ void column_strip(const Args<IO> &a, int strip, int64_t split, int64_t splits, float &sum_g, float &sum_b) {
    constexpr int SLICES = THREADS / COLUMNS;
    constexpr int UNROLL = 8;
    __shared__ Sum sums[2][SLICES][COLUMNS + 1];
    const int lane = threadIdx.x % COLUMNS;
    const int slice = threadIdx.x / COLUMNS;
    const int c = strip * COLUMNS + lane;
    Sum sg = 0, sb = 0;
    if (c < a.cols) {
        const int64_t step = SLICES * splits;
        for (int64_t row0 = SLICES * split + slice; row0 < a.rows; row0 += step * UNROLL) {
            // (beyond the last row: the last one, counted as nothing; loads under conditions, or next to their use, wait one by one)
            typename Io<IO>::elem dy[UNROLL], x[UNROLL];
            float mean[UNROLL], rstd[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int64_t row = row0 + u * step < a.rows ? row0 + u * step : a.rows - 1;
                dy[u] = a.dy[row * a.cols + c];
                x[u] = a.x[row * a.cols + c];
                mean[u] = a.mean[row];
                rstd[u] = a.rstd[row];
            }
            asm volatile("" ::: "memory");
            float d[UNROLL], xh[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const bool here = row0 + u * step < a.rows;
                d[u] = here ? Io<IO>::scalar(&dy[u]) : 0.0f;
                xh[u] = here ? (Io<IO>::scalar(&x[u]) - mean[u]) * rstd[u] : 0.0f;
            }
            float g = 0.0f, b = 0.0f;
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                g = __builtin_fmaf(d[u], xh[u], g);
                b += d[u];
            }
            sg += g;
            sb += b;
        }
    }
    sums[0][slice][lane] = sg;
    sums[1][slice][lane] = sb;
    __syncthreads();
    if (threadIdx.x >= COLUMNS) return;
    sg = sb = 0;
#pragma unroll 8
    for (int i = 0; i < SLICES; ++i) {
        sg += sums[0][i][lane];
        sb += sums[1][i][lane];
    }
    sum_g = static_cast<float>(sg);
    sum_b = static_cast<float>(sb);
}

// A strip over all rows, to the results: the few-rows form.
constexpr int kStripColumns = 16;
template <int IO, int THREADS>
__device__ __forceinline__ void whole_strip(const Args<IO> &a, int strip) {
    float sum_g, sum_b;
    column_strip<IO, THREADS, kStripColumns, float>(a, strip, 0, 1, sum_g, sum_b);  // (few rows)
    const int c = strip * kStripColumns + threadIdx.x;
    if (threadIdx.x < kStripColumns && c < a.cols) {
        if (a.dgamma) a.dgamma[c] = sum_g;
        if (a.dbeta) a.dbeta[c] = sum_b;
    }
}
template <int IO, int THREADS>
__global__ __launch_bounds__(THREADS) void layernorm_backward_strips_kernel(Args<IO> a) {
    whole_strip<IO, THREADS>(a, blockIdx.x);
}

// One batch of rows as a thread loads it.
template <int IO, int VPL, bool RES>
struct RowLoads {
    typename Io<IO>::raw dy[VPL], x[VPL], res[RES ? VPL : 1];
    float mean, rstd;
};

// Four floats at any address of a float.
typedef float4v float4_any __attribute__((aligned(4)));

// ---- a row in registers: of LPR lanes of a wavefront (LPR <= 64, 64 / LPR rows per wavefront, kWaves wavefronts per
// workgroup), or of a workgroup of LPR threads; VPL vectors per thread, VPL = ceil(vectors / LPR).
// A wavefront or workgroup walks over batches of rows, one row per lane group.  The next batch's loads are issued before
// the present one's arithmetic (up to 512 threads: a 1024-thread workgroup has 128 registers per thread, which the sums
// and one row fill; it also converts what it loaded once for the sums and once more for dx), and nothing in the loop is loaded or stored under a condition (see load_whole):
//   - threads beyond a row's last whole vector take the row's last 16 bytes again; they store what the others store
//     there, and leave out of the sums the columns that they share with others (FULL: there are none);
//   - lane groups beyond the last row take the last row again, which is in their own batch, likewise.
constexpr int kWaves = 4;
template <int LPR>
constexpr int group_threads() {
    return LPR > 64 ? LPR : 64 * kWaves;
}
template <int IO, int LPR, int VPL, bool RES, bool FULL>
__global__ __launch_bounds__(group_threads<LPR>(), LPR == 1024 ? 4 : LPR <= 64 && VPL * Io<IO>::E >= 24 ? 1 : 2) void layernorm_backward_rows_kernel(Args<IO> a) {
    constexpr int E = Io<IO>::E;
    constexpr int THREADS = group_threads<LPR>();
    constexpr bool BLOCK = LPR > 64;       // a workgroup per row
    constexpr bool AHEAD = LPR < 1024;
    constexpr int RPB = BLOCK ? 1 : 64 / LPR;  // rows per batch
    typedef typename Io<IO>::elem Elem;
    typedef RowLoads<IO, VPL, RES> Loads;
    __shared__ float slots[2][THREADS / 64][2];
    const int wv = BLOCK ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sub = BLOCK ? 0 : (threadIdx.x & 63) / LPR;
    const int l = threadIdx.x % LPR;
    const int cols = a.cols;
    if (static_cast<int>(blockIdx.x) >= a.row_groups) {
        // few rows: dgamma and dbeta by workgroups of their own in the same launch (see launch_rows)
        whole_strip<IO, THREADS>(a, static_cast<int>(blockIdx.x) - a.row_groups);
        return;
    }
    const uint32_t row_bytes = static_cast<uint32_t>(cols) * sizeof(Elem);

    // vector k of this thread starts `vec_at(k)` bytes into its row; the last one's first `seen` columns are another
    // thread's, too
    uint32_t last_at = Io<IO>::kBytes * (l + (VPL - 1) * LPR);
    int seen = 0;
    if constexpr (!FULL) {
        const uint32_t most = row_bytes - Io<IO>::kBytes;
        if (last_at > most) {
            const uint32_t past = (last_at - most) / sizeof(Elem);
            seen = past < E ? static_cast<int>(past) : E;
            last_at = most;
        }
    }
    auto vec_at = [&](int k) { return k + 1 < VPL ? Io<IO>::kBytes * static_cast<uint32_t>(l + k * LPR) : last_at; };

    typename Io<IO>::raw gamma[VPL];
    float one[E];
#pragma unroll
    for (int e = 0; e < E; ++e) one[e] = 1.0f;
#pragma unroll
    for (int k = 0; k < VPL; ++k) gamma[k] = a.gamma ? load_whole<IO, FULL>(a.gamma, vec_at(k)) : pack<IO>(one);
    float acc_g[VPL][E], acc_b[VPL][E];
#pragma unroll
    for (int k = 0; k < VPL; ++k)
#pragma unroll
        for (int e = 0; e < E; ++e) acc_g[k][e] = acc_b[k][e] = 0.0f;

    // batch t of this walker
    const int64_t walkers = BLOCK ? a.row_groups : static_cast<int64_t>(a.row_groups) * kWaves;
    const int64_t first = BLOCK ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * kWaves + wv;
    const int64_t batches = (a.rows + RPB - 1) / RPB;
    const int64_t n = first < batches ? (batches - first + walkers - 1) / walkers : 0;
    auto row_of = [&](int64_t t) { return (first + t * walkers) * RPB; };
    // the lane group's row within the batch at row0, the last row's batch having fewer
    auto row_in_batch = [&](int64_t row0) {
        const int64_t left = a.rows - row0;
        return RPB > 1 && left < RPB && sub >= left ? static_cast<int>(left) - 1 : sub;
    };

    auto fetch = [&](Loads &r, int64_t t) {
        const int64_t row0 = row_of(t);
        const int in_batch = row_in_batch(row0);
        const Elem *dy = a.dy + row0 * cols, *x = a.x + row0 * cols, *res = RES ? a.dres + row0 * cols : nullptr;
        const uint32_t at = static_cast<uint32_t>(in_batch) * row_bytes;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            r.dy[k] = load_whole<IO, FULL>(dy, at + vec_at(k));
            r.x[k] = load_whole<IO, FULL>(x, at + vec_at(k));
            if constexpr (RES) r.res[k] = load_whole<IO, FULL>(res, at + vec_at(k));
        }
        r.mean = a.mean[row0 + in_batch];
        r.rstd = a.rstd[row0 + in_batch];
        asm volatile("" ::: "memory");  // the loads stay ahead of what follows
    };

    // LAST: the batch may be the one with lane groups beyond the last row
    // One vector converted: xh and g = dy; then, the column sums taken of them, g times gamma.
    auto convert = [&](const Loads &cur, int k, float (&xh)[E], float (&g)[E]) {
        Io<IO>::unpack(cur.x[k], xh);
        Io<IO>::unpack(cur.dy[k], g);
#pragma unroll
        for (int e = 0; e < E; ++e) xh[e] = (xh[e] - cur.mean) * cur.rstd;
    };
    auto times_gamma = [&](int k, float (&g)[E]) {
        if constexpr (!AHEAD) convert_again<IO>(gamma[k]);
        float w[E];
        Io<IO>::unpack(gamma[k], w);
#pragma unroll
        for (int e = 0; e < E; ++e) g[e] *= w[e];
    };
    auto finish = [&](Loads &cur, int64_t t, auto last) {
        constexpr bool LAST = decltype(last)::value && RPB > 1;
        const int64_t row0 = row_of(t);
        const int in_batch = LAST ? row_in_batch(row0) : sub;
        if constexpr (AHEAD) {
            // what this batch loaded is looked at from here on only: conversions moved up between the next batch's
            // addresses would have the wavefront wait for this batch before it asks for the next one
#pragma unroll
            for (int k = 0; k < VPL; ++k) asm volatile("" : "+v"(cur.dy[k]), "+v"(cur.x[k]));
        }
        float xh[AHEAD ? VPL : 1][E], g[AHEAD ? VPL : 1][E];
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            float(&xk)[E] = xh[AHEAD ? k : 0], (&gk)[E] = g[AHEAD ? k : 0];
            convert(cur, k, xk, gk);
            float up[E];  // dy of the columns that this thread counts
#pragma unroll
            for (int e = 0; e < E; ++e) {
                up[e] = gk[e];
                if constexpr (!FULL) {
                    if (k + 1 == VPL) up[e] = e >= seen ? up[e] : 0.0f;
                }
                if constexpr (LAST) up[e] = in_batch == sub ? up[e] : 0.0f;
                acc_g[k][e] = __builtin_fmaf(up[e], xk[e], acc_g[k][e]);
                acc_b[k][e] += up[e];
            }
            times_gamma(k, gk);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                float gs = gk[e];
                if constexpr (!FULL) {
                    if (k + 1 == VPL) gs = e >= seen ? gs : 0.0f;
                }
                s[0] += gs;
                s[1] = __builtin_fmaf(gs, xk[e], s[1]);
            }
        }
        if constexpr (BLOCK) {
            if constexpr (RES && !FULL) {
                // dx may be dres, and a row's last 16 bytes are several threads': all of them have read before one writes
#pragma unroll
                for (int k = 0; k < VPL; ++k) asm volatile("" : "+v"(cur.res[k]));
            }
            block_sum<THREADS / 64, 2>(s, slots[t & 1]);
        } else {
            s[0] = wave::allreduce<LPR, wave::Sum>(s[0]);
            s[1] = wave::allreduce<LPR, wave::Sum>(s[1]);
        }
        const float s1 = s[0] * a.inv_n, s2 = s[1] * a.inv_d;
        Elem *dx = a.dx + row0 * cols;
        const uint32_t at = static_cast<uint32_t>(in_batch) * row_bytes;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            float o[E], res[E];
            float(&xk)[E] = xh[AHEAD ? k : 0], (&gk)[E] = g[AHEAD ? k : 0];
            if constexpr (!AHEAD) {
                convert_again<IO>(cur.x[k]);
                convert_again<IO>(cur.dy[k]);
                convert(cur, k, xk, gk);
                times_gamma(k, gk);
            }
            if constexpr (RES) Io<IO>::unpack(cur.res[k], res);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                o[e] = cur.rstd * __builtin_fmaf(-xk[e], s2, gk[e] - s1);
                if constexpr (RES) o[e] += res[e];
            }
            store_whole<IO, FULL>(dx, at + vec_at(k), o);
        }
    };
    typedef std::integral_constant<bool, false> Whole;
    typedef std::integral_constant<bool, true> Last;

    // Two sets of registers in turn (moving one into the other would wait for its loads).  The loop is entered the way
    // it comes round, with one set's loads and the other's stores on their way, so that its waits can be exact.
    if constexpr (!AHEAD) {
        Loads only;
        for (int64_t t = 0; t < n; ++t) {
            fetch(only, t);
            finish(only, t, Whole{});
        }
    } else if (n > 0) {
        Loads even, odd;
        int64_t t = 0;
        fetch(even, 0);
        if (n > 1) {
            fetch(odd, 1);
            finish(even, 0, Whole{});
            for (t = 1; t + 2 < n; t += 2) {
                fetch(even, t + 1);
                finish(odd, t, Whole{});
                fetch(odd, t + 2);
                finish(even, t + 1, Whole{});
            }
            if (t + 1 < n) {
                fetch(even, t + 1);
                finish(odd, t, Whole{});
                ++t;
            } else {
                even = odd;
            }
        }
        finish(even, t, Last{});
    }
    // Where this workgroup's column sums go: its partial row, or the results themselves when it is the only one.
    float *to_g = a.dgamma, *to_b = a.dbeta;
    if (a.row_groups > 1) {
        if (!a.partial) return;
        to_g = a.partial + static_cast<int64_t>(blockIdx.x) * 2 * cols;
        to_b = to_g + cols;
    } else if (!to_g && !to_b) {
        return;
    }
    // the columns of vector k that this thread counts, at base + column
    auto put = [&](float *base, int k, const float (&v)[E]) {
        float *at = base + vec_at(k) / sizeof(Elem);
        if (FULL || k + 1 < VPL || seen == 0) {
#pragma unroll
            for (int e = 0; e < E; e += 4)
                *reinterpret_cast<float4_any *>(at + e) = float4v{v[e], v[e + 1], v[e + 2], v[e + 3]};
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e >= seen) at[e] = v[e];
        }
    };
    if constexpr (BLOCK) {
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            if (to_g) put(to_g, k, acc_g[k]);
            if (to_b) put(to_b, k, acc_b[k]);
        }
    } else {
        // every lane group's sums side by side in LDS, then added in order, column by column
        constexpr int GROUPS = kWaves * RPB;
        extern __shared__ float column_sums[];  // [GROUPS][2][cols]
        float *mine = column_sums + (wv * RPB + sub) * 2 * cols;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            put(mine, k, acc_g[k]);
            put(mine + cols, k, acc_b[k]);
        }
        __syncthreads();
        for (int c = threadIdx.x; c < 2 * cols; c += THREADS) {
            float sum = 0.0f;
#pragma unroll 8
            for (int i = 0; i < GROUPS; ++i) sum += column_sums[i * 2 * cols + c];
            float *to = c < cols ? to_g : to_b;
            if (to) to[c < cols ? c : c - cols] = sum;
        }
    }
}

// ---- rows of any length: the sums first, then a second read; no share of dgamma and dbeta (the column kernel's): dy and x are
// read three times where those are wanted (1 GiB of bf16 rows of 20000 columns 1137 us, 2.8 TB/s of dy, x and dx; 40000 columns 1230)
template <int IO, int THREADS, bool RAGGED>
__global__ __launch_bounds__(THREADS) void layernorm_backward_reread_kernel(Args<IO> a) {
    constexpr int E = Io<IO>::E;
    constexpr int UNROLL = 2;
    typedef typename Io<IO>::elem Elem;
    __shared__ float slots[2][THREADS / 64][2];
    const int cols = a.cols;
    const int nvec = row_vectors<IO, RAGGED>(cols);
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
                    const int j = j0 + u * THREADS;
                    rd[u] = rx[u] = rg[u] = typename Io<IO>::raw{};
                    if (j < nvec) {
                        rd[u] = load_row_vec<IO, RAGGED, false>(dy, 0, j, cols);
                        rx[u] = load_row_vec<IO, RAGGED, false>(x, 0, j, cols);
                        if (a.gamma) rg[u] = load_row_vec<IO, RAGGED, false>(a.gamma, 0, j, cols);
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
            if (a.dres) Io<IO>::unpack(load_row_vec<IO, RAGGED, true>(a.dres + row * cols, 0, j, cols), res);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                g[e] = rstd * __builtin_fmaf(-xh[e], s2, g[e] - s1);
                if (a.dres) g[e] += res[e];
            }
            store_row_vec_any<IO, RAGGED>(whole_lines, dst, 0, j, cols, g);
        });
    }
}

// ---- dgamma and dbeta alone: workgroup (strip, split) takes 64 columns and every gridDim.y-th group of rows.  Without
// a workspace there is one split, and a few workgroups read everything (16384 x 768 bf16 0.57 ms; with one 17 us in all).
template <int IO>
__global__ __launch_bounds__(256) void layernorm_backward_columns_kernel(Args<IO> a) {
    float sg, sb;
    column_strip<IO, 256, 64, double>(a, blockIdx.x, blockIdx.y, gridDim.y, sg, sb);
    const int c = static_cast<int>(blockIdx.x) * 64 + threadIdx.x;
    if (threadIdx.x >= 64 || c >= a.cols) return;
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
        constexpr int UNROLL = 4;
        for (int p0 = slice; p0 < groups; p0 += 64 * UNROLL) {
            float v[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) v[u] = p0 + 64 * u < groups ? partial[(p0 + 64 * u) * width + c] : 0.0f;
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) s += v[u];
        }
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
constexpr int64_t kUnits = 256;  // compute units of an MI355X
constexpr int64_t kFewRows = 256;
constexpr int64_t kMostColumns = 16384;  // of a row that a workgroup's registers hold
int64_t max_groups(int64_t rows) {
    return rows < 2 * kUnits ? rows : 2 * kUnits;
}
// Groups of rows that the column kernel takes side by side: some 2048 workgroups in all, sixteen rows and more each.
int64_t column_splits(int64_t rows, int64_t cols) {
    int64_t splits = 2048 / ((cols + 63) / 64);
    if (splits > (rows + 15) / 16) splits = (rows + 15) / 16;
    if (splits > max_groups(rows)) splits = max_groups(rows);
    return splits < 1 ? 1 : splits;
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
    const int64_t splits = a.partial ? column_splits(a.rows, a.cols) : 1;
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

template <int IO, int LPR, int VPL, bool FULL>
int launch_rows(Args<IO> a) {
    constexpr int THREADS = group_threads<LPR>();
    constexpr int64_t kRows = LPR > 64 ? 1 : kWaves * (64 / LPR);  // per workgroup and trip
    // One workgroup per compute unit: with the next batch's loads always on their way, more of them only spread the
    // addresses in flight (65536 x 4096 bf16 with dres: one 363 us, two 388, three 414).  Two where a workgroup's batch is
    // 8 KB or less (98304 x 1024 fp32: one 5.4 TB/s, two 5.9).
    const bool light = THREADS * VPL * 16 * (a.dres ? 3 : 2) <= 8192;
    const int64_t grid = even_grid((a.rows + kRows - 1) / kRows, light ? 2 * kUnits : kUnits);
    a.row_groups = static_cast<int>(grid);
    // Few rows: no second launch.  Workgroups of the same launch read the rows once more, from the caches, for dgamma and
    // dbeta (in a graph, 128 x 768 fp32 5.8 -> 3.2 us, 256 x 4096 bf16 13.1 -> 5.2, 256 x 128 bf16 5.1 -> 4.5; at 512 rows 7.5
    // against 7.4, 13.9 against 14.8 and 5.1 against 7.1).  Where dx overwrites what they read, they come first, in a launch of
    // their own, which gives the same bits.
    int strips = 0;
    if ((a.dgamma || a.dbeta) && grid > 1 && a.rows <= kFewRows) {
        a.partial = nullptr;
        strips = (a.cols + kStripColumns - 1) / kStripColumns;
        if (a.dx == a.dy || a.dx == a.x) {
            layernorm_backward_strips_kernel<IO, THREADS><<<dim3(static_cast<unsigned>(strips)), dim3(THREADS), 0, a.stream>>>(a);
            KO_CHECK_LAUNCH();
            strips = 0;
        }
    } else if (const int st = columns_first(a, grid); st != KO_OK) {
        return st;
    }
    const size_t lds = LPR > 64 ? 0 : static_cast<size_t>(kRows) * 2 * a.cols * sizeof(float);  // 48 KB at most
    const dim3 g(static_cast<unsigned>(grid + strips)), b(THREADS);
    if (a.dres) layernorm_backward_rows_kernel<IO, LPR, VPL, true, FULL><<<g, b, lds, a.stream>>>(a);
    else layernorm_backward_rows_kernel<IO, LPR, VPL, false, FULL><<<g, b, lds, a.stream>>>(a);
    KO_CHECK_LAUNCH();
    return reduce_last(a, grid);
}

template <int IO, int LPR, int VPL>
int launch_rows_any(const Args<IO> &a, bool whole) {
    if (whole && a.cols == LPR * VPL * Io<IO>::E) return launch_rows<IO, LPR, VPL, true>(a);
    return launch_rows<IO, LPR, VPL, false>(a);
}

template <int IO, int THREADS, bool RAGGED>
int launch_long(const Args<IO> &a) {
    if (const int st = launch_columns(a); st != KO_OK) return st;  // (dx may overwrite dy or x)
    layernorm_backward_reread_kernel<IO, THREADS, RAGGED><<<row_grid(a.rows, THREADS), dim3(THREADS), 0, a.stream>>>(a);
    KO_CHECK_LAUNCH();
    return KO_OK;
}

// `whole`: rows of whole 16-byte vectors on 16-byte boundaries
template <int IO>
int dispatch(const Args<IO> &a, bool whole) {
    const int nvec = (a.cols + Io<IO>::E - 1) / Io<IO>::E;
    if (a.cols < Io<IO>::E) return launch_long<IO, 64, true>(a);  // (shorter than a vector)
    int lpr = 0, vpl = 0;
    if (choose_row_group(nvec, 3, &lpr, &vpl)) {
#define KO_WAVE(L, V) if (lpr == L && vpl == V) return launch_rows_any<IO, L, V>(a, whole)
        KO_WAVE(8, 1); KO_WAVE(8, 2); KO_WAVE(8, 3);
        KO_WAVE(16, 1); KO_WAVE(16, 2); KO_WAVE(16, 3);
        KO_WAVE(32, 1); KO_WAVE(32, 2); KO_WAVE(32, 3);
        KO_WAVE(64, 1); KO_WAVE(64, 2); KO_WAVE(64, 3);
#undef KO_WAVE
    }
    if (nvec <= 256) return launch_rows_any<IO, 256, 1>(a, whole);
    if (nvec <= 512) return launch_rows_any<IO, 256, 2>(a, whole);
    if (nvec <= 1024) return launch_rows_any<IO, 512, 2>(a, whole);
    if (nvec <= 2048) return launch_rows_any<IO, 1024, 2>(a, whole);
    if constexpr (Io<IO>::E == 4) {
        if (nvec <= 3 * 1024) return launch_rows_any<IO, 1024, 3>(a, whole);
        if (nvec <= 4096) return launch_rows_any<IO, 1024, 4>(a, whole);
    }
    return whole ? launch_long<IO, 1024, false>(a) : launch_long<IO, 1024, true>(a);
}

size_t workspace_bytes(int64_t rows, int64_t cols) {
    if (rows <= 1 || cols <= 0 || cols > kMaxColumns) return 0;
    const int64_t groups = cols <= kMostColumns ? max_groups(rows) : column_splits(rows, cols);
    return groups > 1 ? static_cast<size_t>(groups) * 2 * static_cast<size_t>(cols) * sizeof(float) : 0;
}

template <int IO>
int entry(const void *dy, const void *x, const float *mean, const float *rstd, const void *gamma, const void *dres, void *dx,
          float *dgamma, float *dbeta, int64_t rows, int64_t cols, int unbiased, void *workspace, size_t bytes,
          ko_stream_t stream) {
    typedef typename Io<IO>::elem Elem;
    if (rows < 0 || cols <= 0)
        return fail(KO_ERR_INVALID_ARGUMENT, "layernorm_backward: rows=%lld cols=%lld", (long long)rows, (long long)cols);
    if (cols > kMaxColumns) return fail(KO_ERR_UNSUPPORTED_SHAPE, "layernorm_backward: cols=%lld too large", (long long)cols);
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
    const Args<IO> a{static_cast<const Elem *>(dy), static_cast<const Elem *>(x), mean, rstd, static_cast<const Elem *>(gamma),
                     static_cast<const Elem *>(dres), static_cast<Elem *>(dx), dgamma, dbeta, rows, static_cast<int>(cols), inv_n,
                     inv_d, partial, as_stream(stream), 0};
    return dispatch<IO>(a, cols % Io<IO>::E == 0 && (rows_at & 15) == 0);
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
