// Gradient of the row softmax for gfx950, fp32 / binary16 / bfloat16 storage, fp32 arithmetic, with the forward
// operator's padding mask.
//
// Per row, y = softmax(x):  dx_j = y_j (dy_j - t),  t = sum_k y_k dy_k.  Two reads and one write of the tensor: the
// kernels hold a row's y and dy in registers between the sum and the write, so both are read once.
//
// Mask: the forward pass replaced the columns from valid_len on by a constant, so their dx is 0.  They still count in
// t where their y is not 0 - a row whose valid scores all lie below about -9900 gives the padding weight.  All masked
// columns of a row held the same value and hold the same y, so y[valid_len] alone tells: when it is 0 (the ordinary
// case) neither y nor dy is read beyond the valid columns, whatever they hold.
//
// Bound: memory.  See the launchers for the shapes' figures.  Rows off 16-byte vectors are bound by latency: their last vector comes
// element by element, one wait after the other, and with a mask behind the loads of the lengths (32M bf16 elements: 1001 columns 55
// us, 1008 columns 34; 100 columns 73, 104 columns 33, masked 96 and 80; 13 columns 216, 16 columns 58; 5 columns 298).
#include "ko_internal.h"

#include "row_reduce.h"

namespace ko {
namespace {

__device__ __forceinline__ int clamp_len(int v, int cols) { return v < 0 ? 0 : (v > cols ? cols : v); }

// The masked columns' share of t, for the rows whose padding has weight: lanes `first`, `first + step`, ... of the
// row.  Columns whose y is 0 add nothing, whatever their dy holds.
template <int IO>
__device__ __forceinline__ float padding_share(const typename Io<IO>::elem *y, const typename Io<IO>::elem *dy, int vlen,
                                               int cols, int first, int step) {
    float t = 0.0f;
    for (int j = vlen + first; j < cols; j += step) {
        const float a = Io<IO>::scalar(y + j);
        if (a != 0.0f) t = __builtin_fmaf(a, Io<IO>::scalar(dy + j), t);
    }
    return t;
}

// ---- a row in the registers of a group of LPR lanes
template <int IO, int LPR, int VPL, bool MASKED, bool RAGGED>
__global__ __launch_bounds__(64) void softmax_backward_wave_kernel(const typename Io<IO>::elem *y_in,
                                                                   const typename Io<IO>::elem *dy_in,
                                                                   typename Io<IO>::elem *dx_out, int64_t rows, int cols,
                                                                   const int32_t *__restrict__ valid_len,
                                                                   int64_t rows_per_seq) {
    constexpr int E = Io<IO>::E;
    constexpr int RPW = 64 / LPR;
    typedef typename Io<IO>::elem Elem;
    const int lane = threadIdx.x & 63;
    const int sub = lane / LPR;
    const int l = lane % LPR;
    const int nvec = row_vectors<IO, RAGGED>(cols);
    const bool whole_lines = rows_are_whole_lines<IO>(cols);
    const uint32_t sub_off = static_cast<uint32_t>(sub) * static_cast<uint32_t>(cols) * sizeof(Elem);
    const int64_t stride = static_cast<int64_t>(gridDim.x) * RPW;
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * RPW; row0 < rows; row0 += stride) {
        const int64_t row = row0 + sub;
        const bool row_ok = row < rows;
        const Elem *y0 = y_in + row0 * cols, *dy0 = dy_in + row0 * cols;
        const Elem *y_row = y_in + row * cols, *dy_row = dy_in + row * cols;
        int vlen = cols;
        float beyond = 0.0f;  // y of the masked columns
        if constexpr (MASKED) {
            // row0 is wave-uniform: scalar loads of the lengths
#pragma unroll
            for (int r = 0; r < RPW; ++r) {
                if (row0 + r < rows) {
                    const int len = clamp_len(valid_len[(row0 + r) / rows_per_seq], cols);
                    if (sub == r) vlen = len;
                }
            }
            if (row_ok && vlen > 0 && vlen < cols) beyond = Io<IO>::scalar(y_row + vlen);
        }
        typename Io<IO>::raw yr[VPL], dr[VPL];
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int j = l + k * LPR;
            yr[k] = typename Io<IO>::raw{};
            dr[k] = typename Io<IO>::raw{};
            if (row_ok && j < nvec && (!MASKED || E * j < vlen)) {
                yr[k] = load_row_vec<IO, RAGGED, true>(y0, sub_off, j, cols);
                dr[k] = load_row_vec<IO, RAGGED, true>(dy0, sub_off, j, cols);
            }
        }
        float y[VPL][E], d[VPL][E];
        float t = 0.0f;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            Io<IO>::unpack(yr[k], y[k]);
            Io<IO>::unpack(dr[k], d[k]);
            if constexpr (MASKED) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (E * (l + k * LPR) + e >= vlen) y[k][e] = d[k][e] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) t = __builtin_fmaf(y[k][e], d[k][e], t);
        }
        if constexpr (MASKED) {
            if (beyond != 0.0f) t += padding_share<IO>(y_row, dy_row, vlen, cols, l, LPR);
        }
        t = wave::allreduce<LPR, wave::Sum>(t);
        Elem *dst0 = dx_out + row0 * cols;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int j = l + k * LPR;
            if (row_ok && j < nvec) {
                float o[E];
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    o[e] = y[k][e] * (d[k][e] - t);
                    if (MASKED && E * j + e >= vlen) o[e] = 0.0f;  // (a NaN t stays with the valid columns)
                }
                store_row_vec_any<IO, RAGGED>(whole_lines, dst0, sub_off, j, cols, o);
            }
        }
    }
}

// ---- a row in the registers of a workgroup
template <int IO, int THREADS, int VPL, bool MASKED, bool RAGGED>
__global__ __launch_bounds__(THREADS) void softmax_backward_block_kernel(const typename Io<IO>::elem *y_in,
                                                                         const typename Io<IO>::elem *dy_in,
                                                                         typename Io<IO>::elem *dx_out, int64_t rows,
                                                                         int cols, const int32_t *__restrict__ valid_len,
                                                                         int64_t rows_per_seq) {
    constexpr int E = Io<IO>::E;
    typedef typename Io<IO>::elem Elem;
    __shared__ float slots[2][THREADS / 64][1];
    const int nvec = row_vectors<IO, RAGGED>(cols);
    const bool whole_lines = rows_are_whole_lines<IO>(cols);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
        const Elem *y_row = y_in + row * cols, *dy_row = dy_in + row * cols;
        int vlen = cols;
        float beyond = 0.0f;
        if constexpr (MASKED) {
            vlen = clamp_len(valid_len[row / rows_per_seq], cols);
            if (vlen > 0 && vlen < cols) beyond = Io<IO>::scalar(y_row + vlen);
        }
        typename Io<IO>::raw yr[VPL], dr[VPL];
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int j = threadIdx.x + k * THREADS;
            yr[k] = typename Io<IO>::raw{};
            dr[k] = typename Io<IO>::raw{};
            if (j < nvec && (!MASKED || E * j < vlen)) {
                yr[k] = load_row_vec<IO, RAGGED, true>(y_row, 0, j, cols);
                dr[k] = load_row_vec<IO, RAGGED, true>(dy_row, 0, j, cols);
            }
        }
        float t[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            float y[E], d[E];
            Io<IO>::unpack(yr[k], y);
            Io<IO>::unpack(dr[k], d);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (!MASKED || E * (static_cast<int>(threadIdx.x) + k * THREADS) + e < vlen) t[0] = __builtin_fmaf(y[e], d[e], t[0]);
        }
        if constexpr (MASKED) {
            if (beyond != 0.0f) t[0] += padding_share<IO>(y_row, dy_row, vlen, cols, threadIdx.x, THREADS);
        }
        block_sum<THREADS / 64, 1>(t, slots[turn]);
        Elem *dst = dx_out + row * cols;
#pragma unroll
        for (int k = 0; k < VPL; ++k) {
            const int j = threadIdx.x + k * THREADS;
            if (j < nvec) {
                float y[E], d[E];
                convert_again<IO>(yr[k]);
                convert_again<IO>(dr[k]);
                Io<IO>::unpack(yr[k], y);
                Io<IO>::unpack(dr[k], d);
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    y[e] = y[e] * (d[e] - t[0]);
                    if (MASKED && E * j + e >= vlen) y[e] = 0.0f;
                }
                store_row_vec_any<IO, RAGGED>(whole_lines, dst, 0, j, cols, y);
            }
        }
    }
}

// ---- longer rows: t first, in one or more pieces per row, then a second read
// One workgroup sums the vectors [lo, hi) of its row.
template <int IO, int THREADS, bool MASKED, bool RAGGED>
__device__ __forceinline__ float piece_dot(const typename Io<IO>::elem *y_row, const typename Io<IO>::elem *dy_row, int lo,
                                           int hi, int vlen, int cols) {
    constexpr int E = Io<IO>::E;
    constexpr int UNROLL = 4;
    float t = 0.0f;
    for (int j0 = lo + static_cast<int>(threadIdx.x); j0 < hi; j0 += THREADS * UNROLL) {
        typename Io<IO>::raw yr[UNROLL], dr[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int j = j0 + u * THREADS;
            yr[u] = typename Io<IO>::raw{};
            dr[u] = typename Io<IO>::raw{};
            if (j < hi && (!MASKED || E * j < vlen)) {
                yr[u] = load_row_vec<IO, RAGGED, false>(y_row, 0, j, cols);
                dr[u] = load_row_vec<IO, RAGGED, false>(dy_row, 0, j, cols);
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            float y[E], d[E];
            Io<IO>::unpack(yr[u], y);
            Io<IO>::unpack(dr[u], d);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (!MASKED || E * (j0 + u * THREADS) + e < vlen) t = __builtin_fmaf(y[e], d[e], t);
        }
    }
    return t;
}

template <int IO, int THREADS, bool MASKED, bool RAGGED>
__device__ __forceinline__ void piece_apply(const typename Io<IO>::elem *y_row, const typename Io<IO>::elem *dy_row,
                                            typename Io<IO>::elem *dx_row, int lo, int hi, int vlen, int cols, float t,
                                            bool whole_lines) {
    constexpr int E = Io<IO>::E;
    constexpr int UNROLL = 4;
    for (int j0 = lo + static_cast<int>(threadIdx.x); j0 < hi; j0 += THREADS * UNROLL) {
        typename Io<IO>::raw yr[UNROLL], dr[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int j = j0 + u * THREADS;
            yr[u] = typename Io<IO>::raw{};
            dr[u] = typename Io<IO>::raw{};
            if (j < hi && (!MASKED || E * j < vlen)) {
                yr[u] = load_row_vec<IO, RAGGED, true>(y_row, 0, j, cols);
                dr[u] = load_row_vec<IO, RAGGED, true>(dy_row, 0, j, cols);
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int j = j0 + u * THREADS;
            if (j >= hi) break;
            float y[E], d[E];
            Io<IO>::unpack(yr[u], y);
            Io<IO>::unpack(dr[u], d);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                y[e] = y[e] * (d[e] - t);
                if (MASKED && E * j + e >= vlen) y[e] = 0.0f;
            }
            store_row_vec_any<IO, RAGGED>(whole_lines, dx_row, 0, j, cols, y);
        }
    }
}

// One workgroup per row, any length.
template <int IO, int THREADS, bool MASKED, bool RAGGED>
__global__ __launch_bounds__(THREADS) void softmax_backward_reread_kernel(const typename Io<IO>::elem *y_in,
                                                                          const typename Io<IO>::elem *dy_in,
                                                                          typename Io<IO>::elem *dx_out, int64_t rows,
                                                                          int cols, const int32_t *__restrict__ valid_len,
                                                                          int64_t rows_per_seq) {
    typedef typename Io<IO>::elem Elem;
    __shared__ float slots[2][THREADS / 64][1];
    const int nvec = row_vectors<IO, RAGGED>(cols);
    const bool whole_lines = rows_are_whole_lines<IO>(cols);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
        const Elem *y_row = y_in + row * cols, *dy_row = dy_in + row * cols;
        int vlen = cols;
        if constexpr (MASKED) vlen = clamp_len(valid_len[row / rows_per_seq], cols);
        float t[1] = {piece_dot<IO, THREADS, MASKED, RAGGED>(y_row, dy_row, 0, nvec, vlen, cols)};
        if constexpr (MASKED) {
            if (vlen > 0 && vlen < cols && Io<IO>::scalar(y_row + vlen) != 0.0f)
                t[0] += padding_share<IO>(y_row, dy_row, vlen, cols, threadIdx.x, THREADS);
        }
        block_sum<THREADS / 64, 1>(t, slots[turn]);
        piece_apply<IO, THREADS, MASKED, RAGGED>(y_row, dy_row, dx_out + row * cols, 0, nvec, vlen, cols, t[0], whole_lines);
    }
}

// A few long rows: workgroup (p, row) takes the row's p-th piece of `piece` vectors; the pieces' sums pass through
// the workspace and are folded in piece order.
template <int IO, int THREADS, bool MASKED, bool RAGGED>
__global__ __launch_bounds__(THREADS) void softmax_backward_pieces_dot_kernel(const typename Io<IO>::elem *y_in,
                                                                              const typename Io<IO>::elem *dy_in, int cols,
                                                                              const int32_t *__restrict__ valid_len,
                                                                              int64_t rows_per_seq, int piece,
                                                                              float *__restrict__ sums) {
    __shared__ float slots[THREADS / 64][1];
    const int nvec = row_vectors<IO, RAGGED>(cols);
    const int64_t row = blockIdx.y;
    const typename Io<IO>::elem *y_row = y_in + row * cols, *dy_row = dy_in + row * cols;
    int vlen = cols;
    if constexpr (MASKED) vlen = clamp_len(valid_len[row / rows_per_seq], cols);
    const int lo = static_cast<int>(blockIdx.x) * piece;
    const int hi = nvec - lo < piece ? nvec : lo + piece;
    float t[1] = {piece_dot<IO, THREADS, MASKED, RAGGED>(y_row, dy_row, lo, hi, vlen, cols)};
    if constexpr (MASKED) {
        if (vlen > 0 && vlen < cols && Io<IO>::scalar(y_row + vlen) != 0.0f)
            t[0] += padding_share<IO>(y_row, dy_row, vlen, cols, static_cast<int>(blockIdx.x) * THREADS + threadIdx.x,
                                      THREADS * gridDim.x);
    }
    block_sum<THREADS / 64, 1>(t, slots);
    if (threadIdx.x == 0) sums[row * gridDim.x + blockIdx.x] = t[0];
}

template <int IO, int THREADS, bool MASKED, bool RAGGED>
__global__ __launch_bounds__(THREADS) void softmax_backward_pieces_apply_kernel(
    const typename Io<IO>::elem *y_in, const typename Io<IO>::elem *dy_in, typename Io<IO>::elem *dx_out, int cols,
    const int32_t *__restrict__ valid_len, int64_t rows_per_seq, int piece, const float *__restrict__ sums) {
    const int nvec = row_vectors<IO, RAGGED>(cols);
    const int64_t row = blockIdx.y;
    int vlen = cols;
    if constexpr (MASKED) vlen = clamp_len(valid_len[row / rows_per_seq], cols);
    const int lo = static_cast<int>(blockIdx.x) * piece;
    const int hi = nvec - lo < piece ? nvec : lo + piece;
    float t = 0.0f;
    for (unsigned p = 0; p < gridDim.x; ++p) t += sums[row * gridDim.x + p];
    piece_apply<IO, THREADS, MASKED, RAGGED>(y_in + row * cols, dy_in + row * cols, dx_out + row * cols, lo, hi, vlen, cols, t,
                                     rows_are_whole_lines<IO>(cols));
}

// ---------------------------------------------------------------------------------------------------- dispatch
template <int IO>
struct Args {
    const typename Io<IO>::elem *y;
    const typename Io<IO>::elem *dy;
    typename Io<IO>::elem *dx;
    int64_t rows;
    int cols;
    const int32_t *valid_len;
    int64_t rows_per_seq;
    float *workspace;
    hipStream_t stream;
};

template <int IO, int LPR, int VPL, bool MASKED, bool RAGGED>
int launch_wave(const Args<IO> &a) {
    constexpr int RPW = 64 / LPR;
    // Residency cap as in the forward kernels (lds_pad_for_residency): a wavefront has y and dy in flight.  With a mask the
    // loads wait for the row's length first, and as many wavefronts as fit hide that (786432 x 512 binary16, three quarters
    // of it valid: 278 us, 318 with 64 KB in flight; 196608 x 2048: 267 against 307).
    const int lds = MASKED ? 0 : lds_pad_for_residency(int64_t{2} * RPW * a.cols * sizeof(typename Io<IO>::elem), 40 * 1024);
    softmax_backward_wave_kernel<IO, LPR, VPL, MASKED, RAGGED><<<row_grid((a.rows + RPW - 1) / RPW, 64), dim3(64), lds, a.stream>>>(
        a.y, a.dy, a.dx, a.rows, a.cols, a.valid_len, a.rows_per_seq);
    KO_CHECK_LAUNCH();
    return KO_OK;
}

template <int IO, int THREADS, int VPL, bool MASKED, bool RAGGED>
int launch_block(const Args<IO> &a) {
    softmax_backward_block_kernel<IO, THREADS, VPL, MASKED, RAGGED><<<row_grid(a.rows, THREADS), dim3(THREADS), 0, a.stream>>>(
        a.y, a.dy, a.dx, a.rows, a.cols, a.valid_len, a.rows_per_seq);
    KO_CHECK_LAUNCH();
    return KO_OK;
}

// Pieces per row of a few long rows: about two workgroups per compute unit in all, pieces of 16 KB and more.
// A function of the sizes alone, so that the workspace can be sized without a device.
constexpr int kPieceUnits = 256;          // compute units of an MI355X
constexpr int64_t kPieceBytes = 16 << 10;
int pieces_per_row(int64_t rows, int64_t row_bytes) {
    if (rows <= 0 || rows * 4 > kPieceUnits || row_bytes < 8 * kPieceBytes) return 1;
    int64_t parts = 2 * kPieceUnits / rows;
    if (parts > row_bytes / kPieceBytes) parts = row_bytes / kPieceBytes;
    return static_cast<int>(parts);
}

template <int IO, bool MASKED, bool RAGGED>
int launch_long(const Args<IO> &a) {
    constexpr int THREADS = 1024;
    softmax_backward_reread_kernel<IO, THREADS, MASKED, RAGGED><<<row_grid(a.rows, THREADS), dim3(THREADS), 0, a.stream>>>(
        a.y, a.dy, a.dx, a.rows, a.cols, a.valid_len, a.rows_per_seq);
    KO_CHECK_LAUNCH();
    return KO_OK;
}

template <int IO, bool MASKED, bool RAGGED>
int launch_pieces(const Args<IO> &a, int parts) {
    constexpr int THREADS = 256;
    const int nvec = (a.cols + Io<IO>::E - 1) / Io<IO>::E;
    const int piece = (nvec + parts - 1) / parts;
    parts = (nvec + piece - 1) / piece;
    const dim3 grid(static_cast<unsigned>(parts), static_cast<unsigned>(a.rows));
    softmax_backward_pieces_dot_kernel<IO, THREADS, MASKED, RAGGED><<<grid, dim3(THREADS), 0, a.stream>>>(
        a.y, a.dy, a.cols, a.valid_len, a.rows_per_seq, piece, a.workspace);
    KO_CHECK_LAUNCH();
    softmax_backward_pieces_apply_kernel<IO, THREADS, MASKED, RAGGED><<<grid, dim3(THREADS), 0, a.stream>>>(
        a.y, a.dy, a.dx, a.cols, a.valid_len, a.rows_per_seq, piece, a.workspace);
    KO_CHECK_LAUNCH();
    return KO_OK;
}

template <int IO, bool MASKED, bool RAGGED>
int dispatch(const Args<IO> &a) {
    const int nvec = (a.cols + Io<IO>::E - 1) / Io<IO>::E;
    if (a.workspace != nullptr) {
        const int parts = pieces_per_row(a.rows, static_cast<int64_t>(a.cols) * sizeof(typename Io<IO>::elem));
        if (parts > 1) return launch_pieces<IO, MASKED, RAGGED>(a, parts);
    }
    int lpr = 0, vpl = 0;
    if (choose_row_group(nvec, 4, &lpr, &vpl)) {
#define KO_WAVE(L, V) if (lpr == L && vpl == V) return launch_wave<IO, L, V, MASKED, RAGGED>(a)
        // With a mask, two rows per group of lanes that would hold one vector each: twice the loads per wait for a length
        // (786432 x 512 binary16 278 us against 299).
        if (MASKED && vpl == 1 && lpr > 8) lpr /= 2, vpl = 2;
        KO_WAVE(8, 1);
        if constexpr (!MASKED) {
            KO_WAVE(16, 1); KO_WAVE(32, 1); KO_WAVE(64, 1);
        }
        KO_WAVE(8, 2); KO_WAVE(8, 3); KO_WAVE(16, 2); KO_WAVE(16, 3); KO_WAVE(32, 2); KO_WAVE(32, 3);
        KO_WAVE(64, 2); KO_WAVE(64, 3); KO_WAVE(64, 4);
#undef KO_WAVE
    }
    if (nvec <= 512) return launch_block<IO, 256, 2, MASKED, RAGGED>(a);
    if (nvec <= 1024) return launch_block<IO, 512, 2, MASKED, RAGGED>(a);
    if (nvec <= 2048) return launch_block<IO, 1024, 2, MASKED, RAGGED>(a);
    if (nvec <= 4096) return launch_block<IO, 1024, 4, MASKED, RAGGED>(a);
    if (nvec <= 8192) return launch_block<IO, 1024, 8, MASKED, RAGGED>(a);
    return launch_long<IO, MASKED, RAGGED>(a);
}

size_t workspace_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0 || cols > kMaxColumns) return 0;
    const int parts = pieces_per_row(rows, cols * 4);  // (16-bit rows are cut into no more pieces)
    return parts > 1 ? static_cast<size_t>(rows) * parts * sizeof(float) : 0;
}

template <int IO>
int entry(const void *y, const void *dy, void *dx, int64_t rows, int64_t cols, const int32_t *valid_len,
          int64_t rows_per_seq, void *workspace, size_t bytes, ko_stream_t stream) {
    typedef typename Io<IO>::elem Elem;
    if (rows < 0 || cols <= 0)
        return fail(KO_ERR_INVALID_ARGUMENT, "softmax_backward: rows=%lld cols=%lld", (long long)rows, (long long)cols);
    if (cols > kMaxColumns) return fail(KO_ERR_UNSUPPORTED_SHAPE, "softmax_backward: cols=%lld too large", (long long)cols);
    if (rows == 0) return KO_OK;
    if (!y || !dy || !dx) return fail(KO_ERR_INVALID_ARGUMENT, "softmax_backward: null y/dy/dx pointer");
    const uintptr_t addresses = reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(dy) | reinterpret_cast<uintptr_t>(dx);
    if (addresses & (sizeof(Elem) - 1))
        return fail(KO_ERR_INVALID_ARGUMENT, "softmax_backward: y/dy/dx must be aligned to their element type");
    if (valid_len && rows_per_seq <= 0)
        return fail(KO_ERR_INVALID_ARGUMENT, "softmax_backward: valid_len given but rows_per_seq=%lld", (long long)rows_per_seq);
    if (workspace && bytes < workspace_bytes(rows, cols))
        return fail(KO_ERR_INVALID_ARGUMENT, "softmax_backward: workspace of %zu bytes, %zu needed", bytes, workspace_bytes(rows, cols));
    if (reinterpret_cast<uintptr_t>(workspace) & 15)
        return fail(KO_ERR_INVALID_ARGUMENT, "softmax_backward: workspace must be 16-byte aligned");
    const Args<IO> a{static_cast<const Elem *>(y), static_cast<const Elem *>(dy), static_cast<Elem *>(dx), rows,
                     static_cast<int>(cols), valid_len, rows_per_seq, static_cast<float *>(workspace), as_stream(stream)};
    if (cols % Io<IO>::E != 0 || (addresses & 15) != 0)
        return valid_len ? dispatch<IO, true, true>(a) : dispatch<IO, false, true>(a);
    return valid_len ? dispatch<IO, true, false>(a) : dispatch<IO, false, false>(a);
}

}  // namespace
}  // namespace ko

KO_EXPORT size_t ko_softmax_backward_workspace_bytes(int64_t rows, int64_t cols) { return ko::workspace_bytes(rows, cols); }

KO_EXPORT int ko_softmax_backward_f32(const float *y, const float *dy, float *dx, int64_t rows, int64_t cols,
                                      const int32_t *valid_len, int64_t rows_per_seq, void *workspace,
                                      size_t workspace_bytes, ko_stream_t stream) {
    return ko::entry<ko::IO_F32>(y, dy, dx, rows, cols, valid_len, rows_per_seq, workspace, workspace_bytes, stream);
}

KO_EXPORT int ko_softmax_backward_16(const void *y, const void *dy, void *dx, int64_t rows, int64_t cols,
                                     const int32_t *valid_len, int64_t rows_per_seq, int dtype, void *workspace,
                                     size_t workspace_bytes, ko_stream_t stream) {
    if (dtype == KO_F16)
        return ko::entry<ko::IO_F16>(y, dy, dx, rows, cols, valid_len, rows_per_seq, workspace, workspace_bytes, stream);
    if (dtype == KO_BF16)
        return ko::entry<ko::IO_BF16>(y, dy, dx, rows, cols, valid_len, rows_per_seq, workspace, workspace_bytes, stream);
    return ko::fail(KO_ERR_INVALID_ARGUMENT, "softmax_backward: dtype=%d is neither KO_F16 nor KO_BF16", dtype);
}
