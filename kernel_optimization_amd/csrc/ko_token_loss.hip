// Losses over rows of logits for gfx950: log-probabilities of labels and their gradient, the clipped policy loss with
// a KL term from the logits to their gradient, and the preference loss on paired sequences.  fp32 / binary16 / bfloat16
// logits, fp32 arithmetic; differences of log-probabilities are taken in 64 bits.
//
// Per row with label l and z = scale x:  m = max x, S = sum_{j != l} exp(scale (x_j - m)), e = exp(scale (x_l - m)),
//   logp = log(e / (S + e)) = -log1p(S / e).
// The label's own column stays out of S: for a likely label (logp near 0) the others' sum is what matters, and in
// 1 + S it would be rounded away.  Gradient of c * logp:  dx_j = -c scale exp(scale (x_j - m)) / (S + e) for j != l, and
// c scale S / (S + e) for the label.
//
// Rows.  A row of logits starts anywhere (ld elements after the last one): its columns are a head up to the first 128-byte
// boundary, whole 16-byte vectors, and a tail.  Head and tail elements are taken one by one by the first threads; the
// vectors carry the row, and what they write are whole lines of the caches, which no two workgroups share (1 GiB of rows of
// 50272 bf16 columns, their odd ones 64 bytes into a line: gradient 383 us with vectors from 64-byte boundaries on).  So a
// vocabulary of 50257 contiguous columns runs on vectors, too.
//
// Bound: memory.  The sums are one pass, relative to the label's logit and, where that is far below the others or far from 0, a second
// one with a running maximum; in pieces of rows and in the policy loss without a gradient, one with a running maximum.  The policy
// loss keeps the whole row in a workgroup's registers between the sum and the gradient, so that the logits are read once and the
// gradient written once.  Gradients of rows that lie differently in the two matrices go element by element, in the policy loss after
// a second read (1 GiB of 50257 bf16 columns into rows of 50264: 962 us instead of 349, policy loss 2310 instead of 365).
#include "ko_internal.h"

#include "row_reduce.h"

#include <cfloat>
#include <cmath>
#include <initializer_list>

namespace ko {
namespace {

constexpr float kLog2e = 0x1.715476p+0f;

// A value that is the same in every lane, in scalar registers: what follows from a row's label stays there, too.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ float uniform(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
}

__device__ __forceinline__ int64_t uniform(int64_t v) {
    const uint64_t b = static_cast<uint64_t>(v);
    const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(b >> 32)));
    return static_cast<int64_t>((hi << 32) | static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(b))));
}

// ---- a row's columns
template <int IO>
struct RowSpan {
    int head;     // single elements before the first vector, up to a 128-byte boundary
    int nvec;     // vectors, from column `head` on
    int singles;  // single elements in all: the head, and what is left after the last vector
};
template <int IO>
__device__ __forceinline__ RowSpan<IO> span_of(const typename Io<IO>::elem *row, int cols) {
    constexpr int E = Io<IO>::E;
    RowSpan<IO> s;
    if constexpr (E == 1) {
        s.head = 0;
        s.nvec = cols;
        s.singles = 0;
    } else {
        constexpr int LINE = 128 / static_cast<int>(sizeof(typename Io<IO>::elem));
        const int past = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 127) / sizeof(typename Io<IO>::elem));
        s.head = (LINE - past) % LINE;
        if (s.head > cols) s.head = cols;
        s.nvec = (cols - s.head) / E;
        s.singles = cols - s.nvec * E;
    }
    return s;
}
// column of the i-th single element
template <int IO>
__device__ __forceinline__ int single_column(const RowSpan<IO> &s, int i) {
    return i < s.head ? i : s.nvec * Io<IO>::E + i;
}

// Where the part-th of `parts` pieces of n vectors begins: pieces are whole 128-byte lines, and the last ones may be empty.
__device__ __forceinline__ int piece_begin(int n, int parts, int part) {
    const int64_t at = static_cast<int64_t>(((n + parts - 1) / parts + 7) & ~7) * part;
    return at < n ? static_cast<int>(at) : n;
}

// ---- running (maximum, sum of exp(scale (x - maximum)))
struct Pair {
    float m, s;
};
// scale log2(e): as one float (all), off by up to 2^-24 of itself, the same way in every exponential of a row, which 100000 of them
// do not average out (1e-6 in a logp of -13); and in two parts.  hi has 16 bits: the second part's products are then large enough
// to count where they are added to rounded ones (next to a hi of 24 bits they are rounded away: logits around 20 gave a logp off by
// 4e-7, in every row alike).  lo is positive.
struct Scale {
    float hi, lo, all;
};
// exp(scale d).  exp_sum: for sums; exp_scaled: where the result is rounded next.
__device__ __forceinline__ float exp_sum(float d, Scale c) { return __builtin_amdgcn_exp2f(__builtin_fmaf(d, c.hi, d * c.lo)); }
__device__ __forceinline__ float exp_scaled(float d, Scale c) { return __builtin_amdgcn_exp2f(d * c.all); }
// c times a label's logit, for sums relative to it: to a multiple of 2^-8.  With bfloat16's few numbers hi x - shift is then mostly exact;
// if it were rounded, that would go by the last bits of shift, the same way in all of a row's columns.
__device__ __forceinline__ float shift_of(float at_label, Scale c) { return __builtin_rintf(at_label * c.all * 256.0f) * 0.00390625f; }
// 2^(c x - shift)
__device__ __forceinline__ float power_of(float x, float shift, Scale c) {
    return __builtin_amdgcn_exp2f(__builtin_fmaf(x, c.lo, __builtin_fmaf(x, c.hi, -shift)));
}
// An empty pair is (-FLT_MAX, 0).

// Adds N values (absent ones: -inf) at once: the sum is rescaled at most once for all of them, and only where a lane of
// the wavefront has met a larger value.
template <int N>
__device__ __forceinline__ void add_values(Pair &p, const float (&v)[N], Scale c) {
    float m = v[0];
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
    if (__any(m > p.m)) {
        const float top = fmaxf(m, p.m);
        p.s *= exp_sum(p.m - top, c);
        p.m = top;
    }
    float s[N < 4 ? N : 4];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const float e = exp_sum(v[i] - p.m, c);
        if (i < 4) s[i] = e;
        else s[i % 4] += e;
    }
    if constexpr (N >= 4) p.s += (s[0] + s[1]) + (s[2] + s[3]);
    else p.s += s[0];
}

// A row's or a piece's pair: its sum in 64 bits.  What a thread sums in 32 bits is off by its own roundings, which average out
// over a thousand threads; the last steps of a tree would not, and a KL term takes the difference of two such numbers.
struct Total {
    float m;
    double s;
};
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int step = 1; step < 64; step <<= 1) v += __shfl_xor(v, step, 64);
    return v;
}
// Sum over a wavefront, the same bits in every lane: sixteen lanes in 32 bits, the four sums of those in 64.
__device__ __forceinline__ double wave_total(float v) {
    const int row = __builtin_bit_cast(int, wave::allreduce<16, wave::Sum>(v));
    auto of = [&](int lane) { return static_cast<double>(__builtin_bit_cast(float, __builtin_amdgcn_readlane(row, lane))); };
    return (of(0) + of(16)) + (of(32) + of(48));
}

// The pairs of a workgroup's threads, the same bits in every thread.  One barrier; `slot` as in block_sum.
template <int WAVES>
__device__ __forceinline__ Total block_pair(Pair p, Total *slot, Scale c) {
    const float m = wave::allreduce<64, wave::Max>(p.m);
    Total r{m, wave_total(p.s * exp_sum(p.m - m, c))};
    if constexpr (WAVES > 1) {
        if ((threadIdx.x & 63) == 0) slot[threadIdx.x >> 6] = r;
        __syncthreads();
        float top = slot[0].m;
#pragma unroll
        for (int w = 1; w < WAVES; ++w) top = fmaxf(top, slot[w].m);
        double s = 0.0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) s += slot[w].s * exp_sum(slot[w].m - top, c);
        r = Total{top, s};
    }
    return r;
}

// From a sum of 2^(c x_j - shift) to one of exp(scale (x_j - x_l)): shift is c x_l rounded, and what the rounding took is a factor
// 2^-rest next to 1.  c x - shift is put together in two steps, the first of which is rounded at some 2^-15 of shift: within 2^-24 up to
// a shift of 2^16.  Beyond that NaN, which callers take as they take a sum that is too large: they sum again, relative to the maximum.
// (Far beyond, the powers here leave their range long before the row's own do.)
__device__ __forceinline__ double to_label(double sum, float at_label, float shift, Scale c) {
    if (!(fabsf(shift) <= 0x1p16f)) return __builtin_nan("");
    const float rest = __builtin_fmaf(at_label, c.lo, __builtin_fmaf(at_label, c.hi, -shift));
    return sum + sum * expm1f(-0.69314718f * rest);
}

// A thread's share of the pair over the vectors [lo, hi) and, if `with_singles`, the single elements of a row, without
// the label's column.
template <int IO, int THREADS>
__device__ __forceinline__ Pair thread_pair(const typename Io<IO>::elem *row, const RowSpan<IO> &span, int lo, int hi,
                                            bool with_singles, int label, Scale c) {
    constexpr int E = Io<IO>::E;
    constexpr int UNROLL = E == 8 ? 4 : 8;
    Pair p{-FLT_MAX, 0.0f};
    const typename Io<IO>::elem *vecs = row + span.head;
    const int in_vecs = label - span.head;                // the label's place among the vectors' elements
    const int label_vec = in_vecs >= 0 ? in_vecs / E : -1;
    for (int j0 = lo + static_cast<int>(threadIdx.x); j0 < hi; j0 += THREADS * UNROLL) {
        typename Io<IO>::raw r[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int j = j0 + u * THREADS;
            r[u] = typename Io<IO>::raw{};
            if (j < hi) r[u] = Io<IO>::template load_raw<true>(vecs + static_cast<int64_t>(E) * j);
        }
        float v[UNROLL * E];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int j = j0 + u * THREADS;
            float x[E];
            Io<IO>::unpack(r[u], x);
            if (j >= hi || j == label_vec) {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (j >= hi || E * j + e == in_vecs) x[e] = -INFINITY;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) v[u * E + e] = x[e];
        }
        add_values(p, v, c);
    }
    if (with_singles) {
        for (int i = threadIdx.x; i < span.singles; i += THREADS) {
            const int column = single_column(span, i);
            const float v[1] = {column == label ? -INFINITY : Io<IO>::scalar(row + column)};
            add_values(p, v, c);
        }
    }
    return p;
}

// ---- a row's scalars
// Logarithms here are of the size of 10 and get subtracted from each other, and a KL term takes such a difference squared: in
// fp32 they would carry an error of 5e-7, ten times that of the sums.  So they are 64-bit numbers, by a short series; the rest
// are fp32 functions (64-bit ones from the library would take as long as 1.5 us per row and, their constants kept in registers,
// a hundred registers of kernels that need them for the row).
struct RowScore {
    double logp;     // log probability of the label
    double logsum;   // log sum_j exp(scale (x_j - top)), the label included
    float top;       // maximum of the row
    float inv_total; // 1 / (S + e)
    float rest;      // S / (S + e): what the label's probability leaves
};
// log(t) of a positive t, within 1e-12 absolute: t = 2^k f, f within sqrt(2) of 1, log f = 2 atanh(u), u = (f - 1) / (f + 1),
// |u| < 0.172, by its series up to u^13.
__device__ __forceinline__ double log_in_parts(double t) {
    if (!(t < 1e30)) return t;
    int k;
    (void)frexpf(static_cast<float>(t), &k);
    double f = ldexp(t, -k);
    if (f < 0.70710678) {
        f *= 2.0;
        --k;
    }
    // the reciprocal in 32 bits and one Newton step
    double r = 1.0f / static_cast<float>(f + 1.0);
    r = __builtin_fma(r, __builtin_fma(-(f + 1.0), r, 1.0), r);
    const double u = (f - 1.0) * r, w = u * u;
    double p = __builtin_fma(w, 1.0 / 13.0, 1.0 / 11.0);
    p = __builtin_fma(w, p, 1.0 / 9.0);
    p = __builtin_fma(w, p, 1.0 / 7.0);
    p = __builtin_fma(w, p, 1.0 / 5.0);
    p = __builtin_fma(w, p, 1.0 / 3.0);
    p = __builtin_fma(w, p, 1.0);
    return __builtin_fma(static_cast<double>(k), 0.69314718055994531, 2.0 * u * p);
}
// exp(scale (x - top)), x <= top: what a row's whole sum is multiplied by.  The argument in base 2 has more than 32 bits, of which the
// hardware takes 32; the others are worked in to first order.  (Rounded to 32 bits at -30 it put 4e-7 on all of a sum.)
__device__ __forceinline__ double exp_below(float x, float top, Scale c) {
    const double a = (static_cast<double>(x) - static_cast<double>(top)) * (static_cast<double>(c.hi) + static_cast<double>(c.lo));
    if (a < -150.0) return 0.0;
    const float rounded = static_cast<float>(a);
    const double e = __builtin_amdgcn_exp2f(rounded);
    return __builtin_fma(e, 0.69314718 * (a - rounded), e);
}
// From the pair of the other columns and the label's logit.
__device__ __forceinline__ RowScore score_row(Total p, float at_label, float scale, Scale c) {
    RowScore r;
    r.top = fmaxf(p.m, at_label);
    const double s = p.s * exp_below(p.m, r.top, c);
    const double z = (static_cast<double>(at_label) - static_cast<double>(r.top)) * static_cast<double>(scale);
    const double e = exp_below(at_label, r.top, c);
    const double total = s + e;
    if (s <= e) {  // a likely label: relative to a logarithm close to 0
        // (e is 1 here: no other column reaches the label's; or 0, in a row of nothing but -inf: NaN)
        r.logp = !(e > 0.0) ? __builtin_nan("") : s < 0.03125 ? -log1pf(static_cast<float>(s)) : -log_in_parts(1.0 + s);
        r.logsum = z - r.logp;
    } else {
        r.logsum = log_in_parts(total);
        r.logp = z - r.logsum;
    }
    r.inv_total = 1.0f / static_cast<float>(total);
    r.rest = static_cast<float>(s) * r.inv_total;
    return r;
}
__device__ __forceinline__ RowScore nan_score() {
    const float nan = __builtin_nanf("");
    return RowScore{nan, nan, nan, nan, nan};
}

// The values of one vector, the first of them element `first` of the row's vectors, become their gradient.
template <int E, class LabelGrad>
__device__ __forceinline__ void gradient_of(float (&x)[E], int first, bool live, int in_vecs, bool holds_label, float top,
                                            float a, LabelGrad label_grad, Scale c) {
    float at_label = 0.0f;
    if (holds_label) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (first + e == in_vecs) at_label = x[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) x[e] = live ? a * exp_scaled(x[e] - top, c) : 0.0f;
    if (live && holds_label) {
        const float g = label_grad(at_label);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (first + e == in_vecs) x[e] = g;
    }
}

// Gradient of one row's vectors [lo, hi) and, if `with_singles`, its single elements: a exp(scale (x - top)) beside the
// label, label_grad(x) at the label.  `live` false: zeros, nothing read.  Every thread reads what it overwrites and nothing
// else, so `out` may be `row`.
template <int IO, int THREADS, class LabelGrad>
__device__ __forceinline__ void write_gradient(const typename Io<IO>::elem *row, typename Io<IO>::elem *out,
                                               const RowSpan<IO> &span, int lo, int hi, bool with_singles, bool live,
                                               int label, float top, float a, LabelGrad label_grad, Scale c) {
    constexpr int E = Io<IO>::E;
    constexpr int UNROLL = E == 8 ? 2 : 4;
    typedef typename Io<IO>::elem Elem;
    const Elem *vecs = row + span.head;
    Elem *out_vecs = out + span.head;
    const int in_vecs = label - span.head;
    const int label_vec = in_vecs >= 0 ? in_vecs / E : -1;
    for (int j0 = lo + static_cast<int>(threadIdx.x); j0 < hi; j0 += THREADS * UNROLL) {
        typename Io<IO>::raw r[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int j = j0 + u * THREADS;
            r[u] = typename Io<IO>::raw{};
            if (live && j < hi) r[u] = Io<IO>::template load_raw<true>(vecs + static_cast<int64_t>(E) * j);
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int j = j0 + u * THREADS;
            if (j >= hi) break;
            float x[E];
            Io<IO>::unpack(r[u], x);
            gradient_of(x, E * j, live, in_vecs, j == label_vec, top, a, label_grad, c);
            store_row_vec<IO>(E > 1, out_vecs, Io<IO>::kBytes * static_cast<uint32_t>(j), x);
        }
    }
    if constexpr (E > 1) {
        for (int i = threadIdx.x; with_singles && i < span.singles; i += THREADS) {
            constexpr int ONE = io_by_element(IO);
            const int column = single_column(span, i);
            float x[1] = {0.0f};
            if (live) {
                x[0] = Io<IO>::scalar(row + column);
                x[0] = column == label ? label_grad(x[0]) : a * exp_scaled(x[0] - top, c);
            }
            Io<ONE>::template store<true>(out + column, x);
        }
    }
}

// ------------------------------------------------------------------------------------- token log-probabilities
template <int IO>
struct ScoreArgs {
    typedef typename Io<IO>::elem Elem;
    const Elem *logits;
    int64_t ld;
    const int32_t *labels;
    float scale;
    Scale c;
    float *logp;
    float *row_stats;  // [rows][2]: maximum, log sum
    int64_t rows;
    int cols;
    hipStream_t stream;
};

template <class A>
__device__ __forceinline__ void put_score(const A &a, int64_t row, bool live, const RowScore &r) {
    a.logp[row] = live ? static_cast<float>(r.logp) : 0.0f;
    if (a.row_stats) {
        a.row_stats[2 * row] = live ? r.top : 0.0f;
        a.row_stats[2 * row + 1] = live ? static_cast<float>(r.logsum) : 0.0f;
    }
}

// One vector's share of a row's sum and maximum.  `ragged`: it may hold the label or lie past the row's end.
template <int IO>
__device__ __forceinline__ void add_vector(const typename Io<IO>::raw &r, int j, bool ragged, int nvec, int in_vecs, float shift,
                                           Scale c, float (&s)[4], float &top) {
    constexpr int E = Io<IO>::E;
    float x[E];
    Io<IO>::unpack(r, x);
    if (ragged) {
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = j >= nvec || E * j + e == in_vecs ? -INFINITY : x[e];
    }
#pragma unroll
    for (int e = 0; e < E; ++e) {
        top = fmaxf(top, x[e]);
        s[e % 4] += power_of(x[e], shift, c);
    }
}
// A thread's single elements.
template <int IO, int THREADS>
__device__ __forceinline__ void add_singles(const typename Io<IO>::elem *src, const RowSpan<IO> &span, int label, float shift, Scale c,
                                            float (&s)[4], float &top) {
    for (int i = threadIdx.x; i < span.singles; i += THREADS) {
        const int column = single_column(span, i);
        const float x = column == label ? -INFINITY : Io<IO>::scalar(src + column);
        top = fmaxf(top, x);
        s[1] += power_of(x, shift, c);
    }
}
// The score of a row from its label's logit, the sum relative to that and the row's maximum.
template <class A>
__device__ __forceinline__ RowScore label_score(const A &a, Total p, float at_label, float top) {
    RowScore score = score_row(p, at_label, a.scale, a.c);
    // the sum is relative to the label: its logarithm relative to the maximum
    score.logsum += (static_cast<double>(score.top) - static_cast<double>(top)) * static_cast<double>(a.scale);
    score.top = top;
    return score;
}

// One workgroup per row, the next batch of U vectors per thread in flight while this one is added up.  As in
// policy_onchip_kernel the exponentials are taken against the label's logit, and the row's maximum is noted by the way; a label
// so unlikely that the sum reaches 2^40, or a sum that is not a number, is summed again with a running maximum.  Bound: memory
// (1 GiB of bf16 logits: 128256 columns 161 us, 6.7 TB/s, 50257 columns 154 us, 7.0 TB/s, 8192 columns 197 us, 4096 columns 200; the
// arithmetic close behind: nine instructions' time per value; six wavefronts per SIMD, which the compiler has to be told: with five
// 8192 columns took 216 us when six took 195).  A running maximum without loads ahead took 329 us at 8192 columns.
template <int IO, int THREADS, int U>
__global__ __launch_bounds__(THREADS) __attribute__((amdgpu_waves_per_eu(6))) void token_logprob_row_kernel(ScoreArgs<IO> a) {
    constexpr int E = Io<IO>::E;
    constexpr int WAVES = THREADS / 64;
    typedef typename Io<IO>::raw Raw;
    __shared__ Total slots[2][WAVES];
    __shared__ Total again[WAVES];
    int turn = 0;  // (alternates between the rows that use the slots: rows without a label pass no barrier)
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const typename Io<IO>::elem *src = a.logits + row * a.ld;
        const RowSpan<IO> span = span_of<IO>(src, a.cols);
        const int label = uniform(a.labels[row]);
        if (label < 0 || label >= a.cols) {
            if (threadIdx.x == 0) put_score(a, row, label >= 0, nan_score());
            continue;
        }
        // vectors past the row's end read as zeros, without traffic
        const Buffer from = buffer_of(src + span.head, Io<IO>::kBytes * span.nvec);
        const float at_label = Io<IO>::scalar(src + label);
        const float shift = shift_of(at_label, a.c);
        const int in_vecs = label - span.head;
        const int label_vec = in_vecs >= 0 && in_vecs < span.nvec * E ? in_vecs / E : -1;
        float top = at_label;
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        auto load = [&](Raw (&r)[U], int first) {
#pragma unroll
            for (int u = 0; u < U; ++u) r[u] = buffer_load<IO>(from, Io<IO>::kBytes * static_cast<uint32_t>(first + u * THREADS));
        };
        auto add = [&](Raw (&r)[U], int first) {
            const int begin = uniform(first - static_cast<int>(threadIdx.x));
            // in this batch, the same in every lane: the label, or the row's end
            const bool ragged = begin + U * THREADS > span.nvec || (label_vec >= begin && label_vec < begin + U * THREADS);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (ragged && begin + u * THREADS >= span.nvec) break;
                add_vector<IO>(r[u], first + u * THREADS, ragged, span.nvec, in_vecs, shift, a.c, s, top);
            }
        };
        Raw r[2][U];
        int j = static_cast<int>(threadIdx.x);
        load(r[0], j);
        while (true) {
            load(r[1], j + U * THREADS);
            add(r[0], j);
            j += U * THREADS;
            if (j - static_cast<int>(threadIdx.x) >= span.nvec) break;
            load(r[0], j + U * THREADS);
            add(r[1], j);
            j += U * THREADS;
            if (j - static_cast<int>(threadIdx.x) >= span.nvec) break;
        }
        add_singles<IO, THREADS>(src, span, label, shift, a.c, s, top);
        top = wave::allreduce<64, wave::Max>(top);
        double sum = wave_total((s[0] + s[1]) + (s[2] + s[3]));
        if constexpr (WAVES > 1) {
            if ((threadIdx.x & 63) == 0) slots[turn][threadIdx.x >> 6] = Total{top, sum};
            __syncthreads();
            top = slots[turn][0].m;
            sum = slots[turn][0].s;
#pragma unroll
            for (int w = 1; w < WAVES; ++w) {
                top = fmaxf(top, slots[turn][w].m);
                sum += slots[turn][w].s;
            }
            turn ^= 1;
        }
        Total p{at_label, to_label(sum, at_label, shift, a.c)};
        if (!(uniform(static_cast<float>(p.s)) < 0x1p40f)) {
            p = block_pair<WAVES>(thread_pair<IO, THREADS>(src, span, 0, span.nvec, true, label, a.c), again, a.c);
            top = fmaxf(p.m, at_label);
            __syncthreads();  // (read before the next row writes them)
        }
        if (threadIdx.x == 0) put_score(a, row, true, label_score(a, p, at_label, top));
    }
}

// Many short rows, of U 64 vectors at most: a wavefront takes kShortRows of them, and the arithmetic of a row's score - several times
// that of its sum, in one lane - is done for all of them at once, a row per lane (1 GiB of bf16 rows: 512 columns 234 us, 1024
// columns 192; when tried, eight rows 227 and 197, a row per wavefront 471 and 281, four rows 252 and 206, sixteen 238 and, for
// want of registers, 257).
constexpr int kShortRows = 8;
// Fewer rows are better off with a wavefront each: eight rows in turn take 2 to 4 us longer than one (64 rows of 512 bf16
// columns: log-probabilities 5.7 us against 3.9, policy loss 8.2 against 4.3), which pays from here on, for the policy loss from
// twice as many.
constexpr int64_t kManyRows = 16384;
template <int IO, int U>
__global__ __launch_bounds__(64) void token_logprob_short_kernel(ScoreArgs<IO> a) {
    typedef typename Io<IO>::elem Elem;
    const int lane = threadIdx.x;
    auto of = [&](float v, int i) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i)); };
    for (int64_t row0 = static_cast<int64_t>(blockIdx.x) * kShortRows; row0 < a.rows; row0 += static_cast<int64_t>(gridDim.x) * kShortRows) {
        const int n = a.rows - row0 < kShortRows ? static_cast<int>(a.rows - row0) : kShortRows;
        const int my_label = lane < n ? a.labels[row0 + lane] : -1;
        const bool reads = my_label >= 0 && my_label < a.cols;
        const float my_at = reads ? Io<IO>::scalar(a.logits + (row0 + lane) * a.ld + my_label) : 0.0f;
        Total mine{my_at, 0.0};
        float my_top = my_at;
        typename Io<IO>::raw r[kShortRows][U];
        // rows without a label are not read: their buffers are empty
#pragma unroll
        for (int i = 0; i < kShortRows; ++i) {
            const Elem *src = a.logits + (row0 + i) * a.ld;
            const RowSpan<IO> span = span_of<IO>(src, a.cols);
            const int label = __builtin_amdgcn_readlane(my_label, i);
            const Buffer from = buffer_of(src + span.head, label >= 0 && label < a.cols ? Io<IO>::kBytes * span.nvec : 0);
#pragma unroll
            for (int u = 0; u < U; ++u) r[i][u] = buffer_load<IO>(from, Io<IO>::kBytes * static_cast<uint32_t>(lane + u * 64));
        }
#pragma unroll
        for (int i = 0; i < kShortRows; ++i) {
            const int label = __builtin_amdgcn_readlane(my_label, i);
            if (label < 0 || label >= a.cols) continue;
            const Elem *src = a.logits + (row0 + i) * a.ld;
            const RowSpan<IO> span = span_of<IO>(src, a.cols);
            const int in_vecs = label - span.head;
            const float at_label = of(my_at, i);
            const float shift = shift_of(at_label, a.c);
            float top = at_label;
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u * 64 >= span.nvec) break;
                add_vector<IO>(r[i][u], lane + u * 64, true, span.nvec, in_vecs, shift, a.c, s, top);
            }
            add_singles<IO, 64>(src, span, label, shift, a.c, s, top);
            top = wave::allreduce<64, wave::Max>(top);
            const double sum = wave_total((s[0] + s[1]) + (s[2] + s[3]));
            if (lane == i) {
                mine.s = sum;
                my_top = top;
            }
        }
        mine.s = to_label(mine.s, my_at, shift_of(my_at, a.c), a.c);
        // unlikely labels, special values: against the maximum, a row at a time
        uint64_t again = __ballot(reads && !(static_cast<float>(mine.s) < 0x1p40f));
        while (again) {
            const int i = __builtin_ctzll(again);
            again &= again - 1;
            const Elem *src = a.logits + (row0 + i) * a.ld;
            const RowSpan<IO> span = span_of<IO>(src, a.cols);
            const Total p = block_pair<1>(thread_pair<IO, 64>(src, span, 0, span.nvec, true, __builtin_amdgcn_readlane(my_label, i), a.c),
                                          nullptr, a.c);
            if (lane == i) {
                mine = p;
                my_top = fmaxf(p.m, my_at);
            }
        }
        if (lane < n) put_score(a, row0 + lane, my_label >= 0, reads ? label_score(a, mine, my_at, my_top) : nan_score());
    }
}

// A few rows: workgroup (p, row) takes the row's p-th piece; pieces' pairs and the label's logit pass through the
// workspace.
// layout: Total [rows][1 + parts]; the first of a row holds the label's logit
template <int IO, int THREADS>
__global__ __launch_bounds__(THREADS) void token_pieces_kernel(const typename Io<IO>::elem *logits, int64_t ld,
                                                               const int32_t *__restrict__ labels,
                                                               const float *__restrict__ weight, int cols, Scale c,
                                                               Total *__restrict__ pairs) {
    __shared__ Total slot[THREADS / 64];
    const int64_t row = blockIdx.y;
    const int label = uniform(labels[row]);
    if (label < 0 || label >= cols || (weight && uniform(weight[row]) == 0.0f)) return;
    const typename Io<IO>::elem *src = logits + row * ld;
    const RowSpan<IO> span = span_of<IO>(src, cols);
    const int parts = static_cast<int>(gridDim.x), part = static_cast<int>(blockIdx.x);
    const int lo = piece_begin(span.nvec, parts, part), hi = piece_begin(span.nvec, parts, part + 1);
    const Total p = block_pair<THREADS / 64>(thread_pair<IO, THREADS>(src, span, lo, hi, part == 0, label, c), slot, c);
    if (threadIdx.x == 0) {
        Total *mine = pairs + row * (1 + parts);
        if (part == 0) mine[0] = Total{Io<IO>::scalar(src + label), 0.0};
        mine[1 + part] = p;
    }
}
// by one wavefront, the same bits in every lane
__device__ __forceinline__ Total fold_pieces(const Total *mine, int parts, Scale c) {
    float m = -FLT_MAX;
    for (int i = 1 + (threadIdx.x & 63); i <= parts; i += 64) m = fmaxf(m, mine[i].m);
    m = wave::allreduce<64, wave::Max>(m);
    double s = 0.0;
    for (int i = 1 + (threadIdx.x & 63); i <= parts; i += 64) s += mine[i].s * exp_sum(mine[i].m - m, c);
    return Total{m, wave_sum(s)};
}

// One wavefront per row.
template <int IO>
__global__ __launch_bounds__(64) void token_logprob_fold_kernel(ScoreArgs<IO> a, const Total *__restrict__ pairs, int parts) {
    const int64_t row = blockIdx.x;
    const int label = uniform(a.labels[row]);
    RowScore r = nan_score();
    const Total *mine = pairs + row * (1 + parts);
    if (label >= 0 && label < a.cols) r = score_row(fold_pieces(mine, parts, a.c), mine[0].m, a.scale, a.c);
    if (threadIdx.x == 0) put_score(a, row, label >= 0, r);
}

// Workgroup (p, row): a piece of the row's gradient.
template <int IO, int THREADS>
__global__ __launch_bounds__(THREADS) void token_logprob_backward_kernel(const typename Io<IO>::elem *logits, int64_t ld,
                                                                         const int32_t *__restrict__ labels, float scale,
                                                                         Scale c, const float *__restrict__ row_stats,
                                                                         const float *__restrict__ dlogp,
                                                                         typename Io<IO>::elem *dlogits, int64_t ldd,
                                                                         int64_t rows, int cols) {
    typedef typename Io<IO>::elem Elem;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const int label = uniform(labels[row]);
        float coeff = uniform(dlogp[row]) * scale;
        const bool live = label >= 0 && coeff != 0.0f;
        if (label >= cols) coeff = __builtin_nanf("");
        const Elem *src = logits + row * ld;
        Elem *dst = dlogits + row * ldd;
        const RowSpan<IO> span = span_of<IO>(dst, cols);
        const int parts = static_cast<int>(gridDim.x), part = static_cast<int>(blockIdx.x);
        const int lo = piece_begin(span.nvec, parts, part), hi = piece_begin(span.nvec, parts, part + 1);
        const float top = live ? uniform(row_stats[2 * row]) : 0.0f;
        const float logsum = live ? uniform(row_stats[2 * row + 1]) : 0.0f;
        const float a = -coeff * __builtin_amdgcn_exp2f(-logsum * kLog2e);
        // coeff (1 - p), from p's logarithm: close to 0 that is where p has lost the difference
        const auto label_grad = [&](float x) { return -coeff * expm1f((x - top) * scale - logsum); };
        write_gradient<IO, THREADS>(src, dst, span, lo, hi, part == 0, live, label, top, a, label_grad, c);
    }
}

// ------------------------------------------------------------------------------------------ clipped policy loss
// Per row with a label and a weight w that is not 0, A its advantage:
//   r = exp(logp - old), L = -min(r A, clip(r, 1 - low, 1 + high) A) + kl_coef k, k = exp(d) - d - 1, d = ref - logp;
//   loss = w L;  d loss / d logp = w (-A r where r is not clipped, + kl_coef (1 - exp(d))).
template <int IO>
struct PolicyArgs {
    typedef typename Io<IO>::elem Elem;
    const Elem *logits;
    int64_t ld;
    const int32_t *labels;
    const float *old_logp;   // null: the policy that sampled is the one that trains, r = 1
    const float *ref_logp;   // null: no KL term
    const float *advantage;
    const float *weight;     // null: 1
    float scale;
    Scale c;
    float clip_low, clip_high, kl_coef;
    float *logp;
    float *kl;
    float *loss;
    Elem *dlogits;           // null: no gradient
    int64_t ldd;
    int64_t rows;
    int cols;
    hipStream_t stream;
};

// What the gradient's writers need of a row.
struct RowGradient {
    float a, label_grad, top;
    bool live;
};

__device__ __forceinline__ RowGradient uniform_gradient(const RowGradient &g) {
    return RowGradient{uniform(g.a), uniform(g.label_grad), uniform(g.top), uniform(static_cast<int>(g.live)) != 0};
}

template <int IO>
__device__ __forceinline__ bool policy_row_counts(const PolicyArgs<IO> &a, int64_t row, int &label) {
    label = uniform(a.labels[row]);
    return label >= 0 && (!a.weight || uniform(a.weight[row]) != 0.0f);
}

// exp(d) - 1 - d, given up = exp(d) - 1: close to 0 the difference cancels, and the series takes over
// (d^2 sum_n d^n / (n + 2)!, the first term left out is below 1e-8 of the first).
__device__ __forceinline__ float kl_of(float d, float up) {
    if (!(fabsf(d) < 0.5f)) return up - d;
    float s = 1.0f / 362880.0f;
    s = __builtin_fmaf(s, d, 1.0f / 40320.0f);
    s = __builtin_fmaf(s, d, 1.0f / 5040.0f);
    s = __builtin_fmaf(s, d, 1.0f / 720.0f);
    s = __builtin_fmaf(s, d, 1.0f / 120.0f);
    s = __builtin_fmaf(s, d, 1.0f / 24.0f);
    s = __builtin_fmaf(s, d, 1.0f / 6.0f);
    s = __builtin_fmaf(s, d, 0.5f);
    return s * d * d;
}

// What a row's loss is made of beside its logits.
struct PolicyRow {
    float advantage, weight, old_logp, ref_logp, at_label;
    int label;
};
template <int IO>
__device__ __forceinline__ PolicyRow policy_inputs(const PolicyArgs<IO> &a, int64_t row, int label, float at_label) {
    return PolicyRow{a.advantage[row], a.weight ? a.weight[row] : 1.0f, a.old_logp ? a.old_logp[row] : 0.0f,
                     a.ref_logp ? a.ref_logp[row] : 0.0f, at_label, label};
}
struct PolicyOptions {
    float scale;
    Scale c;
    float clip_low, clip_high, kl_coef;
    int cols;
    bool old, ref;
};
template <int IO>
__device__ __forceinline__ PolicyOptions options_of(const PolicyArgs<IO> &a) {
    return PolicyOptions{a.scale, a.c, a.clip_low, a.clip_high, a.kl_coef, a.cols, a.old_logp != nullptr, a.ref_logp != nullptr};
}
struct PolicyResult {
    float logp, kl, loss;
    RowGradient gradient;
};
// One thread's work for a row that counts: p is the pair of the other columns.
__device__ __forceinline__ PolicyResult policy_row(const PolicyOptions &o, const PolicyRow &in, Total p) {
    const RowScore r = in.label < o.cols ? score_row(p, in.at_label, o.scale, o.c) : nan_score();
    const double adv = in.advantage, w = in.weight;
    // (without an old logp: 1, for a label at -inf too, and NaN where logp is)
    const double ratio = o.old ? expf(static_cast<float>(r.logp - static_cast<double>(in.old_logp))) : r.logp == r.logp ? 1.0 : r.logp;
    const double low = 1.0 - o.clip_low, high = 1.0 + o.clip_high;
    double kept = ratio, slope = -adv * ratio;
    if (adv > 0.0 ? ratio > high : ratio < low) {
        kept = adv > 0.0 ? high : low;
        slope = 0.0;
    }
    if (adv == 0.0 && ratio == ratio) slope = kept = 0.0;  // (no surrogate, however large the ratio; a broken row stays NaN)
    double total = -adv * kept;
    float kl = 0.0f;
    if (o.ref) {
        const float d = static_cast<float>(static_cast<double>(in.ref_logp) - r.logp);
        const float up = expm1f(d);
        kl = kl_of(d, up);
        if (o.kl_coef != 0.0f) {
            total += static_cast<double>(o.kl_coef) * kl;
            slope -= static_cast<double>(o.kl_coef) * up;
        }
    }
    const float coeff = static_cast<float>(w * slope * o.scale);
    // a row whose gradient is 0 is written without a second look at its logits
    return PolicyResult{static_cast<float>(r.logp), kl, static_cast<float>(w * total),
                        RowGradient{-coeff * r.inv_total, coeff * r.rest, r.top, coeff != 0.0f}};
}
template <int IO>
__device__ __forceinline__ void put_policy(const PolicyArgs<IO> &a, int64_t row, const PolicyResult &r) {
    if (a.logp) a.logp[row] = r.logp;
    if (a.kl) a.kl[row] = r.kl;
    a.loss[row] = r.loss;
}
__device__ __forceinline__ PolicyResult no_policy() { return PolicyResult{0.0f, 0.0f, 0.0f, RowGradient{0.0f, 0.0f, 0.0f, false}}; }

// One workgroup per row, any length and alignment: the sums, then a second read.  (Six wavefronts per SIMD as in
// token_logprob_row_kernel: 32768 rows of 8192 bf16 columns without a gradient 300 us with five, 230 with six.)
template <int IO, int THREADS>
__global__ __launch_bounds__(THREADS, THREADS < 1024 ? 6 : 1) void policy_reread_kernel(PolicyArgs<IO> a) {
    __shared__ Total slots[2][THREADS / 64];
    __shared__ RowGradient shared[2];
    int turn = 1;  // (alternates between the rows that count: others pass no barrier)
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        int label;
        const bool counts = policy_row_counts(a, row, label);
        const typename Io<IO>::elem *src = a.logits + row * a.ld;
        const RowSpan<IO> span = span_of<IO>(a.dlogits ? a.dlogits + row * a.ldd : src, a.cols);
        if (counts) {
            turn ^= 1;
            float at_label = 0.0f;
            Total p{-FLT_MAX, 0.0};
            if (label < a.cols) {
                at_label = Io<IO>::scalar(src + label);
                p = block_pair<THREADS / 64>(thread_pair<IO, THREADS>(src, span, 0, span.nvec, true, label, a.c), slots[turn],
                                             a.c);
            }
            if (threadIdx.x == 0) {
                const PolicyResult r = policy_row(options_of(a), policy_inputs(a, row, label, at_label), p);
                put_policy(a, row, r);
                shared[turn] = r.gradient;
            }
            __syncthreads();
        } else if (threadIdx.x == 0) {
            put_policy(a, row, no_policy());
        }
        if (!a.dlogits) continue;
        const RowGradient g = counts ? uniform_gradient(shared[turn]) : RowGradient{0.0f, 0.0f, 0.0f, false};
        const auto label_grad = [&](float) { return g.label_grad; };
        write_gradient<IO, THREADS>(src, a.dlogits + row * a.ldd, span, 0, span.nvec, true, g.live, label, g.top, g.a,
                                    label_grad, a.c);
    }
}

// A few rows, after token_pieces_kernel: workgroup (p, row) folds the row's pairs and writes the p-th piece.
template <int IO, int THREADS>
__global__ __launch_bounds__(THREADS) void policy_pieces_kernel(PolicyArgs<IO> a, const Total *__restrict__ pairs, int parts) {
    __shared__ RowGradient shared;
    const int64_t row = blockIdx.y;
    const int part = static_cast<int>(blockIdx.x);
    int label;
    const bool counts = policy_row_counts(a, row, label);
    if (threadIdx.x < 64) {
        PolicyResult r = no_policy();
        const Total *mine = pairs + row * (1 + parts);
        if (counts) {
            Total p{-FLT_MAX, 0.0};
            if (label < a.cols) p = fold_pieces(mine, parts, a.c);
            r = policy_row(options_of(a), policy_inputs(a, row, label, label < a.cols ? mine[0].m : 0.0f), p);
        }
        if (threadIdx.x == 0) {
            if (part == 0) put_policy(a, row, r);
            shared = r.gradient;
        }
    }
    __syncthreads();
    if (!a.dlogits) return;
    const RowGradient g = uniform_gradient(shared);
    const typename Io<IO>::elem *src = a.logits + row * a.ld;
    const RowSpan<IO> span = span_of<IO>(a.dlogits + row * a.ldd, a.cols);
    const int lo = piece_begin(span.nvec, parts, part), hi = piece_begin(span.nvec, parts, part + 1);
    const auto label_grad = [&](float) { return g.label_grad; };
    write_gradient<IO, THREADS>(src, a.dlogits + row * a.ldd, span, lo, hi, part == 0, g.live, label, g.top, g.a, label_grad,
                                a.c);
}

// Many short rows, of 64 vectors at most, as in token_logprob_short_kernel: the rows stay in the registers of a wavefront, the losses
// are worked out a row per lane, and each row's gradient follows (1 GiB of bf16 logits in rows of 512 columns 399 us, 5.4 TB/s, and
// 443 with loss_sum, whose launch follows the million rows; a wavefront per row 545 without it).
template <int IO>
__global__ __launch_bounds__(64) void policy_short_kernel(PolicyArgs<IO> a) {
    constexpr int E = Io<IO>::E;
    typedef typename Io<IO>::elem Elem;
    const int lane = threadIdx.x;
    const int64_t row0 = (blockIdx.x + static_cast<int64_t>(blockIdx.y) * gridDim.x) * kShortRows;
    if (row0 >= a.rows) return;
    const int n = a.rows - row0 < kShortRows ? static_cast<int>(a.rows - row0) : kShortRows;
    auto of = [&](float v, int i) { return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), i)); };
    const int my_label = lane < n ? a.labels[row0 + lane] : -1;
    const bool counts = my_label >= 0 && (!a.weight || a.weight[row0 + lane] != 0.0f);
    const bool reads = counts && my_label < a.cols;
    const uint64_t reading = __ballot(reads);
    const float my_at = reads ? Io<IO>::scalar(a.logits + (row0 + lane) * a.ld + my_label) : 0.0f;
    PolicyRow in{};
    if (counts) in = policy_inputs(a, row0 + lane, my_label, my_at);
    Total mine{my_at, 0.0};
    typename Io<IO>::raw r[kShortRows];
#pragma unroll
    for (int i = 0; i < kShortRows; ++i) {  // (rows that are not read have empty buffers)
        const RowSpan<IO> span = span_of<IO>(a.dlogits + (row0 + i) * a.ldd, a.cols);
        const Buffer from = buffer_of(a.logits + (row0 + i) * a.ld + span.head, reading >> i & 1 ? Io<IO>::kBytes * span.nvec : 0);
        r[i] = buffer_load<IO>(from, Io<IO>::kBytes * static_cast<uint32_t>(lane));
    }
#pragma unroll
    for (int i = 0; i < kShortRows; ++i) {
        if (!(reading >> i & 1)) continue;
        const Elem *src = a.logits + (row0 + i) * a.ld;
        const RowSpan<IO> span = span_of<IO>(a.dlogits + (row0 + i) * a.ldd, a.cols);
        const int label = __builtin_amdgcn_readlane(my_label, i);
        const float shift = shift_of(of(my_at, i), a.c);
        float top = 0.0f;
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        add_vector<IO>(r[i], lane, true, span.nvec, label - span.head, shift, a.c, s, top);
        add_singles<IO, 64>(src, span, label, shift, a.c, s, top);
        const double sum = wave_total((s[0] + s[1]) + (s[2] + s[3]));
        if (lane == i) mine.s = sum;
    }
    mine.s = to_label(mine.s, my_at, shift_of(my_at, a.c), a.c);
    uint64_t again = __ballot(reads && !(static_cast<float>(mine.s) < 0x1p40f));
    while (again) {
        const int i = __builtin_ctzll(again);
        again &= again - 1;
        const Elem *src = a.logits + (row0 + i) * a.ld;
        const RowSpan<IO> span = span_of<IO>(a.dlogits + (row0 + i) * a.ldd, a.cols);
        const Total p = block_pair<1>(thread_pair<IO, 64>(src, span, 0, span.nvec, true, __builtin_amdgcn_readlane(my_label, i), a.c),
                                      nullptr, a.c);
        if (lane == i) mine = p;
    }
    const PolicyResult res = counts ? policy_row(options_of(a), in, mine) : no_policy();
    if (lane < n) put_policy(a, row0 + lane, res);
#pragma unroll
    for (int i = 0; i < kShortRows; ++i) {
        if (i >= n) break;
        const Elem *src = a.logits + (row0 + i) * a.ld;
        Elem *dst = a.dlogits + (row0 + i) * a.ldd;
        const RowSpan<IO> span = span_of<IO>(dst, a.cols);
        const int label = __builtin_amdgcn_readlane(my_label, i);
        const float factor = of(res.gradient.a, i), at_label = of(res.gradient.label_grad, i), top = of(res.gradient.top, i);
        const bool live = __builtin_amdgcn_readlane(static_cast<int>(res.gradient.live), i) != 0;
        const int in_vecs = label - span.head;
        convert_again<IO>(r[i]);
        float x[E];
        Io<IO>::unpack(r[i], x);
#pragma unroll
        for (int e = 0; e < E; ++e)
            x[e] = !live ? 0.0f : E * lane + e == in_vecs ? at_label : factor * exp_scaled(x[e] - top, a.c);
        buffer_store<IO>(buffer_of(dst + span.head, Io<IO>::kBytes * span.nvec), Io<IO>::kBytes * static_cast<uint32_t>(lane), x);
        for (int j = lane; j < span.singles; j += 64) {
            constexpr int ONE = io_by_element(IO);
            const int column = single_column(span, j);
            float v[1] = {0.0f};
            if (live) {
                v[0] = Io<IO>::scalar(src + column);
                v[0] = column == label ? at_label : factor * exp_scaled(v[0] - top, a.c);
            }
            Io<ONE>::template store<true>(dst + column, v);
        }
    }
}

// A row in the registers of a workgroup, VPT vectors per thread, one workgroup per row: one read, one write.  (Workgroups that
// walk over rows and load the next one into the registers that the gradient leaves were built and measured: 430 us against
// 386 at 4186 rows of 128256 bf16, 5.6 TB/s.  The dispatcher's order of rows serves the memory better than any fixed walk.)
// Exponentials are taken against the label's logit, not the row's maximum: exp(scale (x - x_l)) = 2^(c x - c x_l) is one fused
// multiply-add and the exponential, a sum needs no running maximum, and logp = -log1p of it.  (With the maximum the arithmetic
// of a row of 128256 took 20 us, as long as its memory traffic.)  A label so unlikely that the sum reaches 2^40, or not a
// number, is summed again from the registers, against the maximum.
// Rows have columns for more than ABOVE vectors: only a thread's last ones can lie past the
// row's end.  REST: rows longer than the registers.  What does not fit is added up before the registers fill, and read a second
// time for its gradient.
// Up to three vectors per thread 1024 threads have to leave room for a second workgroup, which the compiler has to be told: in 79
// registers instead of 58 a compute unit held one of them (24576 bf16 columns 515 us, 344 with two).
template <int IO, int ABOVE, int THREADS, int VPT, bool REST = false>
__global__ __launch_bounds__(THREADS, THREADS == 1024 && VPT <= 3 ? 8 : 1) void policy_onchip_kernel(PolicyArgs<IO> a) {
    constexpr int E = Io<IO>::E;
    // (up to a 128-byte boundary a row loses less than eight of the vectors that its columns make: it has ABOVE - 7 at least)
    constexpr int WHOLE = ABOVE < 7 ? 0 : (ABOVE - 7) / THREADS;
    constexpr int SINGLES = (128 / static_cast<int>(sizeof(typename Io<IO>::elem)) + E - 2 + THREADS - 1) / THREADS;
    typedef typename Io<IO>::elem Elem;
    __shared__ double sums[THREADS / 64];
    __shared__ Total slots[THREADS / 64];
    __shared__ RowGradient shared;
    const int64_t row = blockIdx.x + static_cast<int64_t>(blockIdx.y) * gridDim.x;
    if (row >= a.rows) return;
    const Elem *src = a.logits + row * a.ld;
    Elem *dst = a.dlogits + row * a.ldd;
    const RowSpan<IO> span = span_of<IO>(dst, a.cols);
    int label;
    if (!policy_row_counts(a, row, label)) {
        if (threadIdx.x == 0) put_policy(a, row, no_policy());
        write_gradient<IO, THREADS>(src, dst, span, 0, span.nvec, true, false, -1, 0.0f, 0.0f, [](float) { return 0.0f; }, a.c);
        return;
    }
    // vectors past the row's end read as zeros and are not written
    const Buffer from = buffer_of(src + span.head, Io<IO>::kBytes * span.nvec);
    const Buffer to = buffer_of(dst + span.head, Io<IO>::kBytes * span.nvec);
    // (offsets are formed from one register at every use, instead of kept for every k)
    uint32_t first = Io<IO>::kBytes * threadIdx.x;
    auto offset_of = [&](int k) {
        asm volatile("" : "+v"(first));
        return first + k * Io<IO>::kBytes * THREADS;
    };
    float at_label = label < a.cols ? Io<IO>::scalar(src + label) : 0.0f;
    float shift = shift_of(at_label, a.c);
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const int in_vecs = label - span.head;
    constexpr int BATCH = 8;  // vectors per thread at a time of the rest
    // the rest's vector at j, with the same exceptions as `others`
    auto rest_others = [&](const typename Io<IO>::raw &v, int j, float (&x)[E]) {
        Io<IO>::unpack(v, x);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = j >= span.nvec || E * j + e == in_vecs ? -INFINITY : x[e];
    };
    if constexpr (REST) {
        for (int j = static_cast<int>(threadIdx.x) + THREADS * VPT; uniform(j) < span.nvec; j += BATCH * THREADS) {
            typename Io<IO>::raw v[BATCH];
#pragma unroll
            for (int u = 0; u < BATCH; ++u) v[u] = buffer_load<IO>(from, Io<IO>::kBytes * static_cast<uint32_t>(j + u * THREADS));
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                if (uniform(j + u * THREADS) >= span.nvec) break;
                float x[E];
                rest_others(v[u], j + u * THREADS, x);
#pragma unroll
                for (int e = 0; e < E; ++e)
                    s[e % 4] += power_of(x[e], shift, a.c);
            }
        }
    }
    typename Io<IO>::raw r[VPT];
#pragma unroll
    for (int k = 0; k < VPT; ++k) r[k] = buffer_load<IO>(from, offset_of(k));
    float single[SINGLES];
    bool has_single[SINGLES];
    int column[SINGLES];
#pragma unroll
    for (int i = 0; i < SINGLES; ++i) {
        const int at = static_cast<int>(threadIdx.x) + i * THREADS;
        has_single[i] = at < span.singles;
        column[i] = single_column(span, at);
        single[i] = -INFINITY;
        if (has_single[i]) single[i] = Io<IO>::scalar(src + column[i]);
    }
    PolicyRow in{};
    if (threadIdx.x == 0) in = policy_inputs(a, row, label, at_label);

    // which of the threads' vectors holds the label (VPT: none)
    const int label_k = in_vecs >= 0 && in_vecs < span.nvec * E ? in_vecs / E / THREADS : VPT;
    // vector k's values, -inf at the label and past the row's end
    auto others = [&](int k, float (&x)[E]) {
        const int j = static_cast<int>(threadIdx.x) + k * THREADS;
        Io<IO>::unpack(r[k], x);
        if (label_k == k) {  // (the same in every lane)
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = E * j + e == in_vecs ? -INFINITY : x[e];
        }
        if (k >= WHOLE) {
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = j < span.nvec ? x[e] : -INFINITY;
        }
    };
    auto other_single = [&](int i) { return has_single[i] && column[i] != label ? single[i] : -INFINITY; };
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        // (in this order: vectors converted ahead would take the registers of a second row)
        asm volatile("" : "+v"(r[k]), "+v"(s[0]), "+v"(s[1]), "+v"(s[2]), "+v"(s[3]));
        float x[E];
        others(k, x);
#pragma unroll
        for (int e = 0; e < E; ++e)
            s[e % 4] += power_of(x[e], shift, a.c);
    }
#pragma unroll
    for (int i = 0; i < SINGLES; ++i)
        s[i % 4] += power_of(other_single(i), shift, a.c);
    double total = wave_total((s[0] + s[1]) + (s[2] + s[3]));
    if constexpr (THREADS > 64) {
        if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = total;
        __syncthreads();
        total = 0.0;
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) total += sums[w];
    }
    Total all{at_label, to_label(total, at_label, shift, a.c)};
    if (!(uniform(static_cast<float>(all.s)) < 0x1p40f) || label >= a.cols) {
        // against the maximum: an unlikely label, special values, or logits that c times overflows
        Pair p{-FLT_MAX, 0.0f};
#pragma unroll
        for (int k = 0; k < VPT; ++k) {
            asm volatile("" : "+v"(r[k]), "+v"(p.s));
            float x[E];
            others(k, x);
            add_values(p, x, a.c);
        }
        if constexpr (REST) {
            for (int j = static_cast<int>(threadIdx.x) + THREADS * VPT; uniform(j) < span.nvec; j += THREADS) {
                float x[E];
                rest_others(buffer_load<IO>(from, Io<IO>::kBytes * static_cast<uint32_t>(j)), j, x);
                add_values(p, x, a.c);
            }
        }
#pragma unroll
        for (int i = 0; i < SINGLES; ++i) {
            const float v[1] = {other_single(i)};
            add_values(p, v, a.c);
        }
        all = block_pair<THREADS / 64>(p, slots, a.c);
    }
    if (threadIdx.x == 0) {
        const PolicyResult res = policy_row(options_of(a), in, all);
        put_policy(a, row, res);
        shared = res.gradient;
    }
    __syncthreads();
    const RowGradient g = uniform_gradient(shared);
    float reference = g.top, less = 0.0f;
    // shift is rounded, in the end to half a step of itself: below 2^24 that makes both powers of the product below differ from what they
    // stand for by a factor of 2 at most; beyond, one may be infinite and the other 0
    constexpr float kMostShift = 0x1p24f;
    if (g.top != at_label || !(fabsf(shift) < kMostShift)) {
        // the reference is the maximum; one that far from 0 is taken off the values (what is close enough to it to count is
        // so exactly, in the storage type too: two numbers of a type within a factor of two differ by one of its numbers)
        shift = g.top * a.c.all;
        if (!(fabsf(shift) < kMostShift)) {
#pragma unroll
            for (int k = 0; k < VPT; ++k) {
                asm volatile("" : "+v"(r[k]));
                float x[E];
                Io<IO>::unpack(r[k], x);
#pragma unroll
                for (int e = 0; e < E; ++e) x[e] -= g.top;
                r[k] = pack<IO>(x);
            }
#pragma unroll
            for (int i = 0; i < SINGLES; ++i) single[i] -= g.top;
            less = g.top;
            reference = shift = 0.0f;
        }
    }
    // factor 2^(c x - shift), c of one float: the result is rounded next.  (A row that counts and has no gradient, factor
    // 0, has finite powers: its products are 0.)
    const float factor = g.a * __builtin_amdgcn_exp2f(-__builtin_fmaf(reference, a.c.all, -shift));
#pragma unroll
    for (int k = 0; k < VPT; ++k) {
        convert_again<IO>(r[k]);
        float x[E];
        Io<IO>::unpack(r[k], x);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = factor * __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], a.c.all, -shift));
        if (label_k == k) {
            const int j = static_cast<int>(threadIdx.x) + k * THREADS;
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = E * j + e == in_vecs ? g.label_grad : x[e];
        }
        buffer_store<IO>(to, offset_of(k), x);
    }
    if constexpr (REST) {
        for (int j = static_cast<int>(threadIdx.x) + THREADS * VPT; uniform(j) < span.nvec; j += BATCH * THREADS) {
            typename Io<IO>::raw v[BATCH];
#pragma unroll
            for (int u = 0; u < BATCH; ++u) v[u] = buffer_load<IO>(from, Io<IO>::kBytes * static_cast<uint32_t>(j + u * THREADS));
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                const int at = j + u * THREADS;
                if (uniform(at) >= span.nvec) break;
                float x[E];
                Io<IO>::unpack(v[u], x);
#pragma unroll
                for (int e = 0; e < E; ++e)
                    x[e] = E * at + e == in_vecs ? g.label_grad
                                                 : factor * __builtin_amdgcn_exp2f(__builtin_fmaf(x[e] - less, a.c.all, -shift));
                buffer_store<IO>(to, Io<IO>::kBytes * static_cast<uint32_t>(at), x);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < SINGLES; ++i) {
        if (has_single[i]) {
            constexpr int ONE = io_by_element(IO);
            const float x[1] = {column[i] == label ? g.label_grad
                                                   : factor * __builtin_amdgcn_exp2f(__builtin_fmaf(single[i], a.c.all, -shift))};
            Io<ONE>::template store<true>(dst + column[i], x);
        }
    }
}

// ------------------------------------------------------------------------------------------------------- sums
// out[0] = factor * sum of n values, in 64 bits and in a fixed order: one workgroup, with sixteen loads per thread in flight
// (a million values 44 us, behind 399 us of kernels over their rows of 512 bf16 columns).
__global__ __launch_bounds__(1024) void loss_sum_kernel(const float *__restrict__ values, int64_t n, float factor, float *out) {
    __shared__ double sums[16];
    double s = 0.0;
    if (n == 0) {  // the sum over no rows
        if (threadIdx.x == 0) out[0] = 0.0f;
        return;
    }
    constexpr int UNROLL = 16;
    int64_t i = threadIdx.x;
    for (; i - threadIdx.x + 1024 * UNROLL <= n; i += 1024 * UNROLL) {
        float v[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) v[u] = values[i + u * 1024];
        double two[2] = {0.0, 0.0};
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) two[u & 1] += v[u];
        s += two[0] + two[1];
    }
    float v[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) v[u] = values[i + u * 1024 < n ? i + u * 1024 : n - 1];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) s += i + u * 1024 < n ? v[u] : 0.0f;
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x != 0) return;
    s = 0.0;
    for (int w = 0; w < 16; ++w) s += sums[w];
    out[0] = static_cast<float>(factor * s);
}

// ------------------------------------------------------------------------------------------------ preference loss
// Pair p: sequence 2p is the chosen one, 2p + 1 the rejected one; sequence i's tokens are [offsets[i], offsets[i + 1]).
//   reward_i = beta sum (logp - ref), h = reward_chosen - reward_rejected,
//   loss = (1 - eps) softplus(-h) + eps softplus(h),  d loss / d h = eps - 1 / (1 + exp(h)).
// Sums in 64 bits; one workgroup per pair.
struct PreferenceArgs {
    const float *logp;
    const float *ref_logp;
    const int32_t *labels;   // null, or: tokens with a negative label count for nothing
    const int32_t *offsets;
    int64_t pairs, tokens;
    float beta, eps, pair_weight;
    float *pair_loss;
    float *rewards;
    float *dlogp;
};
// Where a pair's sequences lie: [at[0], at[1]) and [at[1], at[2]).  Offsets are the caller's device data: none of them leads
// outside the tokens, and within the pair none leads backwards.
__device__ __forceinline__ void pair_span(const PreferenceArgs &a, int64_t pair, int64_t (&at)[3]) {
    for (int i = 0; i < 3; ++i) {
        at[i] = a.offsets[2 * pair + i];
        if (at[i] < (i ? at[i - 1] : 0)) at[i] = i ? at[i - 1] : 0;
        if (at[i] > a.tokens) at[i] = a.tokens;
    }
}
// Where a pair's gradient begins: at the largest offset up to its own, which in ascending offsets is its own.  Offsets that go
// backwards from one pair to the next let pairs share tokens; no token's gradient is then written by two of them, one of which
// would win by its timing.  `most`: a lane's largest offset among those up to the pair's.
__device__ __forceinline__ int wave_most(int v, int64_t own) {
    if (!__any(v > own)) return static_cast<int>(own);  // (the ordinary case)
#pragma unroll
    for (int step = 1; step < 64; step <<= 1) {
        const int other = __shfl_xor(v, step, 64);
        v = v > other ? v : other;
    }
    return v;
}
__device__ __forceinline__ int64_t gradient_from(const PreferenceArgs &a, int most, int64_t own) {
    const int64_t from = most > own ? most : own;
    return from < a.tokens ? from : a.tokens;
}
// A thread's share of a pair's sums, `thread` of `threads`.
__device__ __forceinline__ void pair_sums(const PreferenceArgs &a, const int64_t (&at)[3], int thread, int threads, double (&s)[2]) {
    s[0] = s[1] = 0.0;
    constexpr int UNROLL = 4;
    for (int64_t t0 = at[0] + thread; t0 < at[2]; t0 += threads * UNROLL) {
        float lp[UNROLL], ref[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int64_t t = t0 + u * threads;
            lp[u] = ref[u] = 0.0f;
            if (t < at[2] && (!a.labels || a.labels[t] >= 0)) {
                lp[u] = a.logp[t];
                ref[u] = a.ref_logp[t];
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) s[t0 + u * threads < at[1] ? 0 : 1] += static_cast<double>(lp[u]) - static_cast<double>(ref[u]);
    }
}
// The pair's loss, from its rewards; `write`: one thread puts the results.  Returns dlogp of the chosen sequence's tokens.
__device__ __forceinline__ float pair_result(const PreferenceArgs &a, int64_t pair, const double (&reward)[2], bool write, float &loss) {
    const double h = reward[0] - reward[1];
    const double slope = a.eps - 1.0 / (1.0 + exp(h));
    if (write) {
        const double both = log1p(exp(-fabs(h)));
        // (a side without a share adds nothing, however far apart the rewards)
        double l = 0.0;
        if (a.eps != 1.0f) l = (1.0 - a.eps) * (both + (h < 0.0 ? -h : 0.0));
        if (a.eps != 0.0f) l += a.eps * (both + (h > 0.0 ? h : 0.0));
        loss = static_cast<float>(l);
        a.pair_loss[pair] = loss;
        if (a.rewards) {
            a.rewards[2 * pair] = static_cast<float>(reward[0]);
            a.rewards[2 * pair + 1] = static_cast<float>(reward[1]);
        }
    }
    return static_cast<float>(slope * a.beta * a.pair_weight);
}
__device__ __forceinline__ void pair_gradient(const PreferenceArgs &a, const int64_t (&at)[3], int64_t from, int thread, int threads,
                                              float up) {
    if (!a.dlogp) return;
    for (int64_t t = from + thread; t < at[2]; t += threads)
        a.dlogp[t] = a.labels && a.labels[t] < 0 ? 0.0f : t < at[1] ? up : -up;
}

// Every pair's largest offset up to its own, for many pairs: into pair_loss, whose entries their pairs' workgroups read before they
// write the losses there.  One workgroup: a prefix maximum over PER pairs per thread at a time, whose offsets pass through LDS, the
// next ones on their way meanwhile (65536 pairs 452 us with this launch, 500 with each thread reading its own stretch of the
// offsets, 384 without).  Up to kManyPairs a pair's workgroup reads the offsets before its own itself (1024 pairs 12.3 us, 11.5
// without); that grows with the square of the pairs.
constexpr int64_t kManyPairs = 1024;
__global__ __launch_bounds__(1024) void preference_offsets_kernel(const int32_t *__restrict__ offsets, int64_t pairs, int32_t *most) {
    constexpr int PER = 4;
    __shared__ int window[2 * PER * 1024];  // offsets 2 base - 1 and on: two per pair
    __shared__ int totals[2][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int next[2 * PER];
    auto fetch = [&](int64_t base) {  // (beyond either end: the last one there)
#pragma unroll
        for (int u = 0; u < 2 * PER; ++u) {
            int64_t at = 2 * base - 1 + static_cast<int>(threadIdx.x) + u * 1024;
            at = at < 0 ? 0 : at;
            next[u] = offsets[at < 2 * pairs ? at : 2 * pairs];
        }
    };
    fetch(0);
    int before = INT32_MIN, turn = 0;
    for (int64_t base = 0; base < pairs; base += 1024 * PER, turn ^= 1) {
#pragma unroll
        for (int u = 0; u < 2 * PER; ++u) window[threadIdx.x + u * 1024] = next[u];
        __syncthreads();
        int v[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int *at = window + 2 * (PER * threadIdx.x + i);
            v[i] = max(at[0], at[1]);
            if (i > 0) v[i] = max(v[i], v[i - 1]);
        }
        if (base + 1024 * PER < pairs) fetch(base + 1024 * PER);
        int sum = v[PER - 1];  // the maximum over the threads up to this one
#pragma unroll
        for (int step = 1; step < 64; step <<= 1) {
            const int other = __shfl_up(sum, step, 64);
            if (lane >= step) sum = max(sum, other);
        }
        if (lane == 63) totals[turn][wave] = sum;
        __syncthreads();
        int earlier = __shfl_up(sum, 1, 64);
        earlier = lane == 0 ? before : max(earlier, before);
        for (int w = 0; w < 16; ++w) {
            if (w < wave) earlier = max(earlier, totals[turn][w]);
            before = max(before, totals[turn][w]);
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int64_t pair = base + PER * static_cast<int>(threadIdx.x) + i;
            if (pair < pairs) most[pair] = max(v[i], earlier);
        }
    }
}

constexpr int kPreferenceThreads = 512;
__global__ __launch_bounds__(kPreferenceThreads) void preference_kernel(PreferenceArgs a) {
    constexpr int WAVES = kPreferenceThreads / 64;
    __shared__ double sums[2][WAVES];
    __shared__ int most[WAVES];
    for (int64_t pair = blockIdx.x; pair < a.pairs; pair += gridDim.x) {
        int64_t at[3];
        pair_span(a, pair, at);
        int mine = INT32_MIN;
        if (a.dlogp) {
            if (a.pairs > kManyPairs) {
                mine = __builtin_bit_cast(int, a.pair_loss[pair]);
            } else {
                constexpr int LOADS = static_cast<int>(2 * kManyPairs / kPreferenceThreads);
                int v[LOADS];
#pragma unroll
                for (int u = 0; u < LOADS; ++u) {
                    const int i = static_cast<int>(threadIdx.x) + u * kPreferenceThreads;
                    v[u] = i < 2 * pair ? a.offsets[i] : INT32_MIN;
                }
#pragma unroll
                for (int u = 0; u < LOADS; ++u) mine = max(mine, v[u]);
            }
        }
        double s[2];
        pair_sums(a, at, threadIdx.x, kPreferenceThreads, s);
        __syncthreads();  // the previous pair's sums have been read
        mine = wave_most(mine, at[0]);
        if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = mine;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            s[i] = wave_sum(s[i]);
            if ((threadIdx.x & 63) == 0) sums[i][threadIdx.x >> 6] = s[i];
        }
        __syncthreads();
        double reward[2];
        for (int i = 0; i < 2; ++i) {
            reward[i] = 0.0;
            for (int w = 0; w < WAVES; ++w) reward[i] += sums[i][w];
            reward[i] *= a.beta;
        }
        for (int w = 0; w < WAVES; ++w) mine = max(mine, most[w]);
        float loss;
        const float up = pair_result(a, pair, reward, threadIdx.x == 0, loss);
        pair_gradient(a, at, gradient_from(a, mine, at[0]), threadIdx.x, kPreferenceThreads, up);
    }
}

// Few pairs of few tokens: all of them in one workgroup, 16 / SIDE wavefronts per pair, and the sum of their losses with them -
// one launch instead of two (called over and over on data in the caches: 2 pairs of 2 x 40 tokens 4.5 us instead of 7.0, 8 pairs of
// 2 x 512 6.3 and 7.1; 8 pairs of 2 x 1000 9.5 against 7.6).  Behind a kernel over logits, with nothing in the caches, 8 pairs of
// 2 x 128 to 2 x 512 tokens take 10.5 to 11.6 us: 5 to 8 pairs have one wavefront each, half of the workgroup, and wait for their labels
// before they ask for the rest.
constexpr int kFewPairs = 16;
constexpr int64_t kFewTokens = 8192;
template <int SIDE>
__global__ __launch_bounds__(1024) void preference_few_kernel(PreferenceArgs a, float *loss_sum) {
    constexpr int WAVES = 16 / SIDE, THREADS = 64 * WAVES;
    __shared__ double sums[2][16];
    __shared__ float losses[SIDE];
    const int wave = threadIdx.x >> 6, pair = wave / WAVES, thread = threadIdx.x % THREADS;
    const bool here = pair < a.pairs;
    int64_t at[3] = {0, 0, 0};
    if (here) pair_span(a, pair, at);
    static_assert(2 * kFewPairs <= 64, "a lane per offset");
    const int lane = threadIdx.x & 63;
    const int offset = here && lane < 2 * pair ? a.offsets[lane] : INT32_MIN;
    double s[2];
    pair_sums(a, at, thread, THREADS, s);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        s[i] = wave_sum(s[i]);
        if ((threadIdx.x & 63) == 0) sums[i][wave] = s[i];
    }
    __syncthreads();
    if (here) {
        double reward[2];
        for (int i = 0; i < 2; ++i) {
            reward[i] = 0.0;
            for (int w = 0; w < WAVES; ++w) reward[i] += sums[i][pair * WAVES + w];
            reward[i] *= a.beta;
        }
        float loss = 0.0f;
        const float up = pair_result(a, pair, reward, thread == 0, loss);
        if (thread == 0) losses[pair] = loss;
        pair_gradient(a, at, gradient_from(a, wave_most(offset, at[0]), at[0]), thread, THREADS, up);
    }
    __syncthreads();
    if (threadIdx.x != 0 || !loss_sum) return;
    double total = 0.0;
    for (int p = 0; p < a.pairs; ++p) total += losses[p];
    loss_sum[0] = static_cast<float>(a.pair_weight * total);
}

// ---------------------------------------------------------------------------------------------------- dispatch
// Pieces per row of a few long rows: a function of the sizes alone, so that the workspace can be sized without a device.  Up to
// 64K columns a workgroup per row takes less time than a second launch (16 rows of 30522 fp32 columns 6.0 us against 7.7, with
// the policy loss 7.3 against 9.4; 32 rows of 50257 binary16 columns with their gradient 17.8 against 21.2); 16 rows of 100000
// take 8.8 us whole and 7.7 in pieces, the policy loss 12.5 and 9.2.  128 rows are enough workgroups of their own (13 us against 21).
constexpr int kPieceUnits = 256;  // compute units of an MI355X
constexpr int64_t kPieceColumns = 4096;
constexpr int64_t kWholeColumns = 64 << 10;
int pieces_per_row(int64_t rows, int64_t cols) {
    if (rows <= 0 || rows * 4 > kPieceUnits || cols <= kWholeColumns) return 1;
    const int64_t parts = 2 * kPieceUnits / rows;
    return static_cast<int>(parts < cols / kPieceColumns ? parts : cols / kPieceColumns);
}
size_t workspace_bytes(int64_t rows, int64_t cols) {
    if (rows <= 0 || cols <= 0 || cols > kMaxColumns) return 0;
    const int parts = pieces_per_row(rows, cols);
    return parts > 1 ? static_cast<size_t>(rows) * (1 + parts) * sizeof(Total) : 0;
}

Scale two_parts(float scale) {
    const double c = static_cast<double>(scale) * 1.4426950408889634;
    int exponent;
    const double fraction = frexp(c, &exponent);
    const float hi = static_cast<float>(ldexp(floor(ldexp(fraction, 16)), exponent - 16));
    // (lo > 0: -inf times either part is -inf)
    const float lo = static_cast<float>(c - hi);
    return Scale{hi, lo > 1e-37f ? lo : 1e-37f, static_cast<float>(c)};
}

// What every entry on rows of logits checks.
int check_logits(const char *who, const void *logits, int64_t ld, const void *labels, size_t size, float scale, int64_t rows,
                 int64_t cols, const void *workspace, size_t bytes) {
    if (rows < 0 || cols <= 0) return fail(KO_ERR_INVALID_ARGUMENT, "%s: rows=%lld cols=%lld", who, (long long)rows, (long long)cols);
    if (cols > kMaxColumns) return fail(KO_ERR_UNSUPPORTED_SHAPE, "%s: cols=%lld too large", who, (long long)cols);
    if (ld < cols) return fail(KO_ERR_INVALID_ARGUMENT, "%s: ld=%lld is less than cols=%lld", who, (long long)ld, (long long)cols);
    if (!(scale >= 1e-20f && scale <= 1e20f)) return fail(KO_ERR_INVALID_ARGUMENT, "%s: scale=%g", who, static_cast<double>(scale));
    if (rows > 0 && (!logits || !labels)) return fail(KO_ERR_INVALID_ARGUMENT, "%s: null logits/labels pointer", who);
    if ((reinterpret_cast<uintptr_t>(logits) & (size - 1)) || (reinterpret_cast<uintptr_t>(labels) & 3))
        return fail(KO_ERR_INVALID_ARGUMENT, "%s: logits/labels must be aligned to their element type", who);
    if (workspace && bytes < workspace_bytes(rows, cols))
        return fail(KO_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes, %zu needed", who, bytes, workspace_bytes(rows, cols));
    if (reinterpret_cast<uintptr_t>(workspace) & 15)
        return fail(KO_ERR_INVALID_ARGUMENT, "%s: workspace must be 16-byte aligned", who);
    return KO_OK;
}
int check_gradient(const char *who, const void *dlogits, int64_t ldd, const void *logits, int64_t ld, size_t size, int64_t rows,
                   int64_t cols) {
    if (ldd < cols) return fail(KO_ERR_INVALID_ARGUMENT, "%s: ldd=%lld is less than cols=%lld", who, (long long)ldd, (long long)cols);
    if (reinterpret_cast<uintptr_t>(dlogits) & (size - 1))
        return fail(KO_ERR_INVALID_ARGUMENT, "%s: dlogits must be aligned to its element type", who);
    if (dlogits && dlogits == logits && rows > 1 && ldd != ld)  // a row's gradient would fall on other rows' logits
        return fail(KO_ERR_INVALID_ARGUMENT, "%s: dlogits is logits, but ldd=%lld is not ld=%lld", who, (long long)ldd, (long long)ld);
    return KO_OK;
}
int check_floats(const char *who, std::initializer_list<const void *> pointers) {
    for (const void *p : pointers)
        if (reinterpret_cast<uintptr_t>(p) & 3) return fail(KO_ERR_INVALID_ARGUMENT, "%s: fp32 arrays must be 4-byte aligned", who);
    return KO_OK;
}
// Rows of logits and of their gradient lie alike: every row starts at the same place of a 16-byte vector in both.
bool rows_lie_alike(const void *logits, int64_t ld, const void *dlogits, int64_t ldd, size_t size) {
    const uintptr_t base = reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(dlogits);
    return (base & 15) == 0 && ((static_cast<uint64_t>(ld) - static_cast<uint64_t>(ldd)) * size & 15) == 0;
}

template <int IO, int THREADS>
int launch_pieces(const typename Io<IO>::elem *logits, int64_t ld, const int32_t *labels, const float *weight, int64_t rows,
                  int cols, Scale c, Total *pairs, int parts, hipStream_t stream) {
    token_pieces_kernel<IO, THREADS><<<dim3(static_cast<unsigned>(parts), static_cast<unsigned>(rows)), dim3(THREADS), 0, stream>>>(
        logits, ld, labels, weight, cols, c, pairs);
    KO_CHECK_LAUNCH();
    return KO_OK;
}

template <int IO>
int logprob_entry(const void *logits, int64_t ld, const int32_t *labels, float scale, float *logp, float *row_stats,
                  int64_t rows, int64_t cols, void *workspace, size_t bytes, ko_stream_t stream) {
    typedef typename Io<IO>::elem Elem;
    static const char *const who = "token_logprob";
    if (const int st = check_logits(who, logits, ld, labels, sizeof(Elem), scale, rows, cols, workspace, bytes); st != KO_OK) return st;
    if (const int st = check_floats(who, {logp, row_stats}); st != KO_OK) return st;
    if (rows == 0) return KO_OK;
    if (!logp) return fail(KO_ERR_INVALID_ARGUMENT, "%s: null logp pointer", who);
    const ScoreArgs<IO> a{static_cast<const Elem *>(logits), ld, labels, scale, two_parts(scale), logp, row_stats, rows,
                          static_cast<int>(cols), as_stream(stream)};
    const int parts = pieces_per_row(rows, cols);
    if (workspace && parts > 1) {
        Total *pairs = static_cast<Total *>(workspace);
        if (const int st = launch_pieces<IO, 256>(a.logits, ld, labels, nullptr, rows, a.cols, a.c, pairs, parts, a.stream); st != KO_OK)
            return st;
        token_logprob_fold_kernel<IO><<<dim3(static_cast<unsigned>(rows)), dim3(64), 0, a.stream>>>(a, pairs, parts);
        KO_CHECK_LAUNCH();
        return KO_OK;
    }
    const dim3 grid = row_grid(rows, 1024);
    const int nvec = a.cols / Io<IO>::E;
    // rows of few vectors: as many threads as make one batch of them (when tried, 1 GiB of bf16 rows: 8192 columns 187 us, 208 with
    // 512 threads; 4096 columns 190, 383 with 256 threads, half of them idle).  Long rows: 1024 threads took 258 us for 1 GiB of rows of
    // 50257 bf16 columns, 512 take 154, and 32 such rows 6.7 against 7.2.
    if (nvec <= 128 && rows >= kManyRows) {
        const dim3 g = row_grid((rows + kShortRows - 1) / kShortRows, 64);
        if (nvec <= 64) token_logprob_short_kernel<IO, 1><<<g, dim3(64), 0, a.stream>>>(a);
        else token_logprob_short_kernel<IO, 2><<<g, dim3(64), 0, a.stream>>>(a);
    } else if (nvec <= 128) token_logprob_row_kernel<IO, 64, 2><<<grid, dim3(64), 0, a.stream>>>(a);
    else if (nvec <= 256) token_logprob_row_kernel<IO, 64, 4><<<grid, dim3(64), 0, a.stream>>>(a);
    else if (nvec <= 512) token_logprob_row_kernel<IO, 128, 4><<<grid, dim3(128), 0, a.stream>>>(a);
    else if (nvec <= 1024) token_logprob_row_kernel<IO, 256, 4><<<grid, dim3(256), 0, a.stream>>>(a);
    else token_logprob_row_kernel<IO, 512, 4><<<grid, dim3(512), 0, a.stream>>>(a);
    KO_CHECK_LAUNCH();
    return KO_OK;
}

template <int IO, int THREADS>
int launch_logprob_backward(const void *logits, int64_t ld, const int32_t *labels, float scale, const float *row_stats,
                            const float *dlogp, void *dlogits, int64_t ldd, int64_t rows, int64_t cols, hipStream_t stream) {
    typedef typename Io<IO>::elem Elem;
    // pieces of two trips of a workgroup
    const int64_t piece = int64_t{THREADS} * 4 * Io<IO>::E;
    const unsigned parts = static_cast<unsigned>((cols + piece - 1) / piece);
    const unsigned grid_rows = static_cast<unsigned>(rows > 65535 ? 65535 : rows);
    token_logprob_backward_kernel<IO, THREADS><<<dim3(parts, grid_rows), dim3(THREADS), 0, stream>>>(
        static_cast<const Elem *>(logits), ld, labels, scale, two_parts(scale), row_stats, dlogp, static_cast<Elem *>(dlogits), ldd,
        rows, static_cast<int>(cols));
    KO_CHECK_LAUNCH();
    return KO_OK;
}

template <int IO>
int logprob_backward_entry(const void *logits, int64_t ld, const int32_t *labels, float scale, const float *row_stats,
                           const float *dlogp, void *dlogits, int64_t ldd, int64_t rows, int64_t cols, ko_stream_t stream) {
    constexpr size_t kSize = sizeof(typename Io<IO>::elem);
    static const char *const who = "token_logprob_backward";
    if (const int st = check_logits(who, logits, ld, labels, kSize, scale, rows, cols, nullptr, 0); st != KO_OK) return st;
    if (const int st = check_gradient(who, dlogits, ldd, logits, ld, kSize, rows, cols); st != KO_OK) return st;
    if (const int st = check_floats(who, {row_stats, dlogp}); st != KO_OK) return st;
    if (rows == 0) return KO_OK;
    if (!row_stats || !dlogp || !dlogits) return fail(KO_ERR_INVALID_ARGUMENT, "%s: null row_stats/dlogp/dlogits pointer", who);
    if (rows_lie_alike(logits, ld, dlogits, ldd, kSize)) {
        // short rows: one wavefront each (1 GiB of bf16 rows: 512 columns 383 us, 740 with 256 threads, 1024 columns 365 against
        // 472, 2048 columns 376 against 343)
        if (cols <= 128 * Io<IO>::E)
            return launch_logprob_backward<IO, 64>(logits, ld, labels, scale, row_stats, dlogp, dlogits, ldd, rows, cols, as_stream(stream));
        return launch_logprob_backward<IO, 256>(logits, ld, labels, scale, row_stats, dlogp, dlogits, ldd, rows, cols, as_stream(stream));
    }
    return launch_logprob_backward<io_by_element(IO), 256>(logits, ld, labels, scale, row_stats, dlogp, dlogits, ldd, rows, cols,
                                                      as_stream(stream));
}

template <int IO, int ABOVE, int THREADS, int VPT, bool REST = false>
int launch_onchip(const PolicyArgs<IO> &a) {
    static_assert(REST ? ABOVE >= THREADS * VPT + 7 : ABOVE < THREADS * VPT, "");
    const int nvec = a.cols / Io<IO>::E;
    if ((ABOVE && nvec <= ABOVE) || (!REST && nvec > THREADS * VPT)) return fail(KO_ERR_UNSUPPORTED_SHAPE, "policy_loss: cols=%d", a.cols);
    // (a grid's threads number less than 2^32 in one dimension)
    const int64_t wide = a.rows < (1 << 20) ? a.rows : (1 << 20);
    const int64_t high = (a.rows + wide - 1) / wide;
    if (high > 65535) return fail(KO_ERR_UNSUPPORTED_SHAPE, "policy_loss: rows=%lld too many", (long long)a.rows);
    const dim3 g(static_cast<unsigned>(wide), static_cast<unsigned>(high)), b(THREADS);
    policy_onchip_kernel<IO, ABOVE, THREADS, VPT, REST><<<g, b, 0, a.stream>>>(a);
    KO_CHECK_LAUNCH();
    return KO_OK;
}

template <int IO>
int launch_short(const PolicyArgs<IO> &a) {
    const int64_t groups = (a.rows + kShortRows - 1) / kShortRows;
    const int64_t wide = groups < (1 << 20) ? groups : (1 << 20);
    const int64_t high = (groups + wide - 1) / wide;
    if (high > 65535) return fail(KO_ERR_UNSUPPORTED_SHAPE, "policy_loss: rows=%lld too many", (long long)a.rows);
    policy_short_kernel<IO><<<dim3(static_cast<unsigned>(wide), static_cast<unsigned>(high)), dim3(64), 0, a.stream>>>(a);
    KO_CHECK_LAUNCH();
    return KO_OK;
}

template <int IO>
int launch_policy(const PolicyArgs<IO> &a, void *workspace) {
    const int parts = pieces_per_row(a.rows, a.cols);
    if (workspace && parts > 1) {
        Total *pairs = static_cast<Total *>(workspace);
        if (const int st = launch_pieces<IO, 256>(a.logits, a.ld, a.labels, a.weight, a.rows, a.cols, a.c, pairs, parts, a.stream);
            st != KO_OK)
            return st;
        const dim3 grid(a.dlogits ? static_cast<unsigned>(parts) : 1u, static_cast<unsigned>(a.rows));
        policy_pieces_kernel<IO, 256><<<grid, dim3(256), 0, a.stream>>>(a, pairs, parts);
        KO_CHECK_LAUNCH();
        return KO_OK;
    }
    if constexpr (Io<IO>::E > 1) {
        const int nvec = a.cols / Io<IO>::E;
        if (a.dlogits) {
            // Four vectors per thread, where the rows fit a workgroup that way: 4096 bf16 columns 338 us for 1 GiB of logits
            // against 356 with eight and 372 with two per thread, 1024 columns 393 against 675 with one.  Long rows: 512 threads
            // (two workgroups per compute unit, one of which loads or stores) as far as their registers go, 49152 columns
            // 369 us against 412 with 1024 threads; three per thread where that is the number (24576 columns 344,
            // with 512 threads and eight 352; 16400 columns 451 and 433).
            if (nvec <= 64 && a.rows >= 2 * kManyRows) return launch_short<IO>(a);
            if (nvec <= 64) return launch_onchip<IO, 0, 64, 1>(a);
            if (nvec <= 128) return launch_onchip<IO, 64, 64, 2>(a);
            if (nvec <= 256) return launch_onchip<IO, 128, 64, 4>(a);
            if (nvec <= 512) return launch_onchip<IO, 256, 128, 4>(a);
            if (nvec <= 1024) return launch_onchip<IO, 512, 256, 4>(a);
            if (nvec <= 3 * 512) return launch_onchip<IO, 1024, 512, 3>(a);
            if (nvec <= 4 * 512) return launch_onchip<IO, 3 * 512, 512, 4>(a);
            if (nvec <= 3 * 1024) return launch_onchip<IO, 4 * 512, 1024, 3>(a);
            if (nvec <= 8 * 512) return launch_onchip<IO, 3 * 1024, 512, 8>(a);
            if (nvec <= 10 * 512) return launch_onchip<IO, 8 * 512, 512, 10>(a);
            if (nvec <= 12 * 512) return launch_onchip<IO, 10 * 512, 512, 12>(a);
            if (nvec <= 16 * 512) return launch_onchip<IO, 12 * 512, 512, 16>(a);
            if (nvec <= 10 * 1024) return launch_onchip<IO, 16 * 512, 1024, 10>(a);
            if (nvec <= 12 * 1024) return launch_onchip<IO, 10 * 1024, 1024, 12>(a);
            if (nvec <= 14 * 1024) return launch_onchip<IO, 12 * 1024, 1024, 14>(a);
            if (nvec <= 16 * 1024) return launch_onchip<IO, 14 * 1024, 1024, 16>(a);
            return launch_onchip<IO, 16 * 1024, 1024, 15, true>(a);
        }
    }
    // no gradient (1 GiB of bf16 logits: 512 columns 2.6 ms, 8192 columns 442 us, 50257 columns 318), and rows that lie differently in
    // the two matrices
    const dim3 grid = row_grid(a.rows, 1024);
    if (a.cols <= 4096) policy_reread_kernel<IO, 256><<<grid, dim3(256), 0, a.stream>>>(a);
    else if (a.cols <= 32768) policy_reread_kernel<IO, 512><<<grid, dim3(512), 0, a.stream>>>(a);
    else policy_reread_kernel<IO, 1024><<<grid, dim3(1024), 0, a.stream>>>(a);
    KO_CHECK_LAUNCH();
    return KO_OK;
}

int launch_loss_sum(const float *values, int64_t n, float factor, float *out, hipStream_t stream) {
    loss_sum_kernel<<<dim3(1), dim3(1024), 0, stream>>>(values, n, factor, out);
    KO_CHECK_LAUNCH();
    return KO_OK;
}

template <int IO>
int policy_entry(const void *logits, int64_t ld, const int32_t *labels, const float *old_logp, const float *ref_logp,
                 const float *advantage, const float *weight, float scale, float clip_low, float clip_high, float kl_coef,
                 float *logp, float *kl, float *loss, float *loss_sum, void *dlogits, int64_t ldd, int64_t rows, int64_t cols,
                 void *workspace, size_t bytes, ko_stream_t stream) {
    typedef typename Io<IO>::elem Elem;
    static const char *const who = "policy_loss";
    if (const int st = check_logits(who, logits, ld, labels, sizeof(Elem), scale, rows, cols, workspace, bytes); st != KO_OK) return st;
    if (dlogits) {
        if (const int st = check_gradient(who, dlogits, ldd, logits, ld, sizeof(Elem), rows, cols); st != KO_OK) return st;
    }
    if (const int st = check_floats(who, {old_logp, ref_logp, advantage, weight, logp, kl, loss, loss_sum}); st != KO_OK) return st;
    if (!(clip_low >= 0.0f && clip_low <= 1.0f) || !(clip_high >= 0.0f && clip_high < INFINITY))
        return fail(KO_ERR_INVALID_ARGUMENT, "%s: clip_low=%g clip_high=%g", who, static_cast<double>(clip_low), static_cast<double>(clip_high));
    if (!(kl_coef > -INFINITY && kl_coef < INFINITY)) return fail(KO_ERR_INVALID_ARGUMENT, "%s: kl_coef=%g", who, static_cast<double>(kl_coef));
    const hipStream_t s = as_stream(stream);
    if (rows == 0) return loss_sum ? launch_loss_sum(nullptr, 0, 1.0f, loss_sum, s) : KO_OK;
    if (!advantage || !loss) return fail(KO_ERR_INVALID_ARGUMENT, "%s: null advantage/loss pointer", who);
    auto run = [&](auto kind) {
        constexpr int KIND = decltype(kind)::value;
        const PolicyArgs<KIND> a{static_cast<const Elem *>(logits), ld, labels, old_logp, ref_logp, advantage, weight, scale,
                                 two_parts(scale), clip_low, clip_high, kl_coef, logp, kl, loss, static_cast<Elem *>(dlogits), ldd,
                                 rows, static_cast<int>(cols), s};
        return launch_policy<KIND>(a, workspace);
    };
    const bool alike = !dlogits || rows_lie_alike(logits, ld, dlogits, ldd, sizeof(Elem));
    const int st = alike ? run(std::integral_constant<int, IO>{}) : run(std::integral_constant<int, io_by_element(IO)>{});
    if (st != KO_OK || !loss_sum) return st;
    return launch_loss_sum(loss, rows, 1.0f, loss_sum, s);
}

}  // namespace
}  // namespace ko

KO_EXPORT size_t ko_token_logprob_workspace_bytes(int64_t rows, int64_t cols) { return ko::workspace_bytes(rows, cols); }

KO_EXPORT int ko_token_logprob_f32(const float *logits, int64_t ld, const int32_t *labels, float scale, float *logp,
                                   float *row_stats, int64_t rows, int64_t cols, void *workspace, size_t workspace_bytes,
                                   ko_stream_t stream) {
    return ko::logprob_entry<ko::IO_F32>(logits, ld, labels, scale, logp, row_stats, rows, cols, workspace, workspace_bytes, stream);
}

KO_EXPORT int ko_token_logprob_16(const void *logits, int64_t ld, const int32_t *labels, float scale, float *logp,
                                  float *row_stats, int64_t rows, int64_t cols, int dtype, void *workspace,
                                  size_t workspace_bytes, ko_stream_t stream) {
    if (dtype == KO_F16)
        return ko::logprob_entry<ko::IO_F16>(logits, ld, labels, scale, logp, row_stats, rows, cols, workspace, workspace_bytes, stream);
    if (dtype == KO_BF16)
        return ko::logprob_entry<ko::IO_BF16>(logits, ld, labels, scale, logp, row_stats, rows, cols, workspace, workspace_bytes, stream);
    return ko::fail(KO_ERR_INVALID_ARGUMENT, "token_logprob: dtype=%d is neither KO_F16 nor KO_BF16", dtype);
}

KO_EXPORT int ko_token_logprob_backward_f32(const float *logits, int64_t ld, const int32_t *labels, float scale,
                                            const float *row_stats, const float *dlogp, float *dlogits, int64_t ldd, int64_t rows,
                                            int64_t cols, ko_stream_t stream) {
    return ko::logprob_backward_entry<ko::IO_F32>(logits, ld, labels, scale, row_stats, dlogp, dlogits, ldd, rows, cols, stream);
}

KO_EXPORT int ko_token_logprob_backward_16(const void *logits, int64_t ld, const int32_t *labels, float scale,
                                           const float *row_stats, const float *dlogp, void *dlogits, int64_t ldd, int64_t rows,
                                           int64_t cols, int dtype, ko_stream_t stream) {
    if (dtype == KO_F16)
        return ko::logprob_backward_entry<ko::IO_F16>(logits, ld, labels, scale, row_stats, dlogp, dlogits, ldd, rows, cols, stream);
    if (dtype == KO_BF16)
        return ko::logprob_backward_entry<ko::IO_BF16>(logits, ld, labels, scale, row_stats, dlogp, dlogits, ldd, rows, cols, stream);
    return ko::fail(KO_ERR_INVALID_ARGUMENT, "token_logprob_backward: dtype=%d is neither KO_F16 nor KO_BF16", dtype);
}

KO_EXPORT int ko_policy_loss_f32(const float *logits, int64_t ld, const int32_t *labels, const float *old_logp,
                                 const float *ref_logp, const float *advantage, const float *weight, float scale, float clip_low,
                                 float clip_high, float kl_coef, float *logp, float *kl, float *loss, float *loss_sum,
                                 float *dlogits, int64_t ldd, int64_t rows, int64_t cols, void *workspace, size_t workspace_bytes,
                                 ko_stream_t stream) {
    return ko::policy_entry<ko::IO_F32>(logits, ld, labels, old_logp, ref_logp, advantage, weight, scale, clip_low, clip_high,
                                        kl_coef, logp, kl, loss, loss_sum, dlogits, ldd, rows, cols, workspace, workspace_bytes,
                                        stream);
}

KO_EXPORT int ko_policy_loss_16(const void *logits, int64_t ld, const int32_t *labels, const float *old_logp,
                                const float *ref_logp, const float *advantage, const float *weight, float scale, float clip_low,
                                float clip_high, float kl_coef, float *logp, float *kl, float *loss, float *loss_sum,
                                void *dlogits, int64_t ldd, int64_t rows, int64_t cols, int dtype, void *workspace,
                                size_t workspace_bytes, ko_stream_t stream) {
    if (dtype == KO_F16)
        return ko::policy_entry<ko::IO_F16>(logits, ld, labels, old_logp, ref_logp, advantage, weight, scale, clip_low, clip_high,
                                            kl_coef, logp, kl, loss, loss_sum, dlogits, ldd, rows, cols, workspace,
                                            workspace_bytes, stream);
    if (dtype == KO_BF16)
        return ko::policy_entry<ko::IO_BF16>(logits, ld, labels, old_logp, ref_logp, advantage, weight, scale, clip_low, clip_high,
                                             kl_coef, logp, kl, loss, loss_sum, dlogits, ldd, rows, cols, workspace,
                                             workspace_bytes, stream);
    return ko::fail(KO_ERR_INVALID_ARGUMENT, "policy_loss: dtype=%d is neither KO_F16 nor KO_BF16", dtype);
}

KO_EXPORT int ko_preference_loss_f32(const float *logp, const float *ref_logp, const int32_t *labels, const int32_t *offsets,
                                     int64_t pairs, int64_t tokens, float beta, float label_smoothing, float pair_weight,
                                     float *pair_loss, float *rewards, float *dlogp, float *loss_sum, ko_stream_t stream) {
    static const char *const who = "preference_loss";
    if (pairs < 0 || tokens < 0 || tokens > 0x7fffffff)
        return ko::fail(KO_ERR_INVALID_ARGUMENT, "%s: pairs=%lld tokens=%lld", who, (long long)pairs, (long long)tokens);
    if (!(beta > -INFINITY && beta < INFINITY) || !(pair_weight > -INFINITY && pair_weight < INFINITY))
        return ko::fail(KO_ERR_INVALID_ARGUMENT, "%s: beta=%g pair_weight=%g", who, static_cast<double>(beta), static_cast<double>(pair_weight));
    if (!(label_smoothing >= 0.0f && label_smoothing <= 1.0f))
        return ko::fail(KO_ERR_INVALID_ARGUMENT, "%s: label_smoothing=%g", who, static_cast<double>(label_smoothing));
    if (const int st = ko::check_floats(who, {logp, ref_logp, labels, offsets, pair_loss, rewards, dlogp, loss_sum}); st != KO_OK)
        return st;
    const hipStream_t s = ko::as_stream(stream);
    if (pairs == 0) return loss_sum ? ko::launch_loss_sum(nullptr, 0, pair_weight, loss_sum, s) : KO_OK;
    if (!offsets || !pair_loss || (tokens > 0 && (!logp || !ref_logp)))
        return ko::fail(KO_ERR_INVALID_ARGUMENT, "%s: null logp/ref_logp/offsets/pair_loss pointer", who);
    const ko::PreferenceArgs a{logp, ref_logp, labels, offsets, pairs, tokens, beta, label_smoothing, pair_weight, pair_loss,
                               rewards, dlogp};
    if (pairs <= ko::kFewPairs && tokens <= ko::kFewTokens) {
        if (pairs <= 2) ko::preference_few_kernel<2><<<dim3(1), dim3(1024), 0, s>>>(a, loss_sum);
        else if (pairs <= 4) ko::preference_few_kernel<4><<<dim3(1), dim3(1024), 0, s>>>(a, loss_sum);
        else ko::preference_few_kernel<16><<<dim3(1), dim3(1024), 0, s>>>(a, loss_sum);
        KO_CHECK_LAUNCH();
        return KO_OK;
    }
    if (dlogp && pairs > ko::kManyPairs) {
        ko::preference_offsets_kernel<<<dim3(1), dim3(1024), 0, s>>>(offsets, pairs, reinterpret_cast<int32_t *>(pair_loss));
        KO_CHECK_LAUNCH();
    }
    ko::preference_kernel<<<ko::row_grid(pairs, ko::kPreferenceThreads), dim3(ko::kPreferenceThreads), 0, s>>>(a);
    KO_CHECK_LAUNCH();
    return loss_sum ? ko::launch_loss_sum(pair_loss, pairs, pair_weight, loss_sum, s) : KO_OK;
}
