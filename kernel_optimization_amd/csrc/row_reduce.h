// What the backward and loss kernels share beside wave64.h: workgroup-wide reductions and addresses.
#pragma once

#include <type_traits>

#include "wave64.h"

namespace ko {

// base + bytes, for addresses formed from a uniform pointer and a 32-bit per-lane offset
template <class T>
__device__ __forceinline__ T *byte_offset(T *base, uint32_t bytes) {
    typedef typename std::conditional<std::is_const<T>::value, const char, char>::type Byte;
    return reinterpret_cast<T *>(reinterpret_cast<Byte *>(base) + bytes);
}

// Makes the compiler take a loaded vector as new: what was converted from it before is converted again where it is
// needed, instead of being kept (16-bit storage: twice the registers of the vector itself).
template <int IO>
__device__ __forceinline__ void convert_again(typename Io<IO>::raw &r) {
    if constexpr (Io<IO>::E > 1) asm volatile("" : "+v"(r));
}

// Sum over a workgroup of WAVES wavefronts of N values at once: wave all-reduces, then every thread folds the
// per-wave partials in wave order (the same bits in every thread).  One barrier: `slot` is not written again before
// every wave has passed the workgroup's next barrier (callers alternate between two slots).
template <int WAVES, int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float (*slot)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = wave::allreduce<64, wave::Sum>(v[i]);
    if constexpr (WAVES == 1) return;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) slot[threadIdx.x >> 6][i] = v[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float r = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) r += slot[w][i];
        v[i] = r;
    }
}

// Lanes per row and vectors per lane for rows of `nvec` vectors held by groups of 8 to 64 lanes: the fewest idle
// vector slots, among equals the widest group (one load instruction then covers the longest piece of a row).
// `max_vpl` bounds the vectors per lane for 64 lanes; narrower groups take at most 3.
inline bool choose_row_group(int nvec, int max_vpl, int *lanes, int *vectors) {
    int best = -1;
    for (int lpr = 8; lpr <= 64; lpr <<= 1) {
        const int vpl = (nvec + lpr - 1) / lpr;
        if (vpl > (lpr < 64 ? 3 : max_vpl)) continue;
        const int waste = lpr * vpl - nvec;
        if (best < 0 || waste <= best) {
            best = waste;
            *lanes = lpr;
            *vectors = vpl;
        }
    }
    return best >= 0;
}

}  // namespace ko
