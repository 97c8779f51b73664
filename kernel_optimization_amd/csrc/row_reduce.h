// What the backward and loss kernels share beside wave64.h: workgroup-wide reductions and addresses.
#pragma once

#include <type_traits>

#include "ko_internal.h"
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

// ---- vectors of rows that start anywhere
// A row whose length is no whole number of 16-byte vectors, or a tensor that does not start on a 16-byte boundary, puts
// rows at any element's address.  Such RAGGED rows are still walked vector by vector, from their first column on: the
// hardware takes 16-byte accesses at any address (the compiler issues them for under-aligned types), at a fraction of
// the cost of one access per element; only the row's last vector, where it is not whole, goes element by element.
template <int IO>
struct Unaligned {
    typedef typename Io<IO>::raw type __attribute__((aligned(sizeof(typename Io<IO>::elem))));
};

// Vectors of a row.
template <int IO, bool RAGGED>
__device__ __forceinline__ int row_vectors(int cols) {
    return RAGGED ? (cols + Io<IO>::E - 1) / Io<IO>::E : cols / Io<IO>::E;
}

// Vector j (of those that row_vectors counts) of the row at `uniform_base + offset` bytes; what lies past the row's end
// is 0.
template <int IO, bool RAGGED, bool NT>
__device__ __forceinline__ typename Io<IO>::raw load_row_vec(const typename Io<IO>::elem *base, uint32_t offset, int j, int cols) {
    constexpr int E = Io<IO>::E;
    typedef typename Io<IO>::raw Raw;
    const typename Io<IO>::elem *p = byte_offset(base, offset + Io<IO>::kBytes * static_cast<uint32_t>(j));
    if constexpr (!RAGGED) {
        return Io<IO>::template load_raw<NT>(p);
    } else {
        if (E * (j + 1) <= cols) {
            typedef typename Unaligned<IO>::type Any;
            if constexpr (NT) return __builtin_nontemporal_load(reinterpret_cast<const Any *>(p));
            return *reinterpret_cast<const Any *>(p);
        }
        Raw r{};
        const int n = cols - E * j;
#pragma unroll
        for (int e = 0; e < E - 1; ++e) {
            if constexpr (E == 4) {
                if (e < n) r[e] = p[e];
            } else {
                if (e < n) r[e / 2] |= static_cast<uint32_t>(p[e]) << (16 * (e & 1));
            }
        }
        return r;
    }
}

// The values of one vector, rounded to the storage type.
template <int IO>
__device__ __forceinline__ typename Io<IO>::raw pack(const float (&v)[Io<IO>::E]) {
    constexpr int E = Io<IO>::E;
    if constexpr (IO == IO_F32) {
        return float4v{v[0], v[1], v[2], v[3]};
    } else if constexpr (IO == IO_F16) {
        typename Io<IO>::half8 h;
#pragma unroll
        for (int e = 0; e < E; ++e) h[e] = static_cast<_Float16>(v[e]);
        return __builtin_bit_cast(uint4v, h);
    } else {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        typedef float float2v __attribute__((ext_vector_type(2)));
        uint4v x;
#pragma unroll
        for (int e = 0; e < E / 2; ++e)
            x[e] = __builtin_bit_cast(uint32_t, __builtin_convertvector(float2v{v[2 * e], v[2 * e + 1]}, bf16x2));
        return x;
    }
}

// Vector j of an output row, counterpart of load_row_vec: whole lines by store_row_vec.
template <int IO, bool RAGGED>
__device__ __forceinline__ void store_row_vec_any(bool whole_lines, typename Io<IO>::elem *base, uint32_t offset, int j, int cols,
                                                  const float (&v)[Io<IO>::E]) {
    constexpr int E = Io<IO>::E;
    const uint32_t at = offset + Io<IO>::kBytes * static_cast<uint32_t>(j);
    if constexpr (!RAGGED) {
        store_row_vec<IO>(whole_lines, base, at, v);
    } else {
        const typename Io<IO>::raw r = pack<IO>(v);
        typename Io<IO>::elem *p = byte_offset(base, at);
        if (E * (j + 1) <= cols) {
            __builtin_nontemporal_store(r, reinterpret_cast<typename Unaligned<IO>::type *>(p));
            return;
        }
        const int n = cols - E * j;
#pragma unroll
        for (int e = 0; e < E - 1; ++e) {
            if constexpr (E == 4) {
                if (e < n) p[e] = r[e];
            } else {
                if (e < n) p[e] = static_cast<uint16_t>(r[e / 2] >> (16 * (e & 1)));
            }
        }
    }
}

// Whole vectors for kernels that keep loads of later rows in flight: no access is made under a condition, since past a
// branch the compiler no longer knows how many accesses are on their way and waits for all of them.
// FULL: rows of whole vectors on 16-byte boundaries; else at any address (`offset` in bytes, a multiple of the element).
template <int IO, bool FULL>
__device__ __forceinline__ typename Io<IO>::raw load_whole(const typename Io<IO>::elem *base, uint32_t offset) {
    if constexpr (FULL) return Io<IO>::template load_raw<true>(byte_offset(base, offset));
    else return __builtin_nontemporal_load(reinterpret_cast<const typename Unaligned<IO>::type *>(byte_offset(base, offset)));
}
template <int IO, bool FULL>
__device__ __forceinline__ void store_whole(typename Io<IO>::elem *base, uint32_t offset, const float (&v)[Io<IO>::E]) {
    const typename Io<IO>::raw r = pack<IO>(v);
    if constexpr (FULL) {
        // written through at once like stream_store16, but by a builtin, which the compiler counts
        constexpr int kNt = 2, kSc1 = 16;      // cache policy bits
        constexpr int kRaw32Bit = 0x00027000;  // resource word 3: raw buffer, 32-bit data
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uint4v, r),
                                               __builtin_amdgcn_make_buffer_rsrc(base, 0, -1, kRaw32Bit), offset, 0, kNt | kSc1);
    } else {
        __builtin_nontemporal_store(r, reinterpret_cast<typename Unaligned<IO>::type *>(byte_offset(base, offset)));
    }
}

// Buffer accesses of 16 bytes at base + offset, dropped (loads: zeros, nothing is fetched) where offset + 16 passes `bytes`:
// what takes the place of a condition in such kernels.  `base` and `bytes` are the same in every lane.
typedef __amdgpu_buffer_rsrc_t Buffer;
__device__ __forceinline__ Buffer buffer_of(const void *base, uint32_t bytes) {
    constexpr int kRaw32Bit = 0x00027000;  // resource word 3: raw buffer, 32-bit data
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, bytes, kRaw32Bit);
}
template <int IO>
__device__ __forceinline__ typename Io<IO>::raw buffer_load(Buffer b, uint32_t offset) {
    return __builtin_bit_cast(typename Io<IO>::raw, __builtin_amdgcn_raw_buffer_load_b128(b, offset, 0, 2 /* nt */));
}
// For vectors that make whole 64-byte lines, written through at once (see store_row_vec).
template <int IO>
__device__ __forceinline__ void buffer_store(Buffer b, uint32_t offset, const float (&v)[Io<IO>::E]) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(uint4v, pack<IO>(v)), b, offset, 0, 2 | 16 /* nt sc1 */);
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

// Longest row of the kernels that count its bytes in 32 bits.
constexpr int64_t kMaxColumns = 1 << 28;

// One workgroup per row (or group of rows), as far as a grid goes: its threads number less than 2^32, and the kernels walk on
// from there.  (The knob is for tests of the walk, which otherwise begins with millions of rows.)
inline dim3 row_grid(int64_t groups, int threads) {
    const int knob = tuning(knob_rows_most_workgroups);
    const int64_t most = knob > 0 ? knob : 0xffffffffll / threads;
    return dim3(static_cast<unsigned>(groups < most ? groups : most));
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
