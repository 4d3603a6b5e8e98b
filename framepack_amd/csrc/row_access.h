// Rows of any alignment and length, 8 elements (16 bytes) a lane: K12 and K13's kernels that read their operands directly.
#pragma once
#include "fp_common.h"

// 8 elements of a row from column c on, zeros behind its end.  The wide access needs no more than the type's alignment
// (unaligned accesses are on for global memory on this target), so rows of any stride and length take it.  A row's partial
// last chunk is read as its last 8 elements and moved into place by `fit` where it is used, so that the load itself is one
// instruction that nothing waits for (as seven conditional loads it cost a row of 4095 columns a third of its time).
// The elements in front of the chunk's own may be written by another lane meanwhile where an output lies on the row: a chunk is not
// used before `fit` has dropped them.
template <typename T> struct vec8;
template <> struct vec8<bf16> { typedef bf16x8 type; };
template <> struct vec8<_Float16> { typedef _Float16 type __attribute__((ext_vector_type(8))); };
template <typename T> struct any8 { typedef typename vec8<T>::type type __attribute__((aligned(2))); };
template <typename T>
__device__ __forceinline__ typename vec8<T>::type load8(const T* row, int c, int cols) {
    typename vec8<T>::type v = {};
    if (cols >= 8) {                                        // (uniform)
        if (c < cols) v = *reinterpret_cast<const typename any8<T>::type*>(row + min(c, cols - 8));
    } else {
#pragma unroll
        for (int j = 0; j < 7; ++j)
            if (c + j < cols) v[j] = row[c + j];
    }
    return v;
}
template <typename V> __device__ __forceinline__ void fit(V& v, int c, int cols) {
    if ((cols & 7) == 0 || cols < 8) return;                // (uniform, as is all but the last line)
    const int s = 8 - (cols & 7);                           // elements in front of the chunk's
    u32x4 d = __builtin_bit_cast(u32x4, v);
    if (s & 1) d = u32x4{__builtin_amdgcn_alignbit(d[1], d[0], 16), __builtin_amdgcn_alignbit(d[2], d[1], 16),
                         __builtin_amdgcn_alignbit(d[3], d[2], 16), d[3] >> 16};
    if (s & 2) d = u32x4{d[1], d[2], d[3], 0u};
    if (s & 4) d = u32x4{d[2], d[3], 0u, 0u};
    if (c < cols && c + 8 > cols) v = __builtin_bit_cast(V, d);
}
template <typename T>
__device__ __forceinline__ void store8(T* row, int c, int cols, const typename vec8<T>::type& v) {
    typedef T A4 __attribute__((ext_vector_type(4), aligned(2)));
    typedef T A2 __attribute__((ext_vector_type(2), aligned(2)));
    if (c + 8 <= cols) {
        *reinterpret_cast<typename any8<T>::type*>(row + c) = v;
    } else if (c < cols) {
        const int n = cols & 7;
        if (n & 4) *reinterpret_cast<A4*>(row + c) = A4{v[0], v[1], v[2], v[3]};
        if (n & 2) *reinterpret_cast<A2*>(row + c + (n & 4)) = n & 4 ? A2{v[4], v[5]} : A2{v[0], v[1]};
        if (n & 1) row[c + n - 1] = n & 4 ? (n & 2 ? v[6] : v[4]) : (n & 2 ? v[2] : v[0]);
    }
}
