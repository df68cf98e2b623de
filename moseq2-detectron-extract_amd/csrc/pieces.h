// Rows of any length and alignment in pieces of 16 bytes (linear.hip, norm.hip).
#pragma once
#include "common.h"

namespace mdx {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// rows start at any element: vector accesses of the element's alignment
// (global_load_dwordx4 takes any address in the unaligned access mode of HSA)
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Un16 { u4 v; };

template <typename T> constexpr int VEC = 16 / (int)sizeof(T);

// 16 bytes shifted down by s bits, 0 <= s < 128
__device__ __forceinline__ u4 shift_down(u4 v, int s) {
    union { u4 u; unsigned long long d[2]; } r;
    r.u = v;
    if (s >= 64) {
        r.d[0] = r.d[1];
        r.d[1] = 0;
        s -= 64;
    }
    if (s) {
        r.d[0] = r.d[0] >> s | r.d[1] << (64 - s);
        r.d[1] >>= s;
    }
    return r.u;
}
// 16 bytes of a row from its element c on, of which the first n exist (n <= 0:
// none); the rest is zero.  The last piece of a row is read as the 16 bytes
// that end with it, shifted down.
template <typename T> __device__ __forceinline__ u4 load_piece(const T *p, int c, int n) {
    constexpr int N = VEC<T>;
    if (n >= N) return reinterpret_cast<const Un16<T> *>(p)->v;
    if (n <= 0) return u4{0, 0, 0, 0};
    if (c + n >= N)
        return shift_down(reinterpret_cast<const Un16<T> *>(p - (N - n))->v, (N - n) * 8 * (int)sizeof(T));
    union { u4 u; T e[N]; } r;
    r.u = u4{0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < N; ++q)
        if (q < n) r.e[q] = p[q];
    return r.u;
}

}  // namespace mdx
