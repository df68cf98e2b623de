// Linear layers of the detector's heads, forward and backward, dense and
// grouped by expert (include/mdx.h: mdx_linear*, mdx_grouped_linear*).
//
//   forward   z = x W^T + b (+ r),  y = act(z)
//   backward  dz = dy act'(z),  dr = dz,  db = sum_m dz,  dx = dz W,  dW = dz^T x
//
// Every product is out[i][j] = sum_r A(i,r) B(j,r) with each operand stored
// either with r contiguous (TA / TB = 0) or with i / j contiguous (1):
//   forward  i = row, j = n, r = k   x 0, W 0
//   dx       i = row, j = k, r = n   dz 0, W 1
//   dW       i = n,   j = k, r = row dz 1, x 1
// so no operand is ever transposed in memory.
#include "common.h"

#include <algorithm>
#include <type_traits>

namespace mdx {
namespace lin {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 *lds_s4;

// rows start at any element: vector accesses of the element's alignment
// (global_load_dwordx4 takes any address in the unaligned access mode of HSA)
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Un16 { u4 v; };
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Un4 { T v[4]; };

template <typename T> constexpr int VEC = 16 / (int)sizeof(T);

// 16 bytes of a row, of which the first n elements exist (n <= 0: none)
template <typename T> __device__ __forceinline__ u4 load_piece(const T *p, long long n) {
    if (n >= VEC<T>) return reinterpret_cast<const Un16<T> *>(p)->v;
    union { u4 u; T e[VEC<T>]; } r;
    r.u = u4{0, 0, 0, 0};
#pragma unroll
    for (int q = 0; q < VEC<T>; ++q)
        if (q < n) r.e[q] = p[q];
    return r.u;
}
template <typename T> __device__ __forceinline__ f4 load4(const T *p, int n) {
    if (n >= 4) {
        const Un4<T> v = *reinterpret_cast<const Un4<T> *>(p);
        return f4{(float)v.v[0], (float)v.v[1], (float)v.v[2], (float)v.v[3]};
    }
    f4 r{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 3; ++q)
        if (q < n) r[q] = (float)p[q];
    return r;
}
// one rounding to the output's type
template <typename T> __device__ __forceinline__ void store4(T *p, f4 v, int n) {
    if (n >= 4) {
        Un4<T> o;
#pragma unroll
        for (int q = 0; q < 4; ++q) o.v[q] = (T)v[q];
        *reinterpret_cast<Un4<T> *>(p) = o;
        return;
    }
#pragma unroll
    for (int q = 0; q < 3; ++q)
        if (q < n) p[q] = (T)v[q];
}

// ---- activations, in float32 ------------------------------------------------
// On the hardware's exp2 and reciprocal (1 ulp each): with the library's erff,
// tanhf and division the epilogue of a 256 x 256 tile took longer than its
// product of 1024 terms.
__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }
// 1 / (1 + exp(-u))
__device__ __forceinline__ float logistic(float u) { return __builtin_amdgcn_rcpf(1.f + fast_exp(-u)); }
// the normal distribution at z: *p its probability (1 + erf(z / sqrt 2)) / 2 by
// formula 7.1.26 of Abramowitz and Stegun (erf to 1.5e-7), returned
// exp(-z^2 / 2), which that formula needs and the density is made of
__device__ __forceinline__ float normal_cdf(float z, float *p) {
    const float x = fabsf(z) * 0.70710678118654752f, t = __builtin_amdgcn_rcpf(1.f + 0.3275911f * x);
    const float e = fast_exp(-x * x);
    const float c =
        0.5f * e * t *
        (0.254829592f + t * (-0.284496736f + t * (1.421413741f + t * (-1.453152027f + t * 1.061405429f))));
    *p = z < 0.f ? c : 1.f - c;
    return e;
}
// the tanh form: (1 + tanh v) / 2 = logistic(2 v), 2 v = C (z + A z^3)
constexpr float TANH_C = 1.59576912160573071f, TANH_A = 0.044715f;

__device__ __forceinline__ float act_value(float z, int act) {
    switch (act) {
        case MDX_ACT_RELU: return z < 0.f ? 0.f : z;  // NaN stays NaN
        case MDX_ACT_GELU: {
            float p;
            normal_cdf(z, &p);
            return z * p;
        }
        case MDX_ACT_GELU_TANH: return z * logistic(TANH_C * (z + TANH_A * z * z * z));
        case MDX_ACT_SILU: return z * logistic(z);
        default: return z;
    }
}
__device__ __forceinline__ float act_slope(float z, int act) {
    switch (act) {
        case MDX_ACT_GELU: {
            float p;
            const float e = normal_cdf(z, &p);
            return p + z * e * 0.39894228040143268f;
        }
        case MDX_ACT_GELU_TANH: {
            const float s = logistic(TANH_C * (z + TANH_A * z * z * z));
            return s + z * s * (1.f - s) * TANH_C * (1.f + 3.f * TANH_A * z * z);
        }
        case MDX_ACT_SILU: {
            const float s = logistic(z);
            return s * (1.f + z * (1.f - s));
        }
        default: return 1.f;
    }
}
// dy act'(z); ReLU selects, so that an infinite gradient of a closed unit is dropped
__device__ __forceinline__ float act_grad(float dy, float z, int act) {
    if (act == MDX_ACT_RELU) return z > 0.f ? dy : 0.f;
    return dy * act_slope(z, act);
}

// ---- one product --------------------------------------------------------
struct Args {
    const void *a, *b;
    long long lda, ldb;  // elements between stored rows
    long long I, R;      // output rows, reduction length (of all groups together when grouped)
    int J;
    const float *bias;   // [J] or null
    const void *res;     // (I, J) or null
    long long ldr;
    void *pre;           // act's argument, or null
    long long ldp;
    void *out;
    long long ldo;
    int act;
    // groups: counts[E] rows each, back to back, at most T in all; a negative
    // count is none and what passes T is cut off, so no count leads outside
    const int *counts;
    int E;
    long long T;
    long long gstride;   // elements between the groups of b (grouped rows) or of out (grouped reduction)
    int zero_tail;       // grouped rows: write zeros in the rows behind the last group
    float *part;         // partial sums [splits][groups][I][J], or null
    int splits;
    int ti, tj;          // output tiles (grouped rows: a bound on them)
};

enum { DENSE = 0, GROUP_ROWS = 1, GROUP_RED = 2 };

struct Span {
    int e;                 // group, E = the rows behind the last one, -1 = none
    long long start, end;  // its rows
    long long tile;        // tile within the group
};

// The group holding output tile `tile` when each group's rows are cut into
// tiles of bm (want < 0), or group `want` itself.  Every wave scans the counts 64 at a
// time with its lanes, so no pass over the counts has to run before.
__device__ __forceinline__ Span find_group(const int *counts, int E, long long T, int bm, long long tile, int want) {
    const int lane = threadIdx.x & 63;
    long long row0 = 0, tile0 = 0;
    for (int base = 0; base < E; base += 64) {
        long long c = base + lane < E ? max(counts[base + lane], 0) : 0;
        long long rows = c;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const long long v = __shfl_up(rows, d);
            if (lane >= d) rows += v;
        }
        const long long s = min(row0 + rows - c, T), e = min(row0 + rows, T);
        const long long mine = want >= 0 ? 0 : (e - s + bm - 1) / bm;
        long long tiles = mine;
        if (want < 0) {
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const long long v = __shfl_up(tiles, d);
                if (lane >= d) tiles += v;
            }
        }
        const long long t1 = tile0 + tiles, t0 = t1 - mine;
        const unsigned long long hit =
            __ballot(base + lane < E && (want >= 0 ? base + lane == want : tile >= t0 && tile < t1));
        if (hit) {
            const int l = __ffsll(hit) - 1;
            return Span{base + l, __shfl(s, l), __shfl(e, l), tile - __shfl(t0, l)};
        }
        row0 = min(row0 + __shfl(rows, 63), T);
        tile0 = __shfl(t1, 63);
    }
    if (want >= 0 ? want == E : row0 < T && tile < tile0 + (T - row0 + bm - 1) / bm)
        return Span{E, row0, T, tile - tile0};
    return Span{-1, 0, 0, 0};
}

// workgroup -> tile: contiguous ranges of tiles for each of the 8 XCDs (their
// L2s are separate), and in a range squares of 8 row tiles, column by column
__device__ __forceinline__ void map_tile(long long id, int ti, int tj, long long &t, int &u) {
    const long long n = (long long)ti * tj, q = n / 8, r = n % 8, x = id % 8;
    id = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + id / 8;
    const long long per = 8ll * tj, g = id / per, in = id - g * per;
    const int rows = (int)min(8ll, ti - 8 * g);
    t = 8 * g + in % rows;
    u = (int)(in / rows);
}

// N neighbouring values of a row as floats, of which n exist
template <typename T, int N> __device__ __forceinline__ void load_row(const T *p, int n, float (&v)[N]) {
    struct __attribute__((packed, aligned(sizeof(T)))) U { T e[N]; };
    if (n >= N) {
        const U u = *reinterpret_cast<const U *>(p);
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = (float)u.e[q];
        return;
    }
#pragma unroll
    for (int q = 0; q < N; ++q) v[q] = q < n ? (float)p[q] : 0.f;
}
template <typename T, int N> __device__ __forceinline__ void store_row(T *p, int n, const float (&v)[N]) {
    struct __attribute__((packed, aligned(sizeof(T)))) U { T e[N]; };
    if (n >= N) {
        U u;
#pragma unroll
        for (int q = 0; q < N; ++q) u.e[q] = (T)v[q];  // the one rounding to the output's type
        *reinterpret_cast<U *>(p) = u;
        return;
    }
#pragma unroll
    for (int q = 0; q < N; ++q)
        if (q < n) p[q] = (T)v[q];
}
// bias, residual, activation and the stores of 16 bytes of a row of outputs
template <typename T>
__device__ __forceinline__ void finish(const Args &g, const float *bias, long long i, int j, float (&v)[VEC<T>]) {
    constexpr int N = VEC<T>;
    const int n = g.J - j;
    float w[N];
    if (bias) {
        load_row<float, N>(bias + j, n, w);
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] += w[q];
    }
    if (g.res) {
        load_row<T, N>(reinterpret_cast<const T *>(g.res) + i * g.ldr + j, n, w);
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] += w[q];
    }
    if (g.pre) store_row<T, N>(reinterpret_cast<T *>(g.pre) + i * g.ldp + j, n, v);
    if (g.act != MDX_ACT_NONE)
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] = act_value(v[q], g.act);
    store_row<T, N>(reinterpret_cast<T *>(g.out) + i * g.ldo + j, n, v);
}

// A wave's 64 x 64 block of sums, acc(i, j) the 16 x 16 tile of rows 16 i,
// columns 16 j (lane: row l & 15, columns 4 (l >> 4)..), 32 rows at a time
// through the wave's own 8.5 KiB of LDS, so that a lane finishes 16 bytes of a
// row and a row's lanes store a whole line.  The block goes to a slice's
// partial sums, to zeros (behind the last group) or to the finished outputs.
constexpr int EPI_PITCH = 68, EPI_BYTES = 32 * EPI_PITCH * 4;
template <typename T, int MODE, typename F>
__device__ __forceinline__ void epilogue(const Args &g, const float *bias, bool tail, char *lds, long long row0,
                                         long long row1, int col0, F acc) {
    constexpr int N = VEC<T>, PER = 64 / N;  // lanes to a row
    const int lane = threadIdx.x & 63;
    float *e = reinterpret_cast<float *>(lds);
    const long long grp = MODE == GROUP_RED ? blockIdx.z * (long long)g.E + blockIdx.y : blockIdx.z;
#pragma unroll
    for (int p = 0; p < 2; ++p) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<f4 *>(e + (16 * i + (lane & 15)) * EPI_PITCH + 16 * j + 4 * (lane >> 4)) =
                    acc(2 * p + i, j);
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll 1
        for (int k = 0; k < 32 * PER / 64; ++k) {
            const int r = (64 * k + lane) / PER, c = (64 * k + lane) % PER * N;
            const long long row = row0 + 32 * p + r;
            const int col = col0 + c, n = g.J - col;
            if (row >= row1 || n <= 0) continue;
            float v[N];
#pragma unroll
            for (int q = 0; q < N / 4; ++q)
                *reinterpret_cast<f4 *>(v + 4 * q) = *reinterpret_cast<const f4 *>(e + r * EPI_PITCH + c + 4 * q);
            if (g.splits > 1) {
                store_row<float, N>(g.part + (grp * g.I + row) * g.J + col, n, v);
            } else if (tail) {
                store_row<T, N>(reinterpret_cast<T *>(g.out) + row * g.ldo + col, n, v);
                if (g.pre) store_row<T, N>(reinterpret_cast<T *>(g.pre) + row * g.ldp + col, n, v);
            } else {
                finish<T>(g, bias, row, col, v);
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    }
}

template <typename T> struct Mma;
template <> struct Mma<__bf16> {
    static __device__ __forceinline__ f4 mul(u4 x, u4 y, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), c, 0, 0, 0);
    }
};
template <> struct Mma<_Float16> {
    static __device__ __forceinline__ f4 mul(u4 x, u4 y, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, y), c, 0, 0, 0);
    }
};
template <> struct Mma<float> {
    // element e of lane (row, q) is r = 4 q + e in both operands: any order of
    // the products gives the same sum
    static __device__ __forceinline__ f4 mul(u4 x, u4 y, f4 c) {
        const f4 a = __builtin_bit_cast(f4, x), b = __builtin_bit_cast(f4, y);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
};

// 128 rows (i) of an operand by 128 bytes of reduction, staged in LDS.
// TR = 0: [128][128 B], 16-B pieces XOR-swizzled by row; a fragment (row
// l & 15, piece 4 s + (l >> 4)) is one b128 read.
// TR = 1: [128 B / sizeof(T)][128]; 16-bit fragments are two transposing
// 64-bit reads (16 lanes give the addresses of a 4 x 16 block, lane i gets
// its column i), 32-bit ones four b32 reads.  The swizzle spreads the rows
// that one read takes over all banks.
template <typename T, bool TR> struct Stage {
    static constexpr int BK = 128 / (int)sizeof(T);
    static constexpr int BYTES = 128 * 128;
    static constexpr int PITCH = TR ? 128 * (int)sizeof(T) : 128;
    static constexpr int PPR = PITCH / 16;           // pieces per stored row
    static constexpr int STEP = 256 / PPR;           // rows between a thread's four pieces

    static __device__ __forceinline__ int swz(int row) {
        if (!TR) return (row >> 1) & 7;
        if (sizeof(T) == 2) return ((row & 3) | (((row >> 3) & 1) << 2)) << 1;
        return ((row >> 2) & 3) << 2;
    }
    // the thread's four pieces of the tile whose first i is i0 and first r is r0
    static __device__ __forceinline__ void load(const T *p, long long ld, long long i0, long long I, long long r0,
                                                long long R, u4 (&v)[4]) {
        const int pc = threadIdx.x % PPR, row = threadIdx.x / PPR;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const long long w = (TR ? r0 : i0) + row + STEP * q, c = (TR ? i0 : r0) + pc * VEC<T>;
            const long long left = w < (TR ? R : I) ? (TR ? I : R) - c : 0;
            v[q] = load_piece(left > 0 ? p + w * ld + c : p, left);
        }
    }
    static __device__ __forceinline__ void write(char *lds, const u4 (&v)[4]) {
        const int pc = threadIdx.x % PPR, row = threadIdx.x / PPR;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int r = row + STEP * q;
            *reinterpret_cast<u4 *>(lds + r * PITCH + ((pc ^ swz(r)) << 4)) = v[q];
        }
    }
    // fragment of rows i0 .. i0 + 15, 64-B step s
    static __device__ __forceinline__ u4 frag(const char *lds, int i0, int s) {
        const int lane = threadIdx.x & 63, f = lane & 15, q = lane >> 4;
        if constexpr (!TR) {
            const int r = i0 + f;
            return *reinterpret_cast<const u4 *>(lds + r * 128 + (((4 * s + q) ^ swz(r)) << 4));
        } else if constexpr (sizeof(T) == 2) {
            const int k = 32 * s + 8 * q + (f >> 2), c = i0 + 4 * (f & 3);
            const char *p = lds + k * PITCH + (((c >> 3) ^ swz(k)) << 4) + (c & 7) * 2;
            union { s4 h[2]; u4 u; } r;
            r.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)p);
            r.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + 4 * PITCH));
            return r.u;
        } else {
            const int k = 16 * s + 4 * q, c = i0 + f;
            const char *p = lds + k * PITCH + (((c >> 2) ^ swz(k)) << 4) + (c & 3) * 4;
            u4 r;
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] = *reinterpret_cast<const uint32_t *>(p + e * PITCH);
            return r;
        }
    }
};

// Tile 128 x 128 per workgroup of 4 waves, each 64 x 64 of 16 x 16 MFMA tiles;
// the reduction in steps of 128 bytes through two LDS buffers, the next step's
// global loads in flight in registers meanwhile.  B is the MFMA's first
// operand, so a lane ends with 4 neighbouring columns of one row.
// Any alignment, any sizes.
template <typename T, bool TA, bool TB, int MODE>
__global__ __launch_bounds__(256, 2) void k_product(Args g) {
    using SA = Stage<T, TA>;
    using SB = Stage<T, TB>;
    __shared__ __attribute__((aligned(16))) char lds[2][SA::BYTES + SB::BYTES];
    static_assert(4 * EPI_BYTES <= sizeof(lds), "the epilogue shares the operands' LDS");
    const T *A = reinterpret_cast<const T *>(g.a), *B = reinterpret_cast<const T *>(g.b);
    const float *bias = g.bias;
    long long t;
    int u;
    map_tile(blockIdx.x, g.ti, g.tj, t, u);
    long long i0 = 128 * t, i1 = g.I, r0 = 0, r1 = g.R;
    const int j0 = 128 * u;
    bool tail = false;
    if (MODE == GROUP_ROWS) {
        const Span s = find_group(g.counts, g.E, g.T, 128, t, -1);
        if (s.e < 0 || (s.e == g.E && !g.zero_tail)) return;
        i0 = s.start + 128 * s.tile;
        i1 = s.end;
        if (s.e == g.E) {
            tail = true;
            r1 = 0;
        } else {
            B += s.e * g.gstride;
            if (bias) bias += (long long)s.e * g.J;
        }
    }
    if (MODE == GROUP_RED) {
        const Span s = find_group(g.counts, g.E, g.T, 1, 0, blockIdx.y);
        r0 = s.start;
        r1 = s.end;
    }
    if (g.splits > 1) {  // this slice of the reduction, whole steps
        const long long steps = (r1 - r0 + SA::BK - 1) / SA::BK, per = (steps + g.splits - 1) / g.splits;
        r0 = min(r1, r0 + blockIdx.z * per * SA::BK);
        r1 = min(r1, r0 + per * SA::BK);
    }

    const int wid = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int wi = (wid >> 1) * 64, wj = (wid & 1) * 64;
    f4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};

    u4 va[4], vb[4];
    const long long steps = (r1 - r0 + SA::BK - 1) / SA::BK;
    if (steps > 0) {
        SA::load(A, g.lda, i0, i1, r0, r1, va);
        SB::load(B, g.ldb, j0, g.J, r0, r1, vb);
        SA::write(lds[0], va);
        SB::write(lds[0] + SA::BYTES, vb);
    }
    for (long long s = 0; s < steps; ++s) {
        __syncthreads();
        if (s + 1 < steps) {
            SA::load(A, g.lda, i0, i1, r0 + (s + 1) * SA::BK, r1, va);
            SB::load(B, g.ldb, j0, g.J, r0 + (s + 1) * SA::BK, r1, vb);
        }
        const char *la = lds[s & 1], *lb = la + SA::BYTES;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            u4 fa[4], fb[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) fa[i] = SA::frag(la, wi + 16 * i, h);
#pragma unroll
            for (int j = 0; j < 4; ++j) fb[j] = SB::frag(lb, wj + 16 * j, h);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = Mma<T>::mul(fb[j], fa[i], acc[i][j]);
        }
        if (s + 1 < steps) {
            SA::write(lds[(s + 1) & 1], va);
            SB::write(lds[(s + 1) & 1] + SA::BYTES, vb);
        }
    }

    if (MODE == GROUP_RED) g.out = reinterpret_cast<T *>(g.out) + blockIdx.y * g.gstride;
    __syncthreads();  // the operands' buffers become the epilogue's
    epilogue<T, MODE>(g, bias, tail, lds[0] + wid * EPI_BYTES, i0 + wi, i1, j0 + wj,
                      [&](int i, int j) { return acc[i][j]; });
}

// ---- the large 16-bit tile ----------------------------------------------
// 256 x 256 outputs per workgroup of 8 waves (one workgroup on a CU), the
// reduction in K-tiles of 64 through two LDS buffers filled by LDS-DMA.  A
// K-tile is four half-tiles of 128 rows (B0, A0, B1, A1: 16 KiB each, two
// 1-KiB DMA instructions of every wave) and four phases, one for each
// quarter of the outputs: (A0,B0) (A0,B1) (A1,B1) (A1,B0).  A half of A is
// 128 neighbouring rows, of which wave (g, n) takes rows 64 g..; half h of B is
// columns 64 n + 32 h .. + 31 of each n, so that a wave's 64 columns lie together.
//
// Phase P of a wave is
//   R(P): LDS reads of one half-tile's fragments, DMA of one half-tile,
//         waits, barrier
//   M(P): 16 MFMAs, barrier
// and the waves of g = 1 run one barrier behind those of g = 0, so that on
// every SIMD one wave multiplies while the other reads.  Between barriers 2P
// and 2P + 1 lie R(P) of g = 0 and M(P - 1) of g = 1, then M(P) and R(P).
//
// Half-tiles are numbered 4 t + {B0 0, A0 1, B1 2, A1 3}.  R(P) reads number
// P + 1 (B0 of the next K-tile in the last phase of one: its registers are
// those of B1, free by then) and issues number P + 8, into the buffer place
// of number P, whose last read, R(P - 1), both groups have retired (lgkmcnt 0)
// before the barrier that opens R(P) of g = 0.  Number P + 2, read next, must
// have landed in every wave before that: each wave lets at most 6 half-tiles
// (12 instructions) stay outstanding, so a DMA has six phases, about 3000
// cycles, to arrive, and the queue is never drained before the end.
//
// Rows beyond the operand are clamped to its last (their products only reach
// outputs that are not stored); beyond the reduction's end both operands read
// zeros, and the K-tiles are rounded up to an even number of at least 4; only
// the first two and the last two can be partial.
__device__ __attribute__((aligned(64))) uint4 zero_piece[4];

constexpr int BIG = 256, BIG_BUF = 65536, BIG_LDS = 2 * BIG_BUF, BIG_HALF = 16384;

// Waits and barriers that no memory access is moved across.  The DMA is
// inline asm, so that the compiler, which would wait for all of it before any
// LDS read, leaves the count of outstanding ones to these waits.
template <int VM> __device__ __forceinline__ void big_wait() {  // vmcnt VM, lgkmcnt 0, any expcnt
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((VM & 15) | ((VM >> 4) << 14) | 0x70);
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void big_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}
// a value that is the same in all lanes, in scalar registers
__device__ __forceinline__ long long uniform(long long v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return (long long)((uint64_t)hi << 32 | lo);
}
// 16 bytes a lane from base + off to 1 KiB of LDS at dst (wave-uniform)
__device__ __forceinline__ void dma16(const void *src, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(dst), "v"(src) : "memory");
}
__device__ __forceinline__ void dma16s(const void *base, uint32_t off, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(off), "s"(base)
                 : "memory");
}

// a lane's part in staging and reading one operand
template <typename T, bool TR, bool ISB> struct BigOperand {
    const char *base;    // first piece of K-tile 0
    long long step;      // bytes between K-tiles
    uint32_t off[2][2];  // DMA source of (half, instruction)
    int r[2];            // reduction index of that piece in its K-tile
    __device__ __forceinline__ void init(const void *p, long long ld, long long i0, long long I, long long r0, int wid,
                                         int lane) {
        base = reinterpret_cast<const char *>(
            uniform((long long)(reinterpret_cast<uintptr_t>(p) + (TR ? r0 * ld + i0 : i0 * ld + r0) * 2)));
        step = TR ? 128 * ld : 128;
#pragma unroll
        for (int d = 0; d < 2; ++d) {
            const int row = TR ? 4 * (2 * wid + d) + (lane >> 4) : 8 * (2 * wid + d) + (lane >> 3);
            const int pc = (TR ? lane & 15 : lane & 7) ^ Stage<T, TR>::swz(row);
            r[d] = TR ? row : 8 * pc;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = TR ? 8 * pc : row, k = ISB ? 64 * (at >> 5) + 32 * h + (at & 31) : 128 * h + at;
                const long long i = min(i0 + k, TR ? I - 8 : I - 1);
                off[h][d] = (uint32_t)(TR ? (row * ld + i - i0) * 2 : (i - i0) * ld * 2 + 16 * pc);
            }
        }
    }
    // half-tile H of K-tile t
    template <int H> __device__ __forceinline__ void issue(long long t, uint32_t dst) const {
#pragma unroll
        for (int d = 0; d < 2; ++d) dma16s(base + t * step, off[H][d], dst + 1024 * d);
    }
    // the same where only `left` elements of the reduction are left from its first on
    template <int H> __device__ __forceinline__ void issue_part(long long t, long long left, uint32_t dst) const {
#pragma unroll
        for (int d = 0; d < 2; ++d)
            dma16(r[d] < left ? base + t * step + off[H][d] : reinterpret_cast<const char *>(zero_piece), dst + 1024 * d);
    }
};

template <typename T, bool TA, bool TB, int MODE>
__global__ __launch_bounds__(512, 2) void k_product_big(Args g) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const char *A = reinterpret_cast<const char *>(g.a), *B = reinterpret_cast<const char *>(g.b);
    const float *bias = g.bias;
    long long t;
    int u;
    map_tile(blockIdx.x, g.ti, g.tj, t, u);
    long long i0 = BIG * t, i1 = g.I, r0 = 0, r1 = g.R;
    const int j0 = BIG * u;
    bool tail = false;
    if (MODE == GROUP_ROWS) {
        const Span s = find_group(g.counts, g.E, g.T, BIG, t, -1);
        if (s.e < 0 || (s.e == g.E && !g.zero_tail)) return;
        i0 = s.start + BIG * s.tile;
        i1 = s.end;
        if (s.e == g.E) {
            tail = true;
        } else {
            B += s.e * g.gstride * 2;
            if (bias) bias += (long long)s.e * g.J;
        }
    }
    if (MODE == GROUP_RED) {
        const Span s = find_group(g.counts, g.E, g.T, 1, 0, blockIdx.y);
        r0 = s.start;
        r1 = s.end;
    }
    if (g.splits > 1) {
        const long long steps = (r1 - r0 + 63) / 64, per = (steps + g.splits - 1) / g.splits;
        r0 = min(r1, r0 + blockIdx.z * per * 64);
        r1 = min(r1, r0 + per * 64);
    }
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = wid >> 2, wn = wid & 3, f = lane & 15, q = lane >> 4;

    f4 acc[2][2][4][2];
#pragma unroll
    for (int k = 0; k < 32; ++k) acc[k >> 4][(k >> 3) & 1][(k >> 1) & 3][k & 1] = f4{0.f, 0.f, 0.f, 0.f};

    if (!tail) {
        BigOperand<T, TA, false> oa;
        BigOperand<T, TB, true> ob;
        oa.init(A, g.lda, i0, i1, r0, wid, lane);
        ob.init(B, g.ldb, j0, g.J, r0, wid, lane);
        const long long len = uniform(r1 - r0), KT = max(4ll, (len + 127) / 128 * 2);
        const uint32_t dst = (uint32_t)(uintptr_t)(lds_s4)lds + 2048u * wid;

        // half-tile Q (B0 A0 B1 A1) of K-tile tt into buffer PAR
        auto issue = [&](auto Q, auto Par, auto Part, long long tt) {
            constexpr int n = decltype(Q)::value;
            const uint32_t d = dst + decltype(Par)::value * BIG_BUF + ((n & 1 ? 0 : 2) + (n >> 1)) * BIG_HALF;
            if constexpr (decltype(Part)::value) {
                if constexpr (n & 1)
                    oa.template issue_part<(n >> 1)>(tt, len - 64 * tt, d);
                else
                    ob.template issue_part<(n >> 1)>(tt, len - 64 * tt, d);
            } else {
                if constexpr (n & 1)
                    oa.template issue<(n >> 1)>(tt, d);
                else
                    ob.template issue<(n >> 1)>(tt, d);
            }
        };
        // fragments of half-tile h: A0 A1 B0 B1 lie in this order in a buffer
        u4 fa[2][4], fx[2][2], fy[2][2];
        auto read_a = [&](int h, int par) {
            const char *p = lds + par * BIG_BUF + h * BIG_HALF;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i) fa[s][i] = Stage<T, TA>::frag(p, 64 * grp + 16 * i, s);
        };
        auto read_b = [&](u4 (&fb)[2][2], int h, int par) {
            const char *p = lds + par * BIG_BUF + (2 + h) * BIG_HALF;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int j = 0; j < 2; ++j) fb[s][j] = Stage<T, TB>::frag(p, 32 * wn + 16 * j, s);
        };
        auto mul = [&](f4 (&c)[4][2], const u4 (&fb)[2][2]) {
            big_barrier();
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) c[i][j] = Mma<T>::mul(fb[s][j], fa[s][i], c[i][j]);
            __builtin_amdgcn_s_setprio(0);
            big_barrier();
        };
        using std::integral_constant;
        constexpr integral_constant<int, 0> c0{};
        constexpr integral_constant<int, 1> c1{};
        constexpr integral_constant<int, 2> c2{};
        constexpr integral_constant<int, 3> c3{};
        // one K-tile in buffer PAR; END: 0 and 3 issue K-tile tt + 2 (3: which
        // may be partial), 1 and 2 are the last two
        auto tile = [&](auto End, auto Par, long long tt, u4 (&x)[2][2], u4 (&y)[2][2]) {
            constexpr int END = decltype(End)::value, PAR = decltype(Par)::value;
            constexpr bool MORE = END == 0 || END == 3;
            constexpr integral_constant<int, END == 3> part{};
            read_a(0, PAR);
            if constexpr (MORE) issue(c0, Par, part, tt + 2);
            big_wait<MORE ? 12 : END == 1 ? 10 : 2>();
            mul(acc[0][0], x);
            read_b(y, 1, PAR);
            if constexpr (MORE) issue(c1, Par, part, tt + 2);
            big_wait<MORE ? 12 : END == 1 ? 8 : 0>();
            mul(acc[0][1], y);
            read_a(1, PAR);
            if constexpr (MORE) issue(c2, Par, part, tt + 2);
            big_wait<MORE ? 12 : END == 1 ? 6 : 0>();
            mul(acc[1][1], y);
            if constexpr (END != 2) read_b(y, 0, 1 - PAR);
            if constexpr (MORE) issue(c3, Par, part, tt + 2);
            big_wait<MORE ? 12 : END == 1 ? 4 : 0>();
            mul(acc[1][0], x);
        };
        issue(c0, c0, c1, 0); issue(c1, c0, c1, 0); issue(c2, c0, c1, 0); issue(c3, c0, c1, 0);
        issue(c0, c1, c1, 1); issue(c1, c1, c1, 1); issue(c2, c1, c1, 1); issue(c3, c1, c1, 1);
        big_wait<12>();
        big_barrier();
        read_b(fx, 0, 0);
        big_wait<12>();
        big_barrier();
        if (grp == 1) big_barrier();  // one behind
        for (long long tt = 0; tt < KT - 4; tt += 2) {
            tile(c0, c0, tt, fx, fy);
            tile(c0, c1, tt + 1, fy, fx);
        }
        tile(c3, c0, KT - 4, fx, fy);
        tile(c3, c1, KT - 3, fy, fx);
        tile(c1, c0, KT - 2, fx, fy);
        tile(c2, c1, KT - 1, fy, fx);
        if (grp == 0) big_barrier();  // every wave crosses as many
    }

    if (MODE == GROUP_RED) g.out = reinterpret_cast<T *>(g.out) + blockIdx.y * g.gstride;
    __syncthreads();  // the operands' buffers become the epilogue's
#pragma unroll
    for (int hi = 0; hi < 2; ++hi)
        epilogue<T, MODE>(g, bias, tail, lds + wid * EPI_BYTES, i0 + 128 * hi + 64 * grp, i1, j0 + 64 * wn,
                          [&](int i, int j) { return acc[hi][j >> 1][i][j & 1]; });
}

// The slices' partial sums, added in their order (no atomics: the same result
// on every call), and the epilogue; one thread per 16 bytes of output.
template <typename T>
__global__ __launch_bounds__(256) void k_product_join(Args g) {
    constexpr int N = VEC<T>;
    const long long per = (g.J + N - 1) / N, id = (long long)blockIdx.x * 256 + threadIdx.x;
    if (id >= g.I * per) return;
    const long long row = id / per;
    const int col = (int)(id - row * per) * N;
    const long long E = gridDim.y;
    float v[N] = {}, w[N];
    for (int s = 0; s < g.splits; ++s) {
        load_row<float, N>(g.part + ((s * E + blockIdx.y) * g.I + row) * g.J + col, g.J - col, w);
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] += w[q];
    }
    g.out = reinterpret_cast<T *>(g.out) + blockIdx.y * g.gstride;
    finish<T>(g, g.bias, row, col, v);
}

// dz = dy act'(z) in T, and the column sums of dz before that rounding.  A
// workgroup takes 128 columns (a lane 4, two rows at once per wave) of one
// slice of one group's rows; sums go to part[group][slice][N].
struct ActArgs {
    const void *dy, *z;
    long long ldy, ldz;
    void *dz;            // or null: sums only
    long long lddz;
    float *part;         // or null: dz only
    const int *counts;   // or null: one group of T rows
    int E;
    long long T;
    int N, act;
};
template <typename T>
__global__ __launch_bounds__(256) void k_act_backward(ActArgs g) {
    long long r0 = 0, r1 = g.T;
    const int e = blockIdx.z;
    if (g.counts) {
        const Span s = find_group(g.counts, g.E, g.T, 1, 0, e);
        r0 = s.start;
        r1 = s.end;
    }
    const long long per = (r1 - r0 + gridDim.y - 1) / gridDim.y;
    r0 = min(r1, r0 + blockIdx.y * per);
    r1 = min(r1, r0 + per);
    const int c = blockIdx.x * 128 + (threadIdx.x & 31) * 4, n = g.N - c;
    f4 sum{0.f, 0.f, 0.f, 0.f};
    if (n > 0) {
        for (long long r = r0 + (threadIdx.x >> 5); r < r1; r += 8) {
            f4 v{0.f, 0.f, 0.f, 0.f};
            if (e < g.E) {
                v = load4(reinterpret_cast<const T *>(g.dy) + r * g.ldy + c, n);
                if (g.act != MDX_ACT_NONE) {
                    const f4 z = load4(reinterpret_cast<const T *>(g.z) + r * g.ldz + c, n);
#pragma unroll
                    for (int q = 0; q < 4; ++q) v[q] = act_grad(v[q], z[q], g.act);
                }
            }
            if (g.dz) store4(reinterpret_cast<T *>(g.dz) + r * g.lddz + c, v, n);
            sum += v;
        }
    }
    if (!g.part || e >= g.E) return;
    __shared__ f4 sh[8][32];
    sh[threadIdx.x >> 5][threadIdx.x & 31] = sum;
    __syncthreads();
    if (threadIdx.x < 32 && n > 0) {
#pragma unroll
        for (int w = 1; w < 8; ++w) sum += sh[w][threadIdx.x];
        store4(g.part + ((long long)e * gridDim.y + blockIdx.y) * g.N + c, sum, n);
    }
}
// db[e][n] = the slices' sums in their order
__global__ __launch_bounds__(256) void k_bias_join(const float *part, int slices, int N, float *db) {
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n >= N) return;
    float v = 0.f;
    for (int s = 0; s < slices; ++s) v += part[((long long)blockIdx.y * slices + s) * N + n];
    db[(long long)blockIdx.y * N + n] = v;
}

// ---- host ---------------------------------------------------------------
static long long ceil128(long long n) { return (n + 127) / 128; }

// slices of the reduction: enough workgroups for two on each of the 256 CUs,
// each of at least 4 steps of 128 bytes
static int choose_splits(long long tiles, long long R, int es) {
    const long long steps = (R * es + 127) / 128;
    long long s = std::min<long long>(512 / std::max<long long>(tiles, 1), steps / 4);
    return (int)std::max<long long>(1, std::min<long long>(s, 16));
}
static int fwd_splits(long long M, int N, int K, int dtype) {
    return choose_splits(ceil128(M) * ceil128(N), K, dtype == 0 ? 4 : 2);
}
static int dw_splits(int E, long long T, int N, int K, int dtype) {
    return choose_splits((long long)E * ceil128(N) * ceil128(K), T / std::max(E, 1), dtype == 0 ? 4 : 2);
}
static int act_slices(int E, long long T, int N) {
    const long long want = std::max<long long>(1, 1024 / (ceil128(N) * E));
    return (int)std::max<long long>(1, std::min<long long>(want, (T / std::max(E, 1) + 31) / 32));
}

// the large tile: both operands in whole aligned pieces of 16 bytes, and
// enough tiles
template <typename T, bool TA, bool TB> static bool use_big(const Args &g, int mode) {
    if (sizeof(T) != 2) return false;
    auto piece = [](const void *p, long long ld) {
        return (reinterpret_cast<uintptr_t>(p) | (uintptr_t)(2 * ld)) % 16 == 0 && ld < (1ll << 22);
    };
    if (!piece(g.a, g.lda) || !piece(g.b, g.ldb) || g.gstride % 8) return false;
    if ((TA ? g.I : g.R) % 8 || (TB ? g.J : g.R) % 8) return false;
    const long long groups = mode == GROUP_RED ? g.E : 1;
    return ceil_div(g.I, BIG) * ceil_div(g.J, BIG) * groups * g.splits >= 128;
}

template <typename T, bool TA, bool TB, int MODE> static int launch_product(Args g, hipStream_t s) {
    const bool big = use_big<T, TA, TB>(g, MODE);
    const int side = big ? BIG : 128, threads = big ? 512 : 256;
    const long long bound = MODE == GROUP_ROWS ? g.E + 1 : 0;  // one partial tile more for each group
    const long long ti = ceil_div(g.I, side) + bound, tj = ceil_div(g.J, side);
    MDX_REQUIRE(ti * tj * threads < (1ll << 32), "mdx_linear: too many output tiles");
    g.ti = (int)ti;
    g.tj = (int)tj;
    const dim3 grid((unsigned)(ti * tj), MODE == GROUP_RED ? g.E : 1, g.splits);
    if constexpr (sizeof(T) == 2) {
        if (big) {
            static const hipError_t attr = hipFuncSetAttribute(
                reinterpret_cast<const void *>(k_product_big<T, TA, TB, MODE>),
                hipFuncAttributeMaxDynamicSharedMemorySize, BIG_LDS);
            MDX_HIP(attr);
            hipLaunchKernelGGL((k_product_big<T, TA, TB, MODE>), grid, dim3(512), BIG_LDS, s, g);
        }
    }
    if (!big) hipLaunchKernelGGL((k_product<T, TA, TB, MODE>), grid, dim3(256), 0, s, g);
    MDX_CHECK_LAUNCH("mdx_linear");
    if (g.splits > 1) {
        const dim3 jg((unsigned)ceil_div(g.I * ceil_div(g.J, VEC<T>), 256), MODE == GROUP_RED ? g.E : 1);
        hipLaunchKernelGGL(k_product_join<T>, jg, dim3(256), 0, s, g);
        MDX_CHECK_LAUNCH("mdx_linear");
    }
    return MDX_OK;
}

struct Shape {
    long long T;  // rows
    int E, N, K;  // E = 0: dense
    int dtype, act;
};
static int check_shape(const char *fn, const Shape &p) {
    MDX_REQUIRE(p.dtype == 0 || p.dtype == 1 || p.dtype == 3, "%s: dtype must be 0 (f32), 1 (f16) or 3 (bf16)", fn);
    MDX_REQUIRE(p.act >= MDX_ACT_NONE && p.act <= MDX_ACT_SILU, "%s: unknown activation %d", fn, p.act);
    MDX_REQUIRE(p.T >= 0 && p.T < (1ll << 31) && p.N > 0 && p.K > 0, "%s: bad shape", fn);
    MDX_REQUIRE(p.E >= 0 && p.E <= 4096, "%s: 1 to 4096 groups", fn);
    return MDX_OK;
}
static bool bad_ld(const void *p, long long ld, long long width) { return p && ld < width; }

template <typename T> static int forward(const Shape &p, Args g, hipStream_t s) {
    if (p.E) return launch_product<T, false, false, GROUP_ROWS>(g, s);
    return launch_product<T, false, false, DENSE>(g, s);
}

struct Back {
    const void *grad, *x, *w, *pre;
    long long ldg, ldx, ldw, ldp;
    const int *counts;
    void *dx, *dw, *dres;
    long long lddx, lddw, lddr;
    float *db;
    int zero_tail;
    char *ws;
};
// workspace: dz | sums of db | partial dW, each 256-B aligned
struct BackPlan {
    bool sums, dz;  // the elementwise pass: for its sums, for dz in the workspace
    int slices, splits;
    long long dz_bytes, part_bytes, dw_bytes;
};
static long long up256(long long n) { return (n + 255) / 256 * 256; }
static BackPlan plan_backward(const Shape &p, bool need_x, bool need_w, bool need_b, bool need_r) {
    BackPlan q{};
    const int E = std::max(p.E, 1), es = p.dtype == 0 ? 4 : 2;
    q.sums = need_b;
    q.dz = p.act != MDX_ACT_NONE && (need_x || need_w) && !need_r;
    q.slices = act_slices(E, p.T, p.N);
    q.splits = need_w ? dw_splits(E, p.T, p.N, p.K, p.dtype) : 1;
    q.dz_bytes = q.dz ? up256(p.T * p.N * es) : 0;
    q.part_bytes = need_b ? up256((long long)E * q.slices * p.N * 4) : 0;
    q.dw_bytes = q.splits > 1 ? up256((long long)q.splits * E * p.N * p.K * 4) : 0;
    return q;
}

template <typename T> static int backward(const Shape &p, const Back &b, hipStream_t s) {
    const BackPlan q = plan_backward(p, b.dx, b.dw, b.db, b.dres);
    const int E = std::max(p.E, 1);
    const void *dz = b.grad;
    long long lddz = b.ldg;
    float *part = reinterpret_cast<float *>(b.ws + q.dz_bytes);
    if (q.dz || b.db || b.dres) {
        ActArgs a{};
        a.dy = b.grad; a.ldy = b.ldg;
        a.z = b.pre; a.ldz = b.ldp;
        a.dz = b.dres ? b.dres : q.dz ? b.ws : nullptr;
        a.lddz = b.dres ? b.lddr : p.N;
        a.part = b.db ? part : nullptr;
        a.counts = b.counts;
        a.E = E; a.T = p.T; a.N = p.N; a.act = p.act;
        const bool tail = p.E && b.dres && b.zero_tail;
        const dim3 grid((unsigned)ceil128(p.N), q.slices, E + tail);
        hipLaunchKernelGGL(k_act_backward<T>, grid, dim3(256), 0, s, a);
        MDX_CHECK_LAUNCH("mdx_linear_backward");
        if (b.db) {
            hipLaunchKernelGGL(k_bias_join, dim3((unsigned)ceil_div(p.N, 256), E), dim3(256), 0, s, part, q.slices,
                               p.N, b.db);
            MDX_CHECK_LAUNCH("mdx_linear_backward");
        }
        if (a.dz && p.act != MDX_ACT_NONE) {
            dz = a.dz;
            lddz = a.lddz;
        }
    }
    if (b.dx && p.T) {
        Args g{};
        g.a = dz; g.lda = lddz;
        g.b = b.w; g.ldb = b.ldw;
        g.I = p.T; g.J = p.K; g.R = p.N;
        g.out = b.dx; g.ldo = b.lddx;
        g.counts = b.counts; g.E = p.E; g.T = p.T;
        g.gstride = (long long)p.N * b.ldw;
        g.zero_tail = b.zero_tail;
        g.splits = 1;
        const int rc = p.E ? launch_product<T, false, true, GROUP_ROWS>(g, s)
                           : launch_product<T, false, true, DENSE>(g, s);
        if (rc != MDX_OK) return rc;
    }
    if (b.dw) {
        Args g{};
        g.a = dz; g.lda = lddz;
        g.b = b.x; g.ldb = b.ldx;
        g.I = p.N; g.J = p.K; g.R = p.T;
        g.out = b.dw; g.ldo = b.lddw;
        g.counts = b.counts; g.E = p.E; g.T = p.T;
        g.gstride = (long long)p.N * b.lddw;
        g.splits = q.splits;
        g.part = reinterpret_cast<float *>(b.ws + q.dz_bytes + q.part_bytes);
        const int rc = p.E ? launch_product<T, true, true, GROUP_RED>(g, s) : launch_product<T, true, true, DENSE>(g, s);
        if (rc != MDX_OK) return rc;
    }
    return MDX_OK;
}

static int run_forward(const char *fn, const Shape &p, const Args &g, hipStream_t s) {
    MDX_REQUIRE(g.a && g.b && g.out, "%s: null pointer", fn);
    MDX_REQUIRE(!bad_ld(g.a, g.lda, p.K) && !bad_ld(g.b, g.ldb, p.K) && !bad_ld(g.res, g.ldr, p.N) &&
                    !bad_ld(g.pre, g.ldp, p.N) && !bad_ld(g.out, g.ldo, p.N),
                "%s: a row stride is below its row's length", fn);
    switch (p.dtype) {
        case 0: return forward<float>(p, g, s);
        case 1: return forward<_Float16>(p, g, s);
        default: return forward<__bf16>(p, g, s);
    }
}
static int run_backward(const char *fn, const Shape &p, const Back &b, int64_t ws_bytes, hipStream_t s) {
    if (p.T > 0) {  // without rows the sums are zero, and nothing is read
        MDX_REQUIRE(b.grad, "%s: null gradient", fn);
        MDX_REQUIRE(p.act == MDX_ACT_NONE || b.pre, "%s: an activation needs the saved pre-activation", fn);
        MDX_REQUIRE(!b.dx || b.w, "%s: dx needs the weight", fn);
        MDX_REQUIRE(!b.dw || b.x, "%s: dw needs the input", fn);
    }
    MDX_REQUIRE(!bad_ld(b.grad, b.ldg, p.N) && !bad_ld(b.x, b.ldx, p.K) && !bad_ld(b.w, b.ldw, p.K) &&
                    !bad_ld(b.pre, b.ldp, p.N) && !bad_ld(b.dx, b.lddx, p.K) && !bad_ld(b.dw, b.lddw, p.K) &&
                    !bad_ld(b.dres, b.lddr, p.N),
                "%s: a row stride is below its row's length", fn);
    const BackPlan q = plan_backward(p, b.dx, b.dw, b.db, b.dres);
    const long long need = q.dz_bytes + q.part_bytes + q.dw_bytes;
    MDX_REQUIRE(need == 0 || (b.ws && ws_bytes >= need), "%s: needs %lld bytes of workspace, got %lld", fn, need,
                (long long)ws_bytes);
    switch (p.dtype) {
        case 0: return backward<float>(p, b, s);
        case 1: return backward<_Float16>(p, b, s);
        default: return backward<__bf16>(p, b, s);
    }
}

}  // namespace lin
}  // namespace mdx

using namespace mdx;
using namespace mdx::lin;

extern "C" int64_t mdx_linear_workspace_bytes(int64_t M, int N, int K, int dtype) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const int s = fwd_splits(M, N, K, dtype);
    return s > 1 ? (int64_t)s * M * N * 4 : 0;
}
extern "C" int mdx_linear(const void *x, int64_t ldx, const void *w, int64_t ldw, const float *bias,
                          const void *residual, int64_t ldr, int64_t M, int N, int K, int act, int dtype, void *pre,
                          int64_t ldp, void *out, int64_t ldo, void *workspace, int64_t workspace_bytes,
                          mdx_stream_t stream) {
    const Shape p{M, 0, N, K, dtype, act};
    if (int rc = check_shape("mdx_linear", p)) return rc;
    if (M == 0) return MDX_OK;
    Args g{};
    g.a = x; g.lda = ldx;
    g.b = w; g.ldb = ldw;
    g.I = M; g.J = N; g.R = K;
    g.bias = bias;
    g.res = residual; g.ldr = ldr;
    g.pre = pre; g.ldp = ldp;
    g.out = out; g.ldo = ldo;
    g.act = act;
    g.splits = fwd_splits(M, N, K, dtype);
    g.part = reinterpret_cast<float *>(workspace);
    if (!workspace || workspace_bytes < (int64_t)g.splits * M * N * 4) g.splits = 1;
    return run_forward("mdx_linear", p, g, as_stream(stream));
}

extern "C" int64_t mdx_linear_backward_workspace_bytes(int64_t M, int N, int K, int act, int dtype, int need_x,
                                                       int need_w, int need_bias, int need_residual) {
    if (M < 0 || N <= 0 || K <= 0) return 0;
    const BackPlan q = plan_backward(Shape{M, 0, N, K, dtype, act}, need_x, need_w, need_bias, need_residual);
    return q.dz_bytes + q.part_bytes + q.dw_bytes;
}
extern "C" int mdx_linear_backward(const void *grad, int64_t ldg, const void *x, int64_t ldx, const void *w,
                                   int64_t ldw, const void *pre, int64_t ldp, int64_t M, int N, int K, int act,
                                   int dtype, void *dx, int64_t lddx, void *dw, int64_t lddw, float *dbias, void *dres,
                                   int64_t lddr, void *workspace, int64_t workspace_bytes, mdx_stream_t stream) {
    const Shape p{M, 0, N, K, dtype, act};
    if (int rc = check_shape("mdx_linear_backward", p)) return rc;
    Back b{};
    b.grad = grad; b.ldg = ldg;
    b.x = x; b.ldx = ldx;
    b.w = w; b.ldw = ldw;
    b.pre = pre; b.ldp = ldp;
    b.dx = dx; b.lddx = lddx;
    b.dw = dw; b.lddw = lddw;
    b.db = dbias;
    b.dres = dres; b.lddr = lddr;
    b.ws = reinterpret_cast<char *>(workspace);
    return run_backward("mdx_linear_backward", p, b, workspace_bytes, as_stream(stream));
}

extern "C" int mdx_grouped_linear(const void *x, int64_t ldx, const void *w, const float *bias, const void *residual,
                                  int64_t ldr, const int *counts, int E, int64_t T, int N, int K, int act, int dtype,
                                  void *pre, int64_t ldp, void *out, int64_t ldo, int zero_tail, mdx_stream_t stream) {
    const Shape p{T, E, N, K, dtype, act};
    if (int rc = check_shape("mdx_grouped_linear", p)) return rc;
    MDX_REQUIRE(E > 0 && counts, "mdx_grouped_linear: needs one group or more, and their counts");
    if (T == 0) return MDX_OK;
    Args g{};
    g.a = x; g.lda = ldx;
    g.b = w; g.ldb = K;
    g.I = T; g.J = N; g.R = K;
    g.bias = bias;
    g.res = residual; g.ldr = ldr;
    g.pre = pre; g.ldp = ldp;
    g.out = out; g.ldo = ldo;
    g.act = act;
    g.counts = counts; g.E = E; g.T = T;
    g.gstride = (long long)N * K;
    g.zero_tail = zero_tail;
    g.splits = 1;
    return run_forward("mdx_grouped_linear", p, g, as_stream(stream));
}

extern "C" int64_t mdx_grouped_linear_backward_workspace_bytes(int E, int64_t T, int N, int K, int act, int dtype,
                                                               int need_x, int need_w, int need_bias,
                                                               int need_residual) {
    if (E <= 0 || T < 0 || N <= 0 || K <= 0) return 0;
    const BackPlan q = plan_backward(Shape{T, E, N, K, dtype, act}, need_x, need_w, need_bias, need_residual);
    return q.dz_bytes + q.part_bytes + q.dw_bytes;
}
extern "C" int mdx_grouped_linear_backward(const void *grad, int64_t ldg, const void *x, int64_t ldx, const void *w,
                                           const void *pre, int64_t ldp, const int *counts, int E, int64_t T, int N,
                                           int K, int act, int dtype, void *dx, int64_t lddx, void *dw, float *dbias,
                                           void *dres, int64_t lddr, int zero_tail, void *workspace,
                                           int64_t workspace_bytes, mdx_stream_t stream) {
    const Shape p{T, E, N, K, dtype, act};
    if (int rc = check_shape("mdx_grouped_linear_backward", p)) return rc;
    MDX_REQUIRE(E > 0 && counts, "mdx_grouped_linear_backward: needs one group or more, and their counts");
    Back b{};
    b.grad = grad; b.ldg = ldg;
    b.x = x; b.ldx = ldx;
    b.w = w; b.ldw = K;
    b.pre = pre; b.ldp = ldp;
    b.counts = counts;
    b.dx = dx; b.lddx = lddx;
    b.dw = dw; b.lddw = K;
    b.db = dbias;
    b.dres = dres; b.lddr = lddr;
    b.zero_tail = zero_tail;
    b.ws = reinterpret_cast<char *>(workspace);
    return run_backward("mdx_grouped_linear_backward", p, b, workspace_bytes, as_stream(stream));
}
