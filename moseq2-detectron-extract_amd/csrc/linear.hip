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
// so no operand is ever transposed in memory.  Sums are float32 in the matrix
// instructions; each output is rounded once.  dz is rounded to the operands'
// type before the two products, since the matrix instructions take nothing
// wider: a term is off by half a step of that type at most (bf16 gradients of
// 8192 x 4096 x 1024 GELU are off by 0.0023 of their size on the whole, where rounded
// outputs alone give 0.0017; fp16 999 x 517 x 1001 SiLU 2.9e-4 and 2.1e-4).  A dz in
// two parts would keep the rest for twice the products' time (8192 x 4096 x 1024:
// 113 us); between separate layers of the type it is rounded just so.  In fp16
// it shares the type's range: beyond 65504 infinite, below 2^-25 zero.
#include "pieces.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace mdx {
namespace lin {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 *lds_s4;

// N values of a row from its element c on as floats, of which the first n exist
template <typename T, int N> __device__ __forceinline__ void load_row(const T *p, int c, int n, float (&v)[N]) {
    constexpr int P = VEC<T>;
#pragma unroll
    for (int k = 0; k < N / P; ++k) {
        union { u4 u; T e[P]; } r;
        r.u = load_piece(p + k * P, c + k * P, n - k * P);
#pragma unroll
        for (int q = 0; q < P; ++q) v[k * P + q] = (float)r.e[q];
    }
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
// ---- activations, in float32 ------------------------------------------------
// On the hardware's exp2 and reciprocal (1 ulp each): with the library's erff,
// tanhf and division the epilogue of a 256 x 256 tile took longer than its
// product of 1024 terms.  That tile is for 16-bit outputs, to which GATE16 gives
// some 15 bits; float32 outputs take GATE32, good to 16 * 2^-24 of the value, whose
// exponents are formed in float64 (an exponent of 100 rounded to float32 alone is
// off by 4e-6 of the power) and given to exp2 in two parts.
enum Gates { GATE16, GATE32 };
template <typename T> constexpr Gates GATES = sizeof(T) == 4 ? GATE32 : GATE16;
constexpr double LOG2E = 1.4426950408889634;
// the normal distribution at z <= 0 is exp(-z^2 / 2) times a smooth function of
// |z|, taken as t = 1 / (1 + a |z|) times a polynomial that was fitted (minimax,
// up to |z| = 14.5, where the product leaves the range of float32) to the
// relative error, so that far tails keep their digits
//   GATE16: a = 0.3, degree 5: 2.2e-5 of the tail, 2.2e-7 in all (3.5e-7 as computed)
//   GATE32: a = 0.4 and t - 0.43, degree 8, from |z| = 1 on: 1e-8; below 1 the odd
//           series' part z R(z^2) beside 1 / 2, whose degree 5 gives 1e-8
constexpr float TAIL16[] = {0.12006758f, 0.113622055f, 0.145469342f, -0.0207057571f, 0.220405522f, -0.0788589624f};
constexpr float TAIL32[] = {0.2594182808f,  0.31709961f,    0.2142576792f,   0.0003599896101f, -0.1069903019f,
                            -0.01009159273f, 0.07743831973f, -0.00430055336f, -0.05770715095f};
constexpr float CENTRE32[] = {0.3989422798f,   -0.06649034774f, 0.009973218223f,
                              -0.001186034065f, 0.0001131538992f, -7.524209733e-06f};
template <int N> __device__ __forceinline__ float polynomial(const float (&c)[N], float x) {
    float v = c[N - 1];
#pragma unroll
    for (int k = N - 2; k >= 0; --k) v = fmaf(v, x, c[k]);
    return v;
}
// 2^u, u <= 0
__device__ __forceinline__ float exp2_of(double u) {
    u = fmax(u, -200.0);
    const float hi = (float)u, e = __builtin_amdgcn_exp2f(hi);
    return fmaf(e * (float)(u - (double)hi), 0.69314718056f, e);
}
// 1 / d, 1 <= d < 4
__device__ __forceinline__ float reciprocal(float d) {
    const float r = __builtin_amdgcn_rcpf(d);
    return fmaf(fmaf(-d, r, 1.f), r, r);
}
// the normal distribution at z: *p its probability (1 + erf(z / sqrt 2)) / 2,
// returned exp(-z^2 / 2), which that needs and the density is made of
template <Gates G> __device__ __forceinline__ float normal_cdf(float z, float *p) {
    const float m = fabsf(z);
    if constexpr (G == GATE16) {
        const float t = __builtin_amdgcn_rcpf(1.f + 0.3f * m);
        const float e = __builtin_amdgcn_exp2f(z * z * (float)(-0.5 * LOG2E));
        const float c = e * t * polynomial(TAIL16, t);
        *p = z < 0.f ? c : 1.f - c;
        return e;
    } else {
        const float e = exp2_of((double)z * z * (-0.5 * LOG2E));
        const float t = __builtin_amdgcn_rcpf(fmaf(0.4f, fminf(m, 1e4f), 1.f));
        const float c = e * t * polynomial(TAIL32, t - 0.43f);
        *p = m < 1.f ? fmaf(z, polynomial(CENTRE32, z * z), 0.5f) : z < 0.f ? c : 1.f - c;
        return e;
    }
}
// 1 / (1 + exp(-v)) and what it lacks to 1, v = z (silu) or 2 sqrt(2 / pi) (z + A z^3)
// (the tanh form: (1 + tanh(v / 2)) / 2).  GATE16 gives 0 where exp(-v) passes the range.
constexpr double TANH_C = 1.5957691216057308, TANH_A = 0.044715;
template <Gates G, int ACT> __device__ __forceinline__ float logistic(float z, float *rest) {
    if constexpr (G == GATE16) {
        constexpr float c = (float)(-TANH_C * LOG2E), a = (float)(-TANH_C * TANH_A * LOG2E);
        const float u = ACT == MDX_ACT_SILU ? (float)-LOG2E * z : z * (c + a * (z * z));
        const float s = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u));
        *rest = 1.f - s;
        return s;
    } else {
        const double x = z, v = ACT == MDX_ACT_SILU ? x : x * (TANH_C + TANH_C * TANH_A * (x * x));
        const float e = exp2_of(-LOG2E * fabs(v)), r = reciprocal(1.f + e);
        *rest = z < 0.f ? r : e * r;
        return z < 0.f ? e * r : r;
    }
}

template <Gates G, int ACT> __device__ __forceinline__ float act_value(float z) {
    float p;
    if constexpr (ACT == MDX_ACT_RELU) return z < 0.f ? 0.f : z;  // NaN stays NaN
    if constexpr (ACT == MDX_ACT_GELU) {
        normal_cdf<G>(z, &p);
        return z * p;
    }
    return z * logistic<G, ACT>(z, &p);
}
// dy act'(z); ReLU selects, so that an infinite gradient of a closed unit is dropped
template <Gates G, int ACT> __device__ __forceinline__ float act_grad(float dy, float z) {
    float p;
    if constexpr (ACT == MDX_ACT_RELU) return z > 0.f ? dy : 0.f;
    if constexpr (ACT == MDX_ACT_GELU) {
        const float e = normal_cdf<G>(z, &p);
        return dy * (p + z * e * 0.39894228040143268f);
    }
    const float s = logistic<G, ACT>(z, &p);
    if constexpr (ACT == MDX_ACT_SILU) return dy * (s * (1.f + z * p));
    // z^2 is cut where the gate has long been 0 or 1, so that it cannot overflow beside them
    return dy * (s + z * s * p * (float)TANH_C * (1.f + (float)(3 * TANH_A) * fminf(z * z, 1e30f)));
}
// a whole piece: the activation is chosen once, not for each element
template <Gates G, int ACT, int N> __device__ __forceinline__ void apply(float (&v)[N]) {
#pragma unroll
    for (int q = 0; q < N; ++q) v[q] = act_value<G, ACT>(v[q]);
}
template <Gates G, int N> __device__ __forceinline__ void apply_act(float (&v)[N], int act) {
    switch (act) {
        case MDX_ACT_RELU: return apply<G, MDX_ACT_RELU>(v);
        case MDX_ACT_GELU: return apply<G, MDX_ACT_GELU>(v);
        case MDX_ACT_GELU_TANH: return apply<G, MDX_ACT_GELU_TANH>(v);
        case MDX_ACT_SILU: return apply<G, MDX_ACT_SILU>(v);
    }
}
template <Gates G, int ACT, int N> __device__ __forceinline__ void apply_grad(float (&v)[N], const float (&z)[N]) {
#pragma unroll
    for (int q = 0; q < N; ++q) v[q] = act_grad<G, ACT>(v[q], z[q]);
}
template <Gates G, int N>
__device__ __forceinline__ void apply_act_grad(float (&v)[N], const float (&z)[N], int act) {
    switch (act) {
        case MDX_ACT_RELU: return apply_grad<G, MDX_ACT_RELU>(v, z);
        case MDX_ACT_GELU: return apply_grad<G, MDX_ACT_GELU>(v, z);
        case MDX_ACT_GELU_TANH: return apply_grad<G, MDX_ACT_GELU_TANH>(v, z);
        case MDX_ACT_SILU: return apply_grad<G, MDX_ACT_SILU>(v, z);
    }
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

// a value that is the same in all lanes, in scalar registers
__device__ __forceinline__ long long uniform(long long v) {
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
    return (long long)((uint64_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32)) << 32 | lo);
}
// inclusive scan of v over the wave, every partial sum cut at most (below
// 2^31), so that no count makes it wrap; lane shifts in the ALU (DPP)
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t dpp_add(uint32_t v, uint32_t most) {
    return min(v + (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false), most);
}
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, uint32_t most) {
    v = dpp_add<0x111, 0xf>(v, most);  // row_shr 1, 2, 4, 8: rows of 16 lanes
    v = dpp_add<0x112, 0xf>(v, most);
    v = dpp_add<0x114, 0xf>(v, most);
    v = dpp_add<0x118, 0xf>(v, most);
    v = dpp_add<0x142, 0xa>(v, most);  // row_bcast 15, 31: the rows before
    return dpp_add<0x143, 0xc>(v, most);
}

struct Span {
    int e;           // group, E = the rows behind the last one, -1 = none
    int start, end;  // its rows
    int tile, tile0; // tile within the group; the group's first tile
};
// 64 groups at once, a lane each: their rows start .. end, cut at T, and their
// first tiles of bm rows.  Every wave that needs a group scans the counts
// itself, so no pass over them has to run before.
struct Groups {
    uint32_t start, end, tile0, tiles;  // of the lane's group
    uint32_t rows, next;                // behind the last of the 64: rows, tiles
    __device__ __forceinline__ Groups(const int *counts, int E, long long T, int bm, int base, uint32_t rows0,
                                      uint32_t first) {
        const int lane = threadIdx.x & 63;
        const uint32_t t = (uint32_t)T, c = base + lane < E ? min((uint32_t)max(counts[base + lane], 0), t) : 0;
        const uint32_t sum = wave_scan(c, t), before = (uint32_t)__shfl_up((int)sum, 1);  // with all lanes active
        end = min(rows0 + sum, t);
        start = min(rows0 + (lane ? before : 0u), t);
        tiles = (end - start + bm - 1) / bm;
        const uint32_t all = wave_scan(tiles, 0x7fffffffu);
        tile0 = first + all - tiles;
        rows = __builtin_amdgcn_readlane(end, 63);
        next = first + __builtin_amdgcn_readlane(all, 63);
    }
    __device__ __forceinline__ Span span(unsigned long long hit, int base, int tile) const {
        const int l = __ffsll(hit) - 1, t0 = (int)__builtin_amdgcn_readlane(tile0, l);
        return Span{base + l, (int)__builtin_amdgcn_readlane(start, l), (int)__builtin_amdgcn_readlane(end, l),
                    tile - t0, t0};
    }
    __device__ __forceinline__ unsigned long long holds(int tile) const {
        return __ballot((uint32_t)tile >= tile0 && (uint32_t)tile < tile0 + tiles);
    }
};
// group `want` (below E), its rows cut into tiles of bm
__device__ __forceinline__ Span find_group(const int *counts, int E, long long T, int bm, int want) {
    uint32_t rows = 0, next = 0;
    for (int base = 0;; base += 64) {
        const Groups g(counts, E, T, bm, base, rows, next);
        if (want < base + 64) return g.span(1ull << (want - base), base, 0);
        rows = g.rows;
        next = g.next;
    }
}
// the group that holds tile `tile`, or the rows behind the last one (e = E), or none
__device__ __forceinline__ Span find_tile(const int *counts, int E, long long T, int bm, int tile) {
    uint32_t rows = 0, next = 0;
    for (int base = 0; base < E; base += 64) {
        const Groups g(counts, E, T, bm, base, rows, next);
        if (const unsigned long long hit = g.holds(tile)) return g.span(hit, base, tile);
        rows = g.rows;
        next = g.next;
    }
    if (rows < (uint32_t)T && tile < (int)(next + ((uint32_t)T - rows + bm - 1) / bm))
        return Span{E, (int)rows, (int)T, tile - (int)next, (int)next};
    return Span{-1, 0, 0, 0, 0};
}

// tile id of ti x tj -> (row tile, column tile): contiguous ranges of tiles for
// each of the 8 XCDs (their L2s are separate; workgroups go to them in turn),
// and in a range squares of 8 row tiles, column by column
__device__ __forceinline__ void map_tile(unsigned id, unsigned ti, unsigned tj, int &t, int &u) {
    const unsigned n = ti * tj, q = n / 8, r = n % 8, x = id % 8;
    id = (x < r ? x * (q + 1) : r * (q + 1) + (x - r) * q) + id / 8;
    const unsigned per = 8 * tj, g = id / per, in = id - g * per, rows = min(8u, ti - 8 * g);
    t = 8 * g + in % rows;
    u = in / rows;
}

// The k-th longest of up to 64 groups (of equal ones the first), and how many
// have more than `rows` rows: long reductions are started first.
__device__ __forceinline__ int ranked_group(const Groups &g, int E, int k) {
    const int lane = threadIdx.x & 63;
    const uint32_t mine = g.end - g.start;
    int rank = 0;
    for (int l = 0; l < E; ++l) {
        const uint32_t n = __builtin_amdgcn_readlane(mine, l);
        rank += n > mine || (n == mine && l < lane);
    }
    return __ffsll(__ballot(lane < E && rank == k)) - 1;
}
__device__ __forceinline__ int groups_above(const Groups &g, uint32_t rows) {
    return __popcll(__ballot(g.end - g.start > rows));  // lanes without a group have none
}

// What a workgroup computes: rows i0 .. of i1, columns from j0, the reduction
// r0 .. r1, and the offsets of its group and slice.
struct Where {
    long long i0, i1, r0, r1, boff, biasoff, ooff;
    int j0, grp;  // grp: place of its partial sums
    bool tail;    // rows behind the last group: zeros
};
// tile id of a product in tiles of bi x bj, its slices in steps of bk; false:
// there is none (the grid of grouped rows is a bound)
template <int MODE> __device__ __forceinline__ bool place(const Args &g, int id, int bi, int bj, int bk, Where &w) {
    w = Where{0, g.I, 0, g.R, 0, 0, 0, 0, 0, false};
    int t, u;
    if (MODE == GROUP_ROWS) {
        const Groups first(g.counts, g.E, g.T, bi, 0, 0, 0);
        uint32_t rows = first.rows, tiles = first.next;
        for (int base = 64; base < g.E; base += 64) {
            const Groups k(g.counts, g.E, g.T, bi, base, rows, tiles);
            rows = k.rows;
            tiles = k.next;
        }
        if (id >= (int)tiles * g.tj) {  // the rows behind come last, so that the XCDs' ranges are even
            id -= (int)tiles * g.tj;
            w.i0 = (long long)rows + (long long)(id / g.tj) * bi;
            w.i1 = g.T;
            w.j0 = id % g.tj * bj;
            w.r1 = 0;
            w.tail = true;
            return g.zero_tail && w.i0 < g.T;
        }
        map_tile(id, tiles, g.tj, t, u);
        const unsigned long long hit = first.holds(t);
        const Span s = hit ? first.span(hit, 0, t) : find_tile(g.counts, g.E, g.T, bi, t);
        w.i0 = s.start + (long long)bi * s.tile;
        w.i1 = s.end;
        w.boff = s.e * g.gstride;
        w.biasoff = (long long)s.e * g.J;
        w.j0 = bj * u;
        return true;
    }
    int z = 0;
    if (MODE == GROUP_RED || g.splits > 1) {  // a group's slices follow each other, the longest group first
        const int per = g.ti * g.tj, k = id / per;
        id -= k * per;
        z = MODE == GROUP_RED ? k % g.splits : k;
        w.grp = z;
        if (MODE == GROUP_RED) {
            int e = k / g.splits;
            Span s;
            if (g.E <= 64) {
                const Groups all(g.counts, g.E, g.T, 1, 0, 0, 0);
                e = ranked_group(all, g.E, e);
                s = all.span(1ull << e, 0, 0);
            } else {
                s = find_group(g.counts, g.E, g.T, 1, e);
            }
            w.grp = z * g.E + e;
            w.r0 = s.start;
            w.r1 = s.end;
            w.ooff = e * g.gstride;
        }
    }
    map_tile(id, g.ti, g.tj, t, u);
    w.i0 = (long long)bi * t;
    w.j0 = bj * u;
    if (g.splits > 1) {  // this slice of the reduction, in whole steps
        const int steps = (int)((w.r1 - w.r0 + bk - 1) / bk), per = (steps + g.splits - 1) / g.splits;
        w.r0 = min(w.r1, w.r0 + (long long)z * per * bk);
        w.r1 = min(w.r1, w.r0 + (long long)per * bk);
    }
    return true;
}

// a row: a part that is the same in all lanes, and the lane's
struct Row {
    long long u;
    int l;
    __device__ __forceinline__ long long at(long long ld) const { return u * ld + l * ld; }
};
// 16 bytes of a row of outputs from their sums v: bias b (zeros if there is
// none), residual, activation and the stores
template <typename T>
__device__ __forceinline__ void finish(const Args &g, long long ooff, Row i, int j, float (&v)[VEC<T>],
                                       const float (&b)[VEC<T>], u4 res) {
    constexpr int N = VEC<T>;
    const int n = g.J - j;
    union { u4 u; T e[N]; } r;
    r.u = res;
    if (g.bias)
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] += b[q];
    if (g.res)
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] += (float)r.e[q];
    if (g.pre) store_row<T, N>(reinterpret_cast<T *>(g.pre) + i.at(g.ldp) + j, n, v);
    apply_act<GATES<T>>(v, g.act);
    store_row<T, N>(reinterpret_cast<T *>(g.out) + ooff + i.at(g.ldo) + j, n, v);
}
template <typename T> __device__ __forceinline__ u4 load_residual(const Args &g, Row i, int j) {
    return g.res ? load_piece(reinterpret_cast<const T *>(g.res) + i.at(g.ldr) + j, j, g.J - j) : u4{0, 0, 0, 0};
}
// where the sums go: a slice's partial sums, zeros behind the last group, or
// the finished outputs
template <typename T>
__device__ __forceinline__ void store_outputs(const Args &g, const Where &w, Row row, int col,
                                              float (&v)[VEC<T>], const float (&b)[VEC<T>], u4 res) {
    constexpr int N = VEC<T>;
    const int n = g.J - col;
    if (g.splits > 1) {
        store_row<float, N>(g.part + w.grp * g.I * g.J + row.at(g.J) + col, n, v);
    } else if (w.tail) {
        store_row<T, N>(reinterpret_cast<T *>(g.out) + row.at(g.ldo) + col, n, v);
        if (g.pre) store_row<T, N>(reinterpret_cast<T *>(g.pre) + row.at(g.ldp) + col, n, v);
    } else {
        finish<T>(g, w.ooff, row, col, v, b, res);
    }
}
// A wave's sums, P blocks of 16 rows by Q columns (64 or 32) from column col0
// on, AT of them at a time: blocks p .., whose first rows are row(p) .., are put
// by put(p, e) into the wave's own epi_bytes(Q, AT) of LDS e and from there
// finished, 16 bytes of a row to a lane, so that a row's lanes store whole
// lines.  A lane's column is the same in all blocks: its bias is loaded once,
// and the residual AT blocks ahead.  Two blocks at a time hide the way through
// LDS (1000 x 1024 x 1024 bf16 GELU in 64-wide tiles 9.6 -> 8.9 us); beside the
// 128 sums of a lane in the 256-wide tile there is room for one.
// put_block is a 16 x 16 tile's part: lane (row l & 15, columns 4 (l >> 4)..);
// slots of 16 bytes are XOR-swizzled by row against bank conflicts.
template <int N, int K = 0, typename F> __device__ __forceinline__ void static_for(F f) {
    if constexpr (K < N) {
        f(std::integral_constant<int, K>{});
        static_for<N, K + 1>(f);
    }
}
constexpr int epi_bytes(int q, int at) { return at * 16 * q * 4; }
template <int Q> __device__ __forceinline__ void put_block(float *e, int j, f4 v) {
    const int lane = threadIdx.x & 63, r = lane & 15, slot = (4 * j + (lane >> 4)) ^ (r & (Q / 4 - 1));
    *reinterpret_cast<f4 *>(e + r * Q + 4 * slot) = v;
}
template <typename T, int Q, int P, int AT, typename R, typename F>
__device__ __forceinline__ void epilogue(const Args &g, const Where &w, char *lds, int col0, R row, F put) {
    constexpr int N = VEC<T>, PER = Q / N, K = 16 * PER / 64;  // PER lanes to a row, K pieces to a lane
    const int lane = threadIdx.x & 63, c = lane % PER * N, col = col0 + c, lr = lane / PER;
    float *e = reinterpret_cast<float *>(lds);
    const bool in = col < g.J, plain = g.splits == 1 && !w.tail;
    float b[N] = {};
    if (g.bias && plain) load_row<float, N>(g.bias + w.biasoff + col, col, in ? g.J - col : 0, b);
    auto each = [&](auto f) {
#pragma unroll
        for (int h = 0; h < AT; ++h)
#pragma unroll
            for (int k = 0; k < K; ++k) f(h, k);
    };
    u4 next[AT][K];
    auto prefetch = [&](int p) {
        each([&](int h, int k) {
            const Row i{row(p + h) + 64 / PER * k, lr};
            next[h][k] = plain && in && i.u + lr < w.i1 ? load_residual<T>(g, i, col) : u4{0, 0, 0, 0};
        });
    };
    prefetch(0);
#pragma unroll 1
    for (int p = 0; p < P; p += AT) {
        put(p, e);
        u4 res[AT][K];
        each([&](int h, int k) { res[h][k] = next[h][k]; });
        if (p + AT < P) prefetch(p + AT);
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
        float v[AT][K][N];
        each([&](int h, int k) {
#pragma unroll
            for (int q = 0; q < N / 4; ++q) {
                const int r = 64 / PER * k + lr;
                *reinterpret_cast<f4 *>(v[h][k] + 4 * q) = *reinterpret_cast<const f4 *>(
                    e + (16 * h + r) * Q + 4 * ((c / 4 + q) ^ (r & (Q / 4 - 1))));
            }
        });
        each([&](int h, int k) {
            const Row i{row(p + h) + 64 / PER * k, lr};
            if (i.u + lr < w.i1 && in) store_outputs<T>(g, w, i, col, v[h][k], b, res[h][k]);
        });
        __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    }
}

// 16 x 16 sums over a fragment of 16 bytes of each operand, in STEPS instructions
template <typename T> struct Mma {
    static constexpr int STEPS = 1;
    static __device__ __forceinline__ f4 mul_step(u4 x, u4 y, f4 c, int) {
        if constexpr (std::is_same<T, __bf16>::value)
            return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), c, 0, 0,
                                                           0);
        else
            return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, x), __builtin_bit_cast(h8, y), c, 0, 0,
                                                          0);
    }
    static __device__ __forceinline__ f4 mul(u4 x, u4 y, f4 c) { return mul_step(x, y, c, 0); }
};
template <> struct Mma<float> {
    // element k of lane (row, q) is r = 4 q + k in both operands: any order of
    // the products gives the same sum
    static constexpr int STEPS = 4;
    static __device__ __forceinline__ f4 mul_step(u4 x, u4 y, f4 c, int k) {
        return __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(f4, x)[k], __builtin_bit_cast(f4, y)[k], c, 0, 0,
                                                    0);
    }
    static __device__ __forceinline__ f4 mul(u4 x, u4 y, f4 c) {
#pragma unroll
        for (int k = 0; k < 4; ++k) c = mul_step(x, y, c, k);
        return c;
    }
};

// SIDE rows (i) of an operand by 128 bytes of reduction, staged in LDS.
// TR = 0: [SIDE][128 B], 16-B pieces XOR-swizzled by row; a fragment (row
// l & 15, piece 4 s + (l >> 4)) is one b128 read.
// TR = 1: [128 B / sizeof(T)][SIDE]; 16-bit fragments are two transposing
// 64-bit reads (16 lanes give the addresses of a 4 x 16 block, lane i gets
// its column i), 32-bit ones four b32 reads.  The swizzle spreads the rows
// that one read takes over all banks.
template <typename T, bool TR, int SIDE> struct Stage {
    static constexpr int BK = 128 / (int)sizeof(T);
    static constexpr int BYTES = SIDE * 128;
    static constexpr int PITCH = TR ? SIDE * (int)sizeof(T) : 128;
    static constexpr int PPR = PITCH / 16;           // pieces per stored row
    static constexpr int STEP = 256 / PPR;           // rows between a thread's pieces
    static constexpr int N = SIDE / 32;              // pieces of each of 256 threads

    static __device__ __forceinline__ int swz(int row) {
        if (!TR) return (row >> 1) & 7;
        if (sizeof(T) == 4) return ((row >> 2) & 3) << 2;
        if (SIDE == 64) return (((row >> 1) & 1) | (((row >> 3) & 1) << 1)) << 1;  // two rows to all banks
        return ((row & 3) | (((row >> 3) & 1) << 2)) << 1;
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

// A thread's part in staging one operand of any alignment through registers:
// its N pieces of a step.  load() brings 16 bytes for each, of the row's end
// where the piece passes it and of anything near where there is no piece;
// write() puts that right on the way to LDS, so that no load is waited for
// before.  Rows shorter than a piece are finished in load() (`tiny`).
template <typename T, bool TR, int SIDE> struct RegOperand {
    using S = Stage<T, TR, SIDE>;
    static constexpr int N = S::N, V = VEC<T>;
    const T *row[N];  // TR 0: the piece's row; TR 1: the piece in its row of the next step
    const T *base;    // TR 1: a piece that can always be read
    long long step;
    int at, end, left;  // TR 0: the piece's first r, the reduction's end; TR 1: its row of the next step, the end
    bool in[N], tiny;       // TR 0: the row exists; TR 1: (left: elements of the piece's row from its first on)
    __device__ __forceinline__ void init(const T *p, long long ld, long long i0, long long I, long long r0_, long long R) {
        const int t = threadIdx.x, pc = t % S::PPR;
        tiny = (TR ? I : R) < V;
        end = (int)R;
        step = S::BK * ld;
        if (TR) {
            const int c = (int)i0 + pc * V;
            at = (int)r0_ + t / S::PPR;
            left = (int)I - c;
            base = p + (tiny ? (left > 0 ? c : 0) : min(c, (int)I - V));
#pragma unroll
            for (int q = 0; q < N; ++q) row[q] = base + (long long)(at + S::STEP * q) * ld;
        } else {
            at = (int)r0_ + pc * V;
#pragma unroll
            for (int q = 0; q < N; ++q) {
                const long long w = i0 + t / S::PPR + S::STEP * q;
                in[q] = w < I;
                row[q] = p + min(w, I - 1) * ld;
            }
        }
    }
    // the next step's pieces
    __device__ __forceinline__ void load(u4 (&v)[N]) {
#pragma unroll
        for (int q = 0; q < N; ++q) {
            if (TR) {
                const bool live = at + S::STEP * q < end;
                if (tiny)
                    v[q] = load_piece(row[q], 0, live ? left : 0);
                else
                    v[q] = reinterpret_cast<const Un16<T> *>(live ? row[q] : base)->v;
                row[q] += step;
            } else if (tiny) {
                v[q] = load_piece(row[q] + (at < end ? at : 0), at, in[q] ? end - at : 0);
            } else {
                v[q] = reinterpret_cast<const Un16<T> *>(row[q] + min(at, end - V))->v;
            }
        }
        at += S::BK;
    }
    // the pieces that load() brought `back` steps ago
    __device__ __forceinline__ void write(char *lds, int back, const u4 (&v)[N]) const {
        const int pc = threadIdx.x % S::PPR, first = threadIdx.x / S::PPR, was = at - back * S::BK;
#pragma unroll
        for (int q = 0; q < N; ++q) {
            const int r = first + S::STEP * q;
            const int n = TR ? (was + S::STEP * q < end ? left : 0) : in[q] ? end - was : 0;
            u4 u = v[q];
            if (!tiny && n < V) u = n > 0 ? shift_down(u, (V - n) * 8 * (int)sizeof(T)) : u4{0, 0, 0, 0};
            *reinterpret_cast<u4 *>(lds + r * S::PITCH + ((pc ^ S::swz(r)) << 4)) = u;
        }
    }
};

// ---- LDS-DMA --------------------------------------------------------------
__device__ __attribute__((aligned(64))) uint4 zero_piece[4];  // what lies beyond the reduction's end

// Waits and barriers that no memory access is moved across.  The DMA is
// inline asm, so that the compiler, which would wait for all of it before any
// LDS read, leaves the count of outstanding ones to these waits.
template <int VM> __device__ __forceinline__ void dma_wait() {  // vmcnt VM, lgkmcnt 0, any expcnt
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((VM & 15) | ((VM >> 4) << 14) | 0x70);
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void dma_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}
// 16 bytes a lane to 1 KiB of LDS at dst (wave-uniform), from src or from
// base + off.  m0 holds the place in LDS, one wait state before its use.  The
// scalar operands may come straight from a v_readfirstlane: a vector memory
// instruction may read such a register only five wait states later, which the
// compiler does not see to inside inline asm.
__device__ __forceinline__ void dma16(const void *src, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(dst)),
                 "v"(src)
                 : "memory", "m0");
}
__device__ __forceinline__ void dma16s(const void *base, uint32_t off, uint32_t dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(
                     __builtin_amdgcn_readfirstlane(dst)),
                 "v"(off), "s"(uniform((long long)(uintptr_t)base))
                 : "memory", "m0");
}

// ---- the small tiles ------------------------------------------------------
// Tile SIDE x SIDE (128 or 64) per workgroup of 4 waves, each a quarter of 16 x
// 16 MFMA tiles, the reduction in steps of 128 bytes.  B is the MFMA's first
// operand, so a lane ends with 4 neighbouring columns of one row.
//
// DMA: both operands in aligned pieces of 16 bytes, brought to LDS directly,
// BUFS - 1 steps ahead, so that a lone workgroup on a CU does not wait out the
// memory's latency at each step; one barrier a step, behind which step s has
// landed everywhere and step s - 1 has been read, so that its buffer is free.
// Otherwise: any alignment and sizes, through registers, two or three steps ahead.
// 64-wide tiles are for products with too few tiles for the CUs: what bounds
// them is a step's latency (DMA 0.28 us a step of 64 in bf16, through registers
// 0.6), and they reach 235 TFLOP/s at 1000 x 1024 x 1024 bf16 (9.1 us) and 510 at
// 1000 x 1024 x 12544 in two slices (50 us).  In float32 the matrix instructions
// bound the 128-wide tile: 1000 x 1024 x 12544 in eight slices takes 208 us, of
// which the join 7.4 (124 TFLOP/s of a peak of 157).
template <typename T, int SIDE, bool DMA> constexpr int BUFS = !DMA || (sizeof(T) == 4 && SIDE == 128) ? 2 : 4;

// a lane's part in staging one operand by DMA: instruction d of wave w brings
// 1 KiB, rows (w SIDE / 32 + d) 64 / PPR ..
template <typename T, bool TR, int SIDE> struct SmallOperand {
    using S = Stage<T, TR, SIDE>;
    const char *base;  // first piece of step 0
    long long step;    // bytes between steps
    uint32_t off[S::N];
    int r[S::N];       // reduction index of the piece in its step
    __device__ __forceinline__ void init(const T *p, long long ld, long long i0, long long I, long long r0, int wid) {
        constexpr int ES = sizeof(T);
        const int lane = threadIdx.x & 63;
        base = reinterpret_cast<const char *>(
            uniform((long long)(reinterpret_cast<uintptr_t>(p) + (TR ? r0 * ld + i0 : i0 * ld + r0) * ES)));
        step = TR ? S::BK * ld * ES : 128;
#pragma unroll
        for (int d = 0; d < S::N; ++d) {
            const int row = (wid * S::N + d) * (64 / S::PPR) + lane / S::PPR, pc = (lane % S::PPR) ^ S::swz(row);
            const long long i = min(i0 + (TR ? pc * VEC<T> : row), TR ? I - VEC<T> : I - 1);
            r[d] = TR ? row : pc * VEC<T>;
            off[d] = (uint32_t)(TR ? (row * ld + i - i0) * ES : (i - i0) * ld * ES + 16 * pc);
        }
    }
    __device__ __forceinline__ void issue(long long s, long long left, uint32_t dst) const {
        if (left >= S::BK) {
#pragma unroll
            for (int d = 0; d < S::N; ++d) dma16s(base + s * step, off[d], dst + 1024 * d);
        } else {
#pragma unroll
            for (int d = 0; d < S::N; ++d)
                dma16(r[d] < left ? base + s * step + off[d] : reinterpret_cast<const char *>(zero_piece),
                      dst + 1024 * d);
        }
    }
};

template <typename T, bool TA, bool TB, int MODE, int SIDE, bool DMA>
__device__ __forceinline__ void small_product(const Args &g, char *lds, int id) {
    using SA = Stage<T, TA, SIDE>;
    using SB = Stage<T, TB, SIDE>;
    constexpr int Q = SIDE / 2, N = Q / 16;  // a wave's quarter, its MFMA tiles each way
    constexpr int STEP = SA::BYTES + SB::BYTES, NB = BUFS<T, SIDE, DMA>;
    static_assert(4 * epi_bytes(Q, 2) <= 2 * STEP, "the epilogue takes the operands' LDS");
    Where w;
    if (!place<MODE>(g, id, SIDE, SIDE, SA::BK, w)) return;
    const T *A = reinterpret_cast<const T *>(g.a), *B = reinterpret_cast<const T *>(g.b) + w.boff;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wi = (wid >> 1) * Q, wj = (wid & 1) * Q;
    f4 acc[N][N];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) acc[i][j] = f4{0.f, 0.f, 0.f, 0.f};
    auto read = [&](u4 (&fa)[2][N], u4 (&fb)[2][N], const char *la) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int i = 0; i < N; ++i) fa[h][i] = SA::frag(la, wi + 16 * i, h);
#pragma unroll
            for (int j = 0; j < N; ++j) fb[h][j] = SB::frag(la + SA::BYTES, wj + 16 * j, h);
        }
    };
    auto multiply = [&](const u4 (&fa)[2][N], const u4 (&fb)[2][N]) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int k = 0; k < Mma<T>::STEPS; ++k)
#pragma unroll
                for (int i = 0; i < N; ++i)
#pragma unroll
                    for (int j = 0; j < N; ++j) acc[i][j] = Mma<T>::mul_step(fb[h][j], fa[h][i], acc[i][j], k);
    };
    const long long len = uniform(w.r1 - w.r0), steps = (len + SA::BK - 1) / SA::BK;
    if constexpr (DMA) {
        SmallOperand<T, TA, SIDE> oa;
        SmallOperand<T, TB, SIDE> ob;
        if (steps > 0) {
            oa.init(A, g.lda, w.i0, w.i1, w.r0, wid);
            ob.init(B, g.ldb, w.j0, g.J, w.r0, wid);
            const uint32_t dst = (uint32_t)(uintptr_t)(lds_s4)lds + 1024u * SA::N * wid;
            auto issue = [&](long long s) {
                const uint32_t d = dst + (uint32_t)(s % NB) * STEP;
                oa.issue(s, len - s * SA::BK, d);
                ob.issue(s, len - s * SA::BK, d + SA::BYTES);
            };
#pragma unroll
            for (int s = 0; s < NB - 1; ++s) issue(s);
            for (long long s = 0; s < steps; ++s) {
                u4 fa[2][N], fb[2][N];
                dma_wait<(NB - 2) * 2 * SA::N>();
                dma_barrier();
                read(fa, fb, lds + (s % NB) * STEP);
                issue(s + NB - 1);  // beyond the end: zeros, so that the count stays the same
                multiply(fa, fb);
            }
            dma_wait<0>();  // nothing may land in the epilogue's LDS
        }
    } else {
        constexpr int AHEAD = SIDE == 64 ? 3 : 2;
        RegOperand<T, TA, SIDE> oa;
        RegOperand<T, TB, SIDE> ob;
        u4 va[AHEAD][SA::N], vb[AHEAD][SB::N];
        if (steps > 0) {
            oa.init(A, g.lda, w.i0, w.i1, w.r0, w.r1);
            ob.init(B, g.ldb, w.j0, g.J, w.r0, w.r1);
#pragma unroll
            for (int d = 0; d < AHEAD; ++d) {
                oa.load(va[d]);
                ob.load(vb[d]);
            }
        }
        for (int s0 = 0; s0 < (int)steps; s0 += AHEAD)
#pragma unroll
            for (int d = 0; d < AHEAD; ++d) {
                const int s = s0 + d;
                if (s >= (int)steps) break;
                char *l = lds + (s & 1) * STEP;  // last read at step s - 2, before the barrier of step s - 1
                oa.write(l, AHEAD, va[d]);
                ob.write(l + SA::BYTES, AHEAD, vb[d]);
                oa.load(va[d]);
                ob.load(vb[d]);
                __syncthreads();
                u4 fa[2][N], fb[2][N];
                read(fa, fb, l);
                multiply(fa, fb);
            }
    }
    __syncthreads();  // the operands' buffers become the epilogue's
    epilogue<T, Q, N, 2>(
        g, w, lds + wid * epi_bytes(Q, 2), w.j0 + wj, [&](int p) { return w.i0 + wi + 16 * p; },
        [&](int p, float *e) {
            static_for<N / 2>([&](auto i) {
                if (p == 2 * i) {
                    static_for<N>([&](auto j) { put_block<Q>(e, j, acc[2 * i][j]); });
                    static_for<N>([&](auto j) { put_block<Q>(e + 16 * Q, j, acc[2 * i + 1][j]); });
                    asm volatile("; block %0" ::"n"(i.value));  // the branches stay apart: merged, they would
                }                                               // index the accumulators, in memory
            });
        });
}

// ---- few rows -----------------------------------------------------------
// x of at most a few rows (or groups of them) against a wide weight: what
// counts is to stream the weight.  A workgroup takes 16 NT columns by 16 MT
// rows; its waves share the reduction (or its slice), each wave 128 bytes of
// every row at a time (lane: row l & 15, two pieces at 32 (l >> 4) bytes), four
// such chunks in flight, straight from memory into the MFMAs; the waves' sums
// meet in LDS.  Rows and columns beyond the end are clamped: their products are
// not stored.  Bound by the weight's way from memory, in small layers by the
// chain of launch, load and join: bf16 1 x 4096 x 4096 8.1 us (4.2 TB/s), 16 x 1024
// x 12544 in slices 12.1 (2.1 TB/s), 4 x 1024 x 1024 3.9 (from call to call in a
// graph; a trace has 4.5 for that kernel alone).
template <typename T, int MODE, int MT, int NT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_product_few(Args g) {
    constexpr int N = VEC<T>, KC = 8 * N, U = 4, ROWS = 16 * MT, COLS = 16 * NT;
    __shared__ __attribute__((aligned(16))) float red[WAVES][ROWS][COLS];
    Where w;
    if (!place<MODE>(g, blockIdx.x, ROWS, COLS, KC, w)) return;
    const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, f = lane & 15, q = lane >> 4;
    const T *A[MT], *B[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
        B[n] = reinterpret_cast<const T *>(g.b) + w.boff + min(w.j0 + 16 * n + f, g.J - 1) * g.ldb + w.r0;
#pragma unroll
    for (int m = 0; m < MT; ++m)
        A[m] = reinterpret_cast<const T *>(g.a) + min(w.i0 + 16 * m + f, w.i1 - 1) * g.lda + w.r0;
    f4 acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = f4{0.f, 0.f, 0.f, 0.f};
    const int K = (int)(w.r1 - w.r0), whole = K / KC, r0 = (int)w.r0;
    if (!w.tail) {
        int c = wid;
        for (; c + (U - 1) * WAVES < whole; c += U * WAVES) {
            u4 b[U][NT][2];
#pragma unroll
            for (int k = 0; k < U; ++k)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int p = 0; p < 2; ++p)
                        b[k][n][p] = reinterpret_cast<const Un16<T> *>(B[n] + (c + k * WAVES) * KC + (2 * q + p) * N)->v;
#pragma unroll
            for (int k = 0; k < U; ++k)
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        const u4 a =
                            reinterpret_cast<const Un16<T> *>(A[m] + (c + k * WAVES) * KC + (2 * q + p) * N)->v;
#pragma unroll
                        for (int n = 0; n < NT; ++n) acc[m][n] = Mma<T>::mul(b[k][n][p], a, acc[m][n]);
                    }
        }
        for (; c * KC < K; c += WAVES)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const int k = c * KC + (2 * q + p) * N;
                u4 b[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) b[n] = load_piece(B[n] + k, r0 + k, K - k);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const u4 a = load_piece(A[m] + k, r0 + k, K - k);
#pragma unroll
                    for (int n = 0; n < NT; ++n) acc[m][n] = Mma<T>::mul(b[n], a, acc[m][n]);
                }
            }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) *reinterpret_cast<f4 *>(&red[wid][16 * m + f][16 * n + 4 * q]) = acc[m][n];
    __syncthreads();
    for (int t = threadIdx.x; t < ROWS * COLS / N; t += 64 * WAVES) {
        const int r = t / (COLS / N), c = t % (COLS / N) * N;
        if (w.i0 + r >= w.i1 || w.j0 + c >= g.J) continue;
        const u4 res = g.splits == 1 && !w.tail ? load_residual<T>(g, Row{w.i0, r}, w.j0 + c) : u4{0, 0, 0, 0};
        float v[N] = {}, b[N] = {};
        if (g.bias && g.splits == 1 && !w.tail)
            load_row<float, N>(g.bias + w.biasoff + w.j0 + c, w.j0 + c, g.J - w.j0 - c, b);
#pragma unroll
        for (int k = 0; k < WAVES; ++k)
#pragma unroll
            for (int e = 0; e < N; ++e) v[e] += red[k][r][c + e];
        store_outputs<T>(g, w, Row{w.i0, r}, w.j0 + c, v, b, res);
    }
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
//
// Bound by the matrix instructions while the reduction runs (1.3 us a K-tile of
// all CUs, 1.65 PFLOP/s of 2.5) and by the epilogue's stores at its end: some 12
// us of a tile are beside the K-tiles, of which half is the burst of stores.  bf16
// 8192 x 8192 x 8192 738 us (1.49 PFLOP/s), 32000 x 1024 x 12544 with ReLU 580 to
// 620 (1.33 to 1.42), 16128 x 4096 x 1024 137 to 145 (0.93 to 0.99).
constexpr int BIG = 256, BIG_BUF = 65536, BIG_LDS = 2 * BIG_BUF, BIG_HALF = 16384;

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
            const int pc = (TR ? lane & 15 : lane & 7) ^ Stage<T, TR, 128>::swz(row);
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

// Tile id of a product.  (Persistent workgroups, which had the next tile's
// first K-tiles on their way during the epilogue, spilled around it and were
// 5 to 45 % slower than a workgroup per tile; tiles of 256 x 128 with K-tiles of
// 32, two on a CU, took 177 us for 16128 x 4096 x 1024 where these took 164, and
// 1028 for 32000 x 1024 x 12544 where these took 584.)
template <typename T, bool TA, bool TB, int MODE>
__device__ __forceinline__ void big_product(const Args &g, char *lds, int id) {
    Where w;
    if (!place<MODE>(g, id, BIG, BIG, 64, w)) return;
    using std::integral_constant;
    constexpr integral_constant<int, 0> c0{};
    constexpr integral_constant<int, 1> c1{};
    constexpr integral_constant<int, 2> c2{};
    constexpr integral_constant<int, 3> c3{};
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = wid >> 2, wn = wid & 3;
    const uint32_t dst = (uint32_t)(uintptr_t)(lds_s4)lds + 2048u * wid;
    f4 acc[2][2][4][2];
#pragma unroll
    for (int k = 0; k < 32; ++k) acc[k >> 4][(k >> 3) & 1][(k >> 1) & 3][k & 1] = f4{0.f, 0.f, 0.f, 0.f};

    if (!w.tail) {
        BigOperand<T, TA, false> oa;
        BigOperand<T, TB, true> ob;
        oa.init(g.a, g.lda, w.i0, w.i1, w.r0, wid, lane);
        ob.init(reinterpret_cast<const T *>(g.b) + w.boff, g.ldb, w.j0, g.J, w.r0, wid, lane);
        const long long len = uniform(w.r1 - w.r0), KT = max(4ll, (len + 127) / 128 * 2);

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
                for (int i = 0; i < 4; ++i) fa[s][i] = Stage<T, TA, 128>::frag(p, 64 * grp + 16 * i, s);
        };
        auto read_b = [&](u4 (&fb)[2][2], int h, int par) {
            const char *p = lds + par * BIG_BUF + (2 + h) * BIG_HALF;
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int j = 0; j < 2; ++j) fb[s][j] = Stage<T, TB, 128>::frag(p, 32 * wn + 16 * j, s);
        };
        auto mul = [&](f4 (&c)[4][2], const u4 (&fb)[2][2]) {
            dma_barrier();
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) c[i][j] = Mma<T>::mul(fb[s][j], fa[s][i], c[i][j]);
            __builtin_amdgcn_s_setprio(0);
            dma_barrier();
        };
        // one K-tile in buffer PAR; END: 0 and 3 issue K-tile tt + 2 (3: which
        // may be partial), 1 and 2 are the last two
        auto tile = [&](auto End, auto Par, long long tt, u4 (&x)[2][2], u4 (&y)[2][2]) {
            constexpr int END = decltype(End)::value, PAR = decltype(Par)::value;
            constexpr bool MORE = END == 0 || END == 3;
            constexpr integral_constant<int, END == 3> part{};
            read_a(0, PAR);
            if constexpr (MORE) issue(c0, Par, part, tt + 2);
            dma_wait<MORE ? 12 : END == 1 ? 10 : 2>();
            mul(acc[0][0], x);
            read_b(y, 1, PAR);
            if constexpr (MORE) issue(c1, Par, part, tt + 2);
            dma_wait<MORE ? 12 : END == 1 ? 8 : 0>();
            mul(acc[0][1], y);
            read_a(1, PAR);
            if constexpr (MORE) issue(c2, Par, part, tt + 2);
            dma_wait<MORE ? 12 : END == 1 ? 6 : 0>();
            mul(acc[1][1], y);
            if constexpr (END != 2) read_b(y, 0, 1 - PAR);
            if constexpr (MORE) issue(c3, Par, part, tt + 2);
            dma_wait<MORE ? 12 : END == 1 ? 4 : 0>();
            mul(acc[1][0], x);
        };
        issue(c0, c0, c1, 0); issue(c1, c0, c1, 0); issue(c2, c0, c1, 0); issue(c3, c0, c1, 0);
        issue(c0, c1, c1, 1); issue(c1, c1, c1, 1); issue(c2, c1, c1, 1); issue(c3, c1, c1, 1);
        dma_wait<12>();
        dma_barrier();
        read_b(fx, 0, 0);
        dma_wait<12>();
        dma_barrier();
        if (grp == 1) dma_barrier();  // one behind
        for (long long tt = 0; tt < KT - 4; tt += 2) {
            tile(c0, c0, tt, fx, fy);
            tile(c0, c1, tt + 1, fy, fx);
        }
        tile(c3, c0, KT - 4, fx, fy);
        tile(c3, c1, KT - 3, fy, fx);
        tile(c1, c0, KT - 2, fx, fy);
        tile(c2, c1, KT - 1, fy, fx);
        if (grp == 0) dma_barrier();  // every wave crosses as many, and has read all of this tile
    }
    epilogue<T, 64, 8, 1>(
        g, w, lds + wid * epi_bytes(64, 1), w.j0 + 64 * wn,
        [&](int p) { return w.i0 + 128 * (p >> 2) + 64 * grp + 16 * (p & 3); },
        [&](int p, float *e) {
            static_for<8>([&](auto k) {
                if (p == k) {
                    static_for<4>([&](auto j) { put_block<64>(e, j, acc[k >> 2][j >> 1][k & 3][j & 1]); });
                    asm volatile("; block %0" ::"n"(k.value));  // as in small_product
                }
            });
        });
}

// ---- the bias's gradient ---------------------------------------------------
// k_act_backward's arguments
struct ActArgs {
    const void *dy, *z;
    long long ldy, ldz;
    void *dz;            // or null: sums only
    long long lddz;
    float *part;         // or null: dz only
    const int *counts;   // or null: one group of T rows
    int E, rows;
    long long T;
    int N, act;
    int zero_tail;       // write zeros to dz behind the last group
};

// units of bias_join: 16 columns of a group; a workgroup of the products'
// launch, which takes its share of LDS with it, has several
constexpr int BIAS_UNITS = 4;
__host__ __device__ inline int bias_units(const ActArgs &g) { return (g.N / 16 + (g.N % 16 != 0)) * (g.E > 1 ? g.E : 1); }

// db[e][n] = the sums of group e's chunks, always added in the same order.  256
// threads have 16 columns, 16 threads to each, so that a hundred chunks are a
// few loads in flight per thread and no chain of waits.
__device__ __forceinline__ void bias_join(const ActArgs &g, float *db, int block) {
    __shared__ float sh[4][16];
    if (threadIdx.x >= 256) return;  // a wave that has ended is at no barrier
    const int per = (g.N + 15) / 16, e = block / per, l = threadIdx.x & 15, w = threadIdx.x >> 4;
    const int col = (block - e * per) * 16 + l;
    long long first = 0, n = (g.T + g.rows - 1) / g.rows;
    if (g.counts) {
        const Span s = find_group(g.counts, g.E, g.T, g.rows, e);
        first = s.tile0;
        n = ((long long)s.end - s.start + g.rows - 1) / g.rows;
    }
    float v = 0.f;
    if (col < g.N) {
        const float *p = g.part + first * g.N + col;
        for (long long k = w; k < n; k += 8 * 16) {
            float t[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) t[q] = k + 16 * q < n ? p[(k + 16 * q) * g.N] : 0.f;
#pragma unroll
            for (int q = 0; q < 8; ++q) v += t[q];
        }
    }
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
    __syncthreads();  // the unit before this one has been read
    if ((threadIdx.x & 63) < 16) sh[threadIdx.x >> 6][l] = v;
    __syncthreads();
    if (threadIdx.x < 16 && col < g.N) {
        v = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) v += sh[k][l];
        db[(long long)e * g.N + col] = v;
    }
}
__global__ __launch_bounds__(256) void k_bias_join(ActArgs g, float *db) { bias_join(g, db, blockIdx.x); }

// ---- kernels ----------------------------------------------------------------
enum Kind { LARGE, DMA128, DMA64, REG128, REG64 };  // MDX_LINEAR_* in mdx.h
constexpr int tile_side(int kind) { return kind == LARGE ? BIG : kind == DMA128 || kind == REG128 ? 128 : 64; }
constexpr int tile_threads(int kind) { return kind == LARGE ? 512 : 256; }
template <typename T> constexpr int tile_lds(int kind) {
    return kind == LARGE    ? BIG_LDS
           : kind == DMA128 ? BUFS<T, 128, true> * 32768
           : kind == DMA64  ? BUFS<T, 64, true> * 16384
           : kind == REG128 ? 65536
                            : 32768;
}
template <typename T, bool TA, bool TB, int MODE, int KIND>
__device__ __forceinline__ void run_tile(const Args &g, char *lds, int id) {
    if constexpr (KIND == LARGE)
        big_product<T, TA, TB, MODE>(g, lds, id);
    else
        small_product<T, TA, TB, MODE, tile_side(KIND), KIND == DMA128 || KIND == DMA64>(g, lds, id);
}
template <typename T, int MODE, int KIND>
__global__ __launch_bounds__(tile_threads(KIND), 2) void k_forward(Args g) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    run_tile<T, false, false, MODE, KIND>(g, lds, blockIdx.x);
}
// dW's tiles and dx's in one launch: they need nothing of each other, and
// either alone often leaves part of the CUs without a tile (8192 x 4096 x 1024
// bf16: 113 us for both, 2 x 69 GFLOP at 1.22 PFLOP/s).  Of dW's nw tiles
// the `first` ones come before dx's, whose reduction is x.R: those that reduce
// more (grouped: of the groups with more rows).  The bias's blocks come last.
template <typename T, bool GROUPED, int KIND>
__global__ __launch_bounds__(tile_threads(KIND), 2) void k_backward(Args w, int nw, int nx, int first, Args x,
                                                                    ActArgs sums, float *db) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    int id = blockIdx.x;
    if (id >= nw + nx) {
        const int units = bias_units(sums), first = (id - nw - nx) * BIAS_UNITS;
        for (int u = first; u < min(units, first + BIAS_UNITS); ++u) bias_join(sums, db, u);
        return;
    }
    if (GROUPED && first < 0)
        first = groups_above(Groups(w.counts, w.E, w.T, 1, 0, 0, 0), (uint32_t)x.R * w.splits) * w.splits * w.ti * w.tj;
    if (id >= first && id < first + nx) {
        run_tile<T, false, true, GROUPED ? GROUP_ROWS : DENSE, KIND>(x, lds, id - first);
    } else {
        if (id >= first) id -= nx;
        run_tile<T, true, true, GROUPED ? GROUP_RED : DENSE, KIND>(w, lds, id);
    }
}

// The slices' partial sums, added in their order (no atomics: the same result
// on every call), and the epilogue; one thread per 16 bytes of output.  Bound by
// HBM: two slices of 4096 x 1024 to bf16 8.7 us for their 42 MB (4.8 TB/s).
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
        load_row<float, N>(g.part + ((s * E + blockIdx.y) * g.I + row) * g.J + col, col, g.J - col, w);
#pragma unroll
        for (int q = 0; q < N; ++q) v[q] += w[q];
    }
    float b[N] = {};
    if (g.bias) load_row<float, N>(g.bias + col, col, g.J - col, b);
    finish<T>(g, blockIdx.y * g.gstride, Row{row, 0}, col, v, b, load_residual<T>(g, Row{row, 0}, col));
}

// dz = dy act'(z) in T, and the column sums of dz before that rounding.  A
// workgroup takes one chunk of `rows` rows of a group by 32 pieces of 16 bytes;
// its sums go to part[chunk][N], and bias_join adds a group's chunks.  Bound by
// HBM: 8192 x 4096 bf16 GELU 44 us for its 201 MB (4.6 TB/s), 8000 x 2048 ReLU 17.4
// (5.6 TB/s).  On its own, since both products take dz, each in another order:
// in their loads it would be computed 4 to 16 times over and bar the direct way
// to LDS.
template <typename T>
__global__ __launch_bounds__(256, 4) void k_act_backward(ActArgs g) {
    constexpr int W = VEC<T>, AT = 2;  // rows of a thread at once
    long long r0 = (long long)blockIdx.y * g.rows, r1 = min(g.T, r0 + g.rows);
    bool tail = false;
    if (g.counts) {
        const Span s = find_tile(g.counts, g.E, g.T, g.rows, blockIdx.y);
        tail = s.e == g.E;
        if (s.e < 0 || (tail && !g.zero_tail)) return;
        r0 = s.start + (long long)s.tile * g.rows;
        r1 = min((long long)s.end, r0 + g.rows);
    }
    const int c = (blockIdx.x * 32 + (threadIdx.x & 31)) * W, n = g.N - c;
    const T *dy = reinterpret_cast<const T *>(g.dy) + c, *z = reinterpret_cast<const T *>(g.z) + c;
    T *dz = reinterpret_cast<T *>(g.dz) + c;
    float sum[W] = {};
    if (n > 0) {
        for (long long r = r0 + (threadIdx.x >> 5); r < r1; r += 8 * AT) {
            float v[AT][W], w[AT][W] = {};
#pragma unroll
            for (int k = 0; k < AT; ++k) {
                const int m = r + 8 * k < r1 && !tail ? n : 0;
                load_row<T, W>(dy + (m ? (r + 8 * k) * g.ldy : 0), c, m, v[k]);
                if (g.act != MDX_ACT_NONE) load_row<T, W>(z + (m ? (r + 8 * k) * g.ldz : 0), c, m, w[k]);
            }
#pragma unroll
            for (int k = 0; k < AT; ++k) {
                if (!tail) apply_act_grad<GATES<T>>(v[k], w[k], g.act);
                if (g.dz && r + 8 * k < r1) store_row<T, W>(dz + (r + 8 * k) * g.lddz, n, v[k]);
#pragma unroll
                for (int q = 0; q < W; ++q) sum[q] += v[k][q];
            }
        }
    }
    if (!g.part || tail) return;
    __shared__ float sh[8][32 * W];
#pragma unroll
    for (int q = 0; q < W; ++q) sh[threadIdx.x >> 5][(threadIdx.x & 31) * W + q] = sum[q];
    __syncthreads();
    for (int k = threadIdx.x; k < 32 * W; k += 256) {
        const int col = blockIdx.x * 32 * W + k;
        float v = sh[0][k];
#pragma unroll
        for (int w = 1; w < 8; ++w) v += sh[w][k];
        if (col < g.N) g.part[(long long)blockIdx.y * g.N + col] = v;
    }
}
// ---- host ---------------------------------------------------------------
constexpr int CUS = 256;  // of an MI355X
// a launch has fewer than 2^32 threads
static bool fits(long long blocks, int threads) { return blocks * threads < (1ll << 32); }

struct Shape {
    long long T;  // rows
    int E, N, K;  // E = 0: dense
    int dtype, act;
    int es() const { return dtype == 0 ? 4 : 2; }
};

// A product as the choice of kernel sees it: its output, the length of its
// reduction, and how many of it there are (grouped: on average).
struct Load {
    long long I, J, R, groups;
    bool red, ragged, split;  // grouped reduction; grouped rows; the reduction may be split
};                            // (of two, the first may be)
struct Choice {
    int kind, splits;  // splits of each load that may be split
    double us;
};
// Microseconds of a step of 128 bytes for a tile alone on its CU, and for each
// of several that share it; of a tile beside its steps; tiles that fit on a CU.
// Measured on square layers of whole tiles (2048 x 2048, 1024 x 1024; reductions
// of 512 and 4096).
struct Cost {
    double alone, shared, fixed;
    int slots;
};
static Cost cost_of(int kind, int es) {
    switch (kind) {
        case LARGE: return {1.3, 1.3, 12.0, 1};
        case DMA128: return es == 4 ? Cost{2.05, 1.9, 8.0, 2} : Cost{0.62, 0.62, 7.0, 1};
        case DMA64: return es == 4 ? Cost{0.65, 0.55, 5.0, 2} : Cost{0.28, 0.175, 4.0, 2};
        case REG128: return es == 4 ? Cost{2.2, 2.0, 8.0, 2} : Cost{1.2, 0.8, 5.0, 2};
        default: return es == 4 ? Cost{0.8, 0.57, 5.0, 4} : Cost{0.6, 0.35, 3.5, 4};
    }
}
// The kernel for one launch of all of `loads`, and the slices of their
// reductions: the least estimate of the rounds in which the CUs work through
// the tiles, and of the join.  (1000 x 1024 x 12544: fp32 128-wide tiles in 8
// slices 205 us, in 4 216, 64-wide in 2 222; bf16 64-wide in 2 slices 46, 128-wide
// in 4 47, 256-wide in 8 51.)
// A kernel whose launch would have too many threads is left out: narrow outputs
// of more than 5e8 rows go to larger tiles than their work asks for.
static Choice choose(const Load *loads, int n, int es, bool aligned, long long most_part) {
    Choice best{REG64, 1, 1e30};
    for (int kind = aligned ? (es == 2 ? LARGE : DMA128) : REG128; kind <= (aligned ? DMA64 : REG64); ++kind) {
        const Cost c = cost_of(kind, es);
        const int side = tile_side(kind);
        for (const int splits : {1, 2, 3, 4, 6, 8, 12, 16}) {
            long long tiles[2], steps[2], all = 0, part = 0, most = 0;
            bool enough = true;  // steps in a slice
            for (int k = 0; k < n; ++k) {
                const Load &l = loads[k];
                const int s = l.split ? splits : 1;
                steps[k] = std::max<long long>(1, ceil_div(ceil_div(l.R * es, 128), s));
                if (s > 1 && steps[k] < 4) enough = false;
                tiles[k] = ceil_div(l.I, side) * ceil_div(l.J, side) * l.groups * s;
                all += tiles[k];
                most += l.ragged ? (ceil_div(l.I * l.groups, side) + l.groups + 1) * ceil_div(l.J, side) : tiles[k];
                if (s > 1) part += 4 * s * l.I * l.J * (l.red ? l.groups : 1);
            }
            if (!enough || part > most_part || !fits(most, tile_threads(kind))) break;
            const long long here = std::min<long long>(c.slots, std::max<long long>(1, ceil_div(all, CUS)));
            const double step = std::max(c.alone, here * c.shared);
            double work = 0, longest = 0;
            for (int k = 0; k < n; ++k) {
                const double t = (double)steps[k] * step + c.fixed;
                work += (double)tiles[k] * t;
                longest = std::max(longest, t);
            }
            const double rounds = std::max(1.0, std::ceil(work / (longest * (double)(CUS * here)) - 0.02));
            const double us = rounds * longest + (part > 0 ? 5.0 + (double)part / 4e6 : 0.0);
            if (us < 0.98 * best.us) best = Choice{kind, splits, us};
            if (!loads[0].split || all >= 8ll * CUS * c.slots) break;  // enough tiles as it is
        }
    }
    return best;
}
static Load forward_load(const Shape &p) {
    const long long E = std::max(p.E, 1);
    return Load{ceil_div(p.T, E), p.N, p.K, E, false, p.E > 0, p.E == 0};
}
// bytes of partial sums of a forward call; nothing in grouped ones is split
static long long part_bytes(long long splits, long long E, long long I, long long J) {
    return splits > 1 ? splits * std::max<long long>(E, 1) * I * J * 4 : 0;
}
constexpr long long PART_MAX = 1ll << 30;

// rows of a chunk of k_act_backward: about eight workgroups for each CU
static int act_rows(long long T, int N, int dtype) {
    const long long cols = ceil_div(N, dtype == 0 ? 128 : 256);
    return (int)std::max<long long>(32, ceil_div(T * cols / 2048, 32) * 32);
}
// chunks of T rows in E groups (0: dense), and the rows behind them
static long long act_chunks(int E, long long T, int rows) {
    return std::max<long long>(1, ceil_div(T, rows)) + (E ? E + 1 : 0);
}

// whether an operand can be taken in aligned pieces of 16 bytes: r its
// reduction (or its rows' length where that is i or j)
static bool pieces(const void *p, long long ld, long long group, long long length, int es) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld * es % 16 == 0 && group * es % 16 == 0 &&
           length * es % 16 == 0 && ld < (1ll << 22);
}
// tiles of a product as run in its launch; grouped rows: a bound, with one
// partial tile more for each group and for the rows behind them
static int set_tiles(Args &g, int mode, int bi, int bj, int threads, long long &n) {
    const long long ti = ceil_div(g.I, bi) + (mode == GROUP_ROWS ? g.E + 1 : 0), tj = ceil_div(g.J, bj);
    n = ti * tj * (mode == GROUP_RED ? g.E : 1) * g.splits;
    MDX_REQUIRE(fits(n, threads), "mdx_linear: too many output tiles");
    g.ti = (int)ti;
    g.tj = (int)tj;
    return MDX_OK;
}
template <typename T, bool GROUP> static int launch_join(const Args &g, hipStream_t s) {
    const dim3 grid((unsigned)ceil_div(g.I * ceil_div(g.J, VEC<T>), 256), GROUP ? g.E : 1);
    hipLaunchKernelGGL(k_product_join<T>, grid, dim3(256), 0, s, g);
    MDX_CHECK_LAUNCH("mdx_linear");
    return MDX_OK;
}
template <typename T, int MODE, int KIND> static int launch_forward(Args g, hipStream_t s) {
    if constexpr (KIND == LARGE && sizeof(T) == 4) return MDX_EINVAL;
    else {
        long long n;
        if (int rc = set_tiles(g, MODE, tile_side(KIND), tile_side(KIND), tile_threads(KIND), n)) return rc;
        hipLaunchKernelGGL((k_forward<T, MODE, KIND>), dim3((unsigned)n), dim3(tile_threads(KIND)), tile_lds<T>(KIND), s,
                           g);
        MDX_CHECK_LAUNCH("mdx_linear");
        return g.splits > 1 ? launch_join<T, false>(g, s) : MDX_OK;
    }
}
// w, x: dW's and dx's product, their pointer out null where not needed; db: the
// bias's gradient from the sums of `sums`, or null
template <typename T, bool GROUPED, int KIND>
static int launch_backward(Args w, Args x, const ActArgs &sums, float *db, hipStream_t s) {
    if constexpr (KIND == LARGE && sizeof(T) == 4) return MDX_EINVAL;
    else {
        long long nw = 0, nx = 0;
        constexpr int side = tile_side(KIND), threads = tile_threads(KIND);
        if (w.out)
            if (int rc = set_tiles(w, GROUPED ? GROUP_RED : DENSE, side, side, threads, nw)) return rc;
        if (x.out)
            if (int rc = set_tiles(x, GROUPED ? GROUP_ROWS : DENSE, side, side, threads, nx)) return rc;
        const long long nb = db ? ceil_div(bias_units(sums), BIAS_UNITS) : 0;
        MDX_REQUIRE(fits(nw + nx + nb, threads), "mdx_linear_backward: too many output tiles");
        // without both, or with more groups than a wave has lanes: dW's first
        const int first = !w.out || !x.out ? (int)nw
                          : GROUPED        ? w.E <= 64 ? -1 : (int)nw
                                           : w.R > x.R * w.splits ? (int)nw : 0;
        hipLaunchKernelGGL((k_backward<T, GROUPED, KIND>), dim3((unsigned)(nw + nx + nb)), dim3(threads),
                           tile_lds<T>(KIND), s, w, (int)nw, (int)nx, first, x, sums, db);
        MDX_CHECK_LAUNCH("mdx_linear_backward");
        return w.out && w.splits > 1 ? launch_join<T, GROUPED>(w, s) : MDX_OK;
    }
}

// Few rows to a group: 16 of them in a tile, or 32 (dense); 32 columns where that still
// gives every CU a few workgroups, else 16 and slices of the reduction until
// every CU has one; 4, 8 or 16 waves to a slice of it.
struct Few {
    int mt, nt, splits, waves;
};
static Few few_plan(long long rows, int E, long long N, long long K, int es) {
    Few f{rows <= 16 ? 1 : 2, 1, 1, 4};
    const long long chunks = ceil_div(K * es, 128), live = std::max(E, 1);
    if (ceil_div(N, 32) * live >= 4 * CUS) f.nt = 2;
    const long long tiles = ceil_div(N, 16 * f.nt) * live;
    if (!E) f.splits = (int)std::max<long long>(1, std::min<long long>(std::min(CUS / tiles, chunks / 32), 8));
    const long long each = ceil_div(chunks, f.splits);
    f.waves = each >= 64 && tiles * f.splits <= 2 * CUS ? 16 : each >= 32 ? 8 : 4;
    return f;
}
template <typename T, int MODE, int MT, int NT> static int launch_few(Args g, int waves, hipStream_t s) {
    long long n;
    if (int rc = set_tiles(g, MODE, 16 * MT, 16 * NT, 64 * waves, n)) return rc;
    const dim3 grid((unsigned)n);
    switch (waves) {
        case 16: hipLaunchKernelGGL((k_product_few<T, MODE, MT, NT, 16>), grid, dim3(1024), 0, s, g); break;
        case 8: hipLaunchKernelGGL((k_product_few<T, MODE, MT, NT, 8>), grid, dim3(512), 0, s, g); break;
        default: hipLaunchKernelGGL((k_product_few<T, MODE, MT, NT, 4>), grid, dim3(256), 0, s, g);
    }
    MDX_CHECK_LAUNCH("mdx_linear");
    return g.splits > 1 ? launch_join<T, false>(g, s) : MDX_OK;
}

static int check_shape(const char *fn, const Shape &p) {
    MDX_REQUIRE(p.dtype == 0 || p.dtype == 1 || p.dtype == 3, "%s: dtype must be 0 (f32), 1 (f16) or 3 (bf16)", fn);
    MDX_REQUIRE(p.act >= MDX_ACT_NONE && p.act <= MDX_ACT_SILU, "%s: unknown activation %d", fn, p.act);
    // positions in a row or column, and a few steps behind them, are 32-bit
    constexpr int most = INT32_MAX - (1 << 16);
    MDX_REQUIRE(p.T >= 0 && p.T <= most && p.N > 0 && p.N <= most && p.K > 0 && p.K <= most, "%s: bad shape", fn);
    MDX_REQUIRE(p.E >= 0 && p.E <= 4096, "%s: 1 to 4096 groups", fn);
    return MDX_OK;
}
static bool bad_ld(const void *p, long long ld, long long width) { return p && ld < width; }

// Whether k_product_few takes a forward call.  It reads weights faster than the
// tiles do, and multiplies slower.  Dense: up to 32 rows (bf16 4096 x 4096: 1 row
// 8.0 us against 12.0, 32 rows 14.1 against 14.9; fp32 14.5 against 29, 25 against
// 29).  Of fp32 groups up to 16 rows each on average (8 x 4096 x 1024: 8 rows 29
// us against 42, 20 rows 43 against 43).  The tiles of 16-bit groups fill the CUs
// between them, so there the few take over with the length of the reduction, a
// row for each 16 steps of 128 bytes (8 x 4096 x 1024: 1 row 10.4 us against 10.7,
// 4 rows 13.5 against 14.1, 8 rows 17.5 against 14.9; 8 x 1024 x 4096: 4 rows 17
// against 22, 16 rows 28 against 22; 4 x 1024 x 12544: 8 rows 23 against 59, 16
// rows 48 against 59), and for each 64 where they are unaligned (8 x 4096 x 1023:
// 1 row 26 us against 19; 8 x 1023 x 4095: 1 row 39 against 45, 4 rows 48 against
// 45).
static bool few_rows(const Shape &p, bool aligned) {
    if (!p.E) return p.T <= 32;
    if (p.dtype == 0) return p.T <= 16ll * p.E;
    const long long steps = ceil_div((long long)p.K * p.es(), 128);
    return p.T <= 16ll * p.E && p.T * (aligned ? 16 : 64) <= steps * p.E;
}
// how a forward call is computed
struct Plan {
    bool few;
    Few f;
    Choice c;
    int splits() const { return few ? f.splits : c.splits; }
};
static Plan plan_forward(const Shape &p, bool aligned, long long most_part) {
    Plan q{few_rows(p, aligned), {}, {}};
    if (q.few) {
        q.f = few_plan(ceil_div(p.T, std::max(p.E, 1)), p.E, p.N, p.K, p.es());
        if (part_bytes(q.f.splits, 0, p.T, p.N) > most_part) q.f.splits = 1;
        // of some 5e8 columns or more the tiles need fewer threads
        const long long ti = p.E ? ceil_div(p.T, 16) + p.E + 1 : ceil_div(p.T, 16 * q.f.mt);
        q.few = fits(ti * ceil_div(p.N, 16 * q.f.nt) * q.f.splits, 64 * q.f.waves);
    }
    if (!q.few) {
        const Load l = forward_load(p);
        q.c = choose(&l, 1, p.es(), aligned, most_part);
    }
    return q;
}
template <typename T, int MODE> static int forward(const Shape &p, Args g, int64_t ws_bytes, hipStream_t s) {
    const int es = sizeof(T);
    const bool al = pieces(g.a, g.lda, 0, g.R, es) && pieces(g.b, g.ldb, g.gstride, g.R, es);
    Plan q = plan_forward(p, al, PART_MAX);
    // without room for the slices of that plan the reduction is not split at all,
    // so that the result does not follow the workspace's size any closer
    if (q.splits() > 1 && (!g.part || ws_bytes < part_bytes(q.splits(), 0, p.T, p.N))) q = plan_forward(p, al, 0);
    g.splits = q.splits();
    if (q.few) {
        if constexpr (MODE == DENSE)
            if (q.f.mt == 2)
                return q.f.nt == 1 ? launch_few<T, MODE, 2, 1>(g, q.f.waves, s) : launch_few<T, MODE, 2, 2>(g, q.f.waves, s);
        return q.f.nt == 1 ? launch_few<T, MODE, 1, 1>(g, q.f.waves, s) : launch_few<T, MODE, 1, 2>(g, q.f.waves, s);
    }
    switch (q.c.kind) {
        case LARGE: return launch_forward<T, MODE, LARGE>(g, s);
        case DMA128: return launch_forward<T, MODE, DMA128>(g, s);
        case DMA64: return launch_forward<T, MODE, DMA64>(g, s);
        case REG128: return launch_forward<T, MODE, REG128>(g, s);
        default: return launch_forward<T, MODE, REG64>(g, s);
    }
}
// room for the split that either kind of kernel chooses, aligned operands or not
static long long forward_bytes(const Shape &p) {
    if (p.E) return 0;
    long long n = 0;
    for (int al = 0; al < 2; ++al) n = std::max(n, part_bytes(plan_forward(p, al, PART_MAX).splits(), 0, p.T, p.N));
    return n;
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
    bool dz;           // dz is kept in the workspace
    int rows;          // of a chunk of the elementwise pass
    Choice products;
    long long dz_bytes, part_bytes, dw_bytes;
};
static long long up256(long long n) { return (n + 255) / 256 * 256; }
static BackPlan plan_backward(const Shape &p, bool need_x, bool need_w, bool need_b, bool need_r, bool aligned) {
    BackPlan q{};
    const long long E = std::max(p.E, 1);
    // chosen for both products whichever are needed, so that a gradient's bits
    // do not depend on which others are asked for
    const Load l[2] = {Load{p.N, p.K, ceil_div(p.T, E), E, true, false, true},
                       Load{ceil_div(p.T, E), p.K, p.N, E, false, p.E > 0, false}};
    q.products = choose(l, 2, p.es(), aligned, PART_MAX);
    q.dz = p.act != MDX_ACT_NONE && (need_x || need_w) && !need_r;
    q.rows = act_rows(p.T, p.N, p.dtype);
    q.dz_bytes = q.dz ? up256(p.T * p.N * p.es()) : 0;
    q.part_bytes = need_b ? up256(act_chunks(p.E, p.T, q.rows) * p.N * 4) : 0;
    q.dw_bytes = need_w ? up256(part_bytes(q.products.splits, p.E, p.N, p.K)) : 0;
    return q;
}
// room for what either kind of kernel chooses, aligned operands or not
static long long backward_bytes(const Shape &p, bool need_x, bool need_w, bool need_b, bool need_r) {
    long long n = 0;
    for (int al = 0; al < 2; ++al) {
        const BackPlan q = plan_backward(p, need_x, need_w, need_b, need_r, al);
        n = std::max(n, q.dz_bytes + q.part_bytes + q.dw_bytes);
    }
    return n;
}

template <typename T, bool GROUPED>
static int backward(const char *fn, const Shape &p, const Back &b, int64_t ws_bytes, hipStream_t s) {
    const int es = sizeof(T);
    // dz as the products take it; its rows in the workspace lie N apart
    const bool kept = p.act != MDX_ACT_NONE;
    const void *dz = !kept ? b.grad : b.dres ? b.dres : b.ws;
    const long long lddz = !kept ? b.ldg : b.dres ? b.lddr : p.N;
    const bool al = pieces(dz, lddz, 0, p.N, es) && pieces(b.x, b.ldx, 0, p.K, es) &&
                    pieces(b.w, b.ldw, (long long)p.N * b.ldw, p.K, es);
    MDX_REQUIRE(!b.db || ceil_div(p.N, 16) * std::max(p.E, 1) < (1 << 23), "%s: too many columns of bias", fn);
    const BackPlan q = plan_backward(p, b.dx, b.dw, b.db, b.dres, al);
    const long long need = q.dz_bytes + q.part_bytes + q.dw_bytes;
    MDX_REQUIRE(reinterpret_cast<uintptr_t>(b.ws) % 16 == 0, "%s: the workspace must be 16-byte aligned", fn);
    MDX_REQUIRE(need == 0 || (b.ws && ws_bytes >= need), "%s: needs %lld bytes of workspace, got %lld", fn, need,
                (long long)ws_bytes);
    ActArgs a{};
    if (q.dz || b.db || b.dres) {
        a.dy = b.grad; a.ldy = b.ldg;
        a.z = b.pre; a.ldz = b.ldp;
        a.dz = b.dres ? b.dres : q.dz ? b.ws : nullptr;
        a.lddz = b.dres ? b.lddr : p.N;
        a.part = b.db ? reinterpret_cast<float *>(b.ws + q.dz_bytes) : nullptr;
        a.counts = b.counts;
        a.E = p.E; a.T = p.T; a.N = p.N; a.act = p.act;
        a.rows = q.rows;
        a.zero_tail = b.dres && b.zero_tail;
        const dim3 grid((unsigned)ceil_div(p.N, 32 * VEC<T>), (unsigned)act_chunks(p.E, p.T, q.rows));
        hipLaunchKernelGGL(k_act_backward<T>, grid, dim3(256), 0, s, a);
        MDX_CHECK_LAUNCH("mdx_linear_backward");
    }
    Args w{}, x{};
    w.splits = x.splits = 1;
    if (b.dw) {
        w.a = dz; w.lda = lddz;
        w.b = b.x; w.ldb = b.ldx;
        w.I = p.N; w.J = p.K; w.R = p.T;
        w.out = b.dw; w.ldo = b.lddw;
        w.counts = b.counts; w.E = p.E; w.T = p.T;
        w.gstride = (long long)p.N * b.lddw;
        w.splits = q.products.splits;
        w.part = reinterpret_cast<float *>(b.ws + q.dz_bytes + q.part_bytes);
    }
    if (b.dx && p.T) {
        x.a = dz; x.lda = lddz;
        x.b = b.w; x.ldb = b.ldw;
        x.I = p.T; x.J = p.K; x.R = p.N;
        x.out = b.dx; x.ldo = b.lddx;
        x.counts = b.counts; x.E = p.E; x.T = p.T;
        x.gstride = (long long)p.N * b.ldw;
        x.zero_tail = b.zero_tail;
    }
    if (!w.out && !x.out) {
        if (b.db) {
            hipLaunchKernelGGL(k_bias_join, dim3((unsigned)bias_units(a)), dim3(256), 0, s, a, b.db);
            MDX_CHECK_LAUNCH("mdx_linear_backward");
        }
        return MDX_OK;
    }
    switch (q.products.kind) {
        case LARGE: return launch_backward<T, GROUPED, LARGE>(w, x, a, b.db, s);
        case DMA128: return launch_backward<T, GROUPED, DMA128>(w, x, a, b.db, s);
        case DMA64: return launch_backward<T, GROUPED, DMA64>(w, x, a, b.db, s);
        case REG128: return launch_backward<T, GROUPED, REG128>(w, x, a, b.db, s);
        default: return launch_backward<T, GROUPED, REG64>(w, x, a, b.db, s);
    }
}

template <typename T> static int forward_any(const Shape &p, const Args &g, int64_t ws_bytes, hipStream_t s) {
    return p.E ? forward<T, GROUP_ROWS>(p, g, ws_bytes, s) : forward<T, DENSE>(p, g, ws_bytes, s);
}
template <typename T>
static int backward_any(const char *fn, const Shape &p, const Back &b, int64_t ws_bytes, hipStream_t s) {
    return p.E ? backward<T, true>(fn, p, b, ws_bytes, s) : backward<T, false>(fn, p, b, ws_bytes, s);
}
static int run_forward(const char *fn, const Shape &p, const Args &g, int64_t ws_bytes, hipStream_t s) {
    MDX_REQUIRE(g.a && g.b && g.out, "%s: null pointer", fn);
    MDX_REQUIRE(reinterpret_cast<uintptr_t>(g.part) % 16 == 0, "%s: the workspace must be 16-byte aligned", fn);
    MDX_REQUIRE(!bad_ld(g.a, g.lda, p.K) && !bad_ld(g.b, g.ldb, p.K) && !bad_ld(g.res, g.ldr, p.N) &&
                    !bad_ld(g.pre, g.ldp, p.N) && !bad_ld(g.out, g.ldo, p.N),
                "%s: a row stride is below its row's length", fn);
    switch (p.dtype) {
        case 0: return forward_any<float>(p, g, ws_bytes, s);
        case 1: return forward_any<_Float16>(p, g, ws_bytes, s);
        default: return forward_any<__bf16>(p, g, ws_bytes, s);
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
    switch (p.dtype) {
        case 0: return backward_any<float>(fn, p, b, ws_bytes, s);
        case 1: return backward_any<_Float16>(fn, p, b, ws_bytes, s);
        default: return backward_any<__bf16>(fn, p, b, ws_bytes, s);
    }
}

}  // namespace lin
}  // namespace mdx

using namespace mdx;
using namespace mdx::lin;

extern "C" int64_t mdx_linear_workspace_bytes(int64_t M, int N, int K, int dtype) {
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    return forward_bytes(Shape{M, 0, N, K, dtype, 0});
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
    g.part = reinterpret_cast<float *>(workspace);
    return run_forward("mdx_linear", p, g, workspace_bytes, as_stream(stream));
}

extern "C" int mdx_linear_plan(int E, int64_t T, int N, int K, int dtype, int aligned, int backward) {
    const Shape p{T, E, N, K, dtype, 0};
    if (int rc = check_shape("mdx_linear_plan", p)) return rc;
    if (backward) {
        const Choice c = plan_backward(p, true, true, false, false, aligned).products;
        return c.kind + 16 * c.splits;
    }
    const Plan q = plan_forward(p, aligned, PART_MAX);
    return (q.few ? MDX_LINEAR_FEW : q.c.kind) + 16 * q.splits();
}

extern "C" int64_t mdx_linear_backward_workspace_bytes(int64_t M, int N, int K, int act, int dtype, int need_x,
                                                       int need_w, int need_bias, int need_residual) {
    if (M < 0 || N <= 0 || K <= 0) return 0;
    return backward_bytes(Shape{M, 0, N, K, dtype, act}, need_x, need_w, need_bias, need_residual);
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
    return run_forward("mdx_grouped_linear", p, g, 0, as_stream(stream));
}

extern "C" int64_t mdx_grouped_linear_backward_workspace_bytes(int E, int64_t T, int N, int K, int act, int dtype,
                                                               int need_x, int need_w, int need_bias,
                                                               int need_residual) {
    if (E <= 0 || T < 0 || N <= 0 || K <= 0) return 0;
    return backward_bytes(Shape{T, E, N, K, dtype, act}, need_x, need_w, need_bias, need_residual);
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
