// Layer norm over the last axis, forward and backward (include/mdx.h:
// mdx_layer_norm*).
//
//   mean = sum x / D,  rstd = 1 / sqrt(sum (x - mean)^2 / D + eps)
//   h = (x - mean) rstd,  y = h g + b
//   dx = rstd (dy g - mean(dy g) - h mean(dy g h)),  dg = sum_rows dy h,  db = sum_rows dy
//
// Both are bound by HBM: a row is read once into registers, its sums are taken
// there in float32 (the variance in a second pass over the registers, around
// the mean), and the result is written once.  Rows wider than the registers
// of a workgroup hold are read again instead (k_norm_wide*).
#include "pieces.h"

#include <algorithm>

namespace mdx {
namespace norm {

template <typename T> struct Piece {
    union { u4 u; T e[VEC<T>]; };
};
template <typename T> __device__ __forceinline__ Piece<T> load(const T *p, int c, int n) {
    Piece<T> r;
    r.u = load_piece(p, c, n);
    return r;
}
template <typename T> __device__ __forceinline__ void store(T *p, const Piece<T> &v, int n) {
    if (n >= VEC<T>) {
        reinterpret_cast<Un16<T> *>(p)->v = v.u;
        return;
    }
#pragma unroll
    for (int q = 0; q < VEC<T>; ++q)
        if (q < n) p[q] = v.e[q];
}

struct Args {
    const void *x, *dy;
    long long ldx, ldy;
    const float *gamma, *beta;  // [D] or null
    long long rows;
    int D;
    float eps;
    void *out;                  // y or dx, or null
    long long ldo;
    float *mean, *rstd;         // [rows]: written forward (or null), read backward
    float *part;                // backward: [workgroups][2][D] partial dg, db, or null
};

// Sums over the TPR threads of a row (TPR <= 64: lanes of a wave; above: the
// workgroup, through LDS), which every thread gets.  Within 16 lanes the adds
// take their operand from another lane directly (DPP); N sums go side by side,
// so that their latencies overlap.
template <int CTRL> __device__ __forceinline__ float dpp_add(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int TPR, int N> __device__ __forceinline__ void row_sums(float (&v)[N], float *sh) {
#pragma unroll
    for (int k = 0; k < N; ++k) {
        v[k] = dpp_add<0xB1>(v[k]);   // lanes 1, 0, 3, 2 of each four
        v[k] = dpp_add<0x4E>(v[k]);   // 2, 3, 0, 1
        v[k] = dpp_add<0x141>(v[k]);  // mirrored in 8
        v[k] = dpp_add<0x140>(v[k]);  // mirrored in 16
    }
#pragma unroll
    for (int d = 16; d < (TPR < 64 ? TPR : 64); d <<= 1)
#pragma unroll
        for (int k = 0; k < N; ++k) v[k] += __shfl_xor(v[k], d);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        __syncthreads();  // the sums before these have been read
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < N; ++k) sh[k * W + (threadIdx.x >> 6)] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < N; ++k) {
            v[k] = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) v[k] += sh[k * W + w];
        }
    }
}
template <int TPR> __device__ __forceinline__ float row_sum(float v, float *sh) {
    float s[1] = {v};
    row_sums<TPR>(s, sh);
    return s[0];
}

// TPR threads hold a row in NP pieces of 16 bytes each.  fetch() brings them as
// they lie in memory, of the row's end where a piece passes it, so that nothing
// waits for them; take() gives one as floats, zeros behind the row.  Rows
// shorter than a piece are finished in fetch() (`tiny`).
template <typename T, int TPR, int NP> struct Rows {
    static constexpr int THREADS = TPR > 256 ? TPR : 256, ROWS = THREADS / TPR, V = VEC<T>;
    int t, D;
    bool tiny;
    __device__ __forceinline__ Rows(int d) : t(threadIdx.x % TPR), D(d), tiny(d < V) {}
    __device__ __forceinline__ int column(int p) const { return (p * TPR + t) * V; }
    __device__ __forceinline__ void fetch(const T *row, u4 (&v)[NP]) const {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const int c = column(p);
            v[p] = tiny ? load(row, 0, c ? 0 : D).u : reinterpret_cast<const Un16<T> *>(row + min(c, D - V))->v;
        }
    }
    __device__ __forceinline__ void take(u4 u, int p, float (&v)[V]) const {
        const int n = D - column(p);
        if (n < V && !tiny) u = n > 0 ? shift_down(u, (V - n) * 8 * (int)sizeof(T)) : u4{0, 0, 0, 0};
        Piece<T> w;
        w.u = u;
#pragma unroll
        for (int q = 0; q < V; ++q) v[q] = (float)w.e[q];
    }
    // gamma or beta of the thread's columns; `none` where there is none
    __device__ __forceinline__ void params(const float *g, float none, float (&v)[NP][V]) const {
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            const int c = column(p);
            if (g && c + V <= D) {
                Un16<float> w[V / 4];
#pragma unroll
                for (int q = 0; q < V / 4; ++q) w[q] = *reinterpret_cast<const Un16<float> *>(g + c + 4 * q);
#pragma unroll
                for (int q = 0; q < V; ++q) v[p][q] = __uint_as_float(w[q / 4].v[q % 4]);
            } else {
#pragma unroll
                for (int q = 0; q < V; ++q) v[p][q] = g && c + q < D ? g[c + q] : none;
            }
        }
    }
};

// The next row of a thread is on its way while it works on one.  Bound by HBM:
// bf16 458752 x 256 98 us (4.8 TB/s), 32000 x 1024 22 (6.0 TB/s, in part from the
// last-level cache), 8000 x 4096 23 (5.6); fp32 2000 x 12544 35 (5.8).
template <typename T, int TPR, int NP>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_norm(Args a) {
    using L = Rows<T, TPR, NP>;
    constexpr int V = L::V;
    __shared__ float sh[16];
    const L l(a.D);
    const int slot = threadIdx.x / TPR;
    const float inv = 1.f / (float)a.D;
    const T *X = reinterpret_cast<const T *>(a.x);
    const long long stride = (long long)gridDim.x * L::ROWS;
    long long r = (long long)blockIdx.x * L::ROWS + slot;
    u4 next[NP];
    l.fetch(X + min(r, a.rows - 1) * a.ldx, next);
    float g[NP][V], b[NP][V];
    l.params(a.gamma, 1.f, g);
    l.params(a.beta, 0.f, b);
    for (; r - slot < a.rows; r += stride) {
        float v[NP][V], s = 0.f;
#pragma unroll
        for (int p = 0; p < NP; ++p) l.take(next[p], p, v[p]);
        l.fetch(X + min(r + stride, a.rows - 1) * a.ldx, next);
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int q = 0; q < V; ++q) s += v[p][q];
        const float mean = row_sum<TPR>(s, sh) * inv;
        s = 0.f;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
#pragma unroll
            for (int q = 0; q < V; ++q) v[p][q] -= mean;
            if (l.column(p) + V > a.D)  // nothing behind the row
#pragma unroll
                for (int q = 0; q < V; ++q) v[p][q] = l.column(p) + q < a.D ? v[p][q] : 0.f;
#pragma unroll
            for (int q = 0; q < V; ++q) s += v[p][q] * v[p][q];
        }
        const float rstd = 1.f / sqrtf(row_sum<TPR>(s, sh) * inv + a.eps);
        if (r >= a.rows) continue;
        T *o = reinterpret_cast<T *>(a.out) + r * a.ldo;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            Piece<T> w;
#pragma unroll
            for (int q = 0; q < V; ++q) w.e[q] = (T)(v[p][q] * rstd * g[p][q] + b[p][q]);
            store(o + l.column(p), w, a.D - l.column(p));
        }
        if (l.t == 0) {
            if (a.mean) a.mean[r] = mean;
            if (a.rstd) a.rstd[r] = rstd;
        }
    }
}

// dx, and each workgroup's share of dg and db: a thread keeps the sums of its
// columns over all rows it takes; the row slots are added through LDS at the
// end.  Bound by HBM up to some 4000 columns (bf16 32000 x 1024 with the join 36 us,
// 5.4 TB/s; 458752 x 256 139, 5.1), beyond by one workgroup's latency from row
// to row: gamma, the sums and one row fill the registers, and nothing else runs
// on the CU meanwhile (2000 x 16384 70 us, 2.8 TB/s).
template <typename T, int TPR, int NP>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void k_norm_backward(Args a) {
    using L = Rows<T, TPR, NP>;
    constexpr int V = L::V;
    // of 32 columns to a thread the registers hold the sums and one row: gamma
    // is read again, and no second row is on its way
    constexpr bool KEEP = NP * V < 32, AHEAD = NP * V < 32;
    __shared__ float sh[32];
    __shared__ float cols[L::ROWS > 1 ? L::THREADS * NP * V : 1];
    const L l(a.D);
    const int slot = threadIdx.x / TPR;
    const float inv = 1.f / (float)a.D;
    const T *X = reinterpret_cast<const T *>(a.x), *DY = reinterpret_cast<const T *>(a.dy);
    const long long stride = (long long)gridDim.x * L::ROWS;
    long long r = (long long)blockIdx.x * L::ROWS + slot;
    u4 nx[NP], ny[NP];
    float nm = 0.f, nr = 0.f;
    auto fetch = [&](long long i) {
        const long long k = min(i, a.rows - 1);
        l.fetch(X + k * a.ldx, nx);
        l.fetch(DY + k * a.ldy, ny);
        nm = a.mean[k];
        nr = a.rstd[k];
    };
    if (AHEAD && a.rows > 0) fetch(r);
    float g[NP][V], dg[NP][V] = {}, db[NP][V] = {};
    if (KEEP) l.params(a.gamma, 1.f, g);
    for (; r - slot < a.rows; r += stride) {
        const bool live = r < a.rows;
        if (!AHEAD) fetch(r);
        // a row that is not there counts as zeros; behind a row dy is zero, so
        // that what x - mean gives there reaches no sum
        if (!live) {
            nm = nr = 0.f;
#pragma unroll
            for (int p = 0; p < NP; ++p) nx[p] = ny[p] = u4{0, 0, 0, 0};
        }
        const float mean = nm, rstd = nr;
        float h[NP][V], d[NP][V], s[2] = {};
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            l.take(nx[p], p, h[p]);
            l.take(ny[p], p, d[p]);
        }
        if (AHEAD) fetch(r + stride);
        if (!KEEP) l.params(a.gamma, 1.f, g);
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
            for (int q = 0; q < V; ++q) {
                h[p][q] = (h[p][q] - mean) * rstd;
                const float e = d[p][q];
                dg[p][q] += e * h[p][q];
                db[p][q] += e;
                d[p][q] = e * g[p][q];
                s[0] += d[p][q];
                s[1] += d[p][q] * h[p][q];
            }
        if (!a.out) continue;
        row_sums<TPR>(s, sh);
        s[0] *= inv;
        s[1] *= inv;
        if (!live) continue;
        T *o = reinterpret_cast<T *>(a.out) + r * a.ldo;
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            Piece<T> w;
#pragma unroll
            for (int q = 0; q < V; ++q) w.e[q] = (T)(rstd * (d[p][q] - s[0] - h[p][q] * s[1]));
            store(o + l.column(p), w, a.D - l.column(p));
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        float *o = a.part + ((long long)blockIdx.x * 2 + k) * a.D;
        if constexpr (L::ROWS > 1) {
            __syncthreads();
#pragma unroll
            for (int p = 0; p < NP; ++p)
#pragma unroll
                for (int q = 0; q < V; ++q) cols[slot * TPR * NP * V + l.column(p) + q] = k ? db[p][q] : dg[p][q];
            __syncthreads();
            for (int c = threadIdx.x; c < TPR * NP * V && c < a.D; c += L::THREADS) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < L::ROWS; ++w) v += cols[w * TPR * NP * V + c];
                o[c] = v;
            }
        } else {
#pragma unroll
            for (int p = 0; p < NP; ++p)
#pragma unroll
                for (int q = 0; q < V; ++q) {
                    const int c = l.column(p) + q;
                    if (c < a.D) o[c] = k ? db[p][q] : dg[p][q];
                }
        }
    }
}

// Any width: a workgroup of 1024 reads its row once for each sum and once to
// write.  A row is still in the L2 when it is read again; what bounds it is the
// chain of three passes (bf16 2000 x 32768 246 us, 1.1 TB/s; backward 366).
template <typename T> __global__ __launch_bounds__(1024) void k_norm_wide(Args a) {
    constexpr int V = VEC<T>;
    __shared__ float sh[16];
    const long long r = blockIdx.x;
    const T *x = reinterpret_cast<const T *>(a.x) + r * a.ldx;
    T *o = reinterpret_cast<T *>(a.out) + r * a.ldo;
    float s = 0.f;
    for (long long c = threadIdx.x * V; c < a.D; c += 1024 * V) {
        const Piece<T> w = load(x + c, (int)c, (int)(a.D - c));
#pragma unroll
        for (int q = 0; q < V; ++q) s += (float)w.e[q];
    }
    const float mean = row_sum<1024>(s, sh) / (float)a.D;
    s = 0.f;
    for (long long c = threadIdx.x * V; c < a.D; c += 1024 * V) {
        const Piece<T> w = load(x + c, (int)c, (int)(a.D - c));
#pragma unroll
        for (int q = 0; q < V; ++q) {
            const float d = c + q < a.D ? (float)w.e[q] - mean : 0.f;
            s += d * d;
        }
    }
    const float rstd = 1.f / sqrtf(row_sum<1024>(s, sh) / (float)a.D + a.eps);
    for (long long c = threadIdx.x * V; c < a.D; c += 1024 * V) {
        Piece<T> w = load(x + c, (int)c, (int)(a.D - c));
#pragma unroll
        for (int q = 0; q < V; ++q)
            if (c + q < a.D)
                w.e[q] = (T)(((float)w.e[q] - mean) * rstd * (a.gamma ? a.gamma[c + q] : 1.f) +
                             (a.beta ? a.beta[c + q] : 0.f));
        store(o + c, w, (int)(a.D - c));
    }
    if (threadIdx.x == 0) {
        if (a.mean) a.mean[r] = mean;
        if (a.rstd) a.rstd[r] = rstd;
    }
}
template <typename T> __global__ __launch_bounds__(1024) void k_norm_wide_backward(Args a) {
    constexpr int V = VEC<T>;
    __shared__ float sh[16];
    const long long r = blockIdx.x;
    const T *x = reinterpret_cast<const T *>(a.x) + r * a.ldx, *dy = reinterpret_cast<const T *>(a.dy) + r * a.ldy;
    T *o = reinterpret_cast<T *>(a.out) + r * a.ldo;
    const float mean = a.mean[r], rstd = a.rstd[r];
    float s1 = 0.f, s2 = 0.f;
    for (long long c = threadIdx.x * V; c < a.D; c += 1024 * V) {
        const Piece<T> w = load(x + c, (int)c, (int)(a.D - c)), y = load(dy + c, (int)c, (int)(a.D - c));
#pragma unroll
        for (int q = 0; q < V; ++q)
            if (c + q < a.D) {
                const float d = (float)y.e[q] * (a.gamma ? a.gamma[c + q] : 1.f);
                s1 += d;
                s2 += d * (((float)w.e[q] - mean) * rstd);
            }
    }
    s1 = row_sum<1024>(s1, sh) / (float)a.D;
    s2 = row_sum<1024>(s2, sh) / (float)a.D;
    for (long long c = threadIdx.x * V; c < a.D; c += 1024 * V) {
        const Piece<T> w = load(x + c, (int)c, (int)(a.D - c)), y = load(dy + c, (int)c, (int)(a.D - c));
        Piece<T> z = w;
#pragma unroll
        for (int q = 0; q < V; ++q)
            if (c + q < a.D) {
                const float d = (float)y.e[q] * (a.gamma ? a.gamma[c + q] : 1.f), h = ((float)w.e[q] - mean) * rstd;
                z.e[q] = (T)(rstd * (d - s1 - h * s2));
            }
        store(o + c, z, (int)(a.D - c));
    }
}
// dg and db of any width, from column `first` on: a workgroup takes 64 columns
// of one slice of the rows
template <typename T> __global__ __launch_bounds__(256) void k_norm_wide_sums(Args a, int first) {
    __shared__ float sh[2][256];
    const long long c = first + (long long)blockIdx.x * 64 + (threadIdx.x & 63);
    const long long per = (a.rows + gridDim.y - 1) / gridDim.y, r1 = min(a.rows, (blockIdx.y + 1) * per);
    float dg = 0.f, db = 0.f;
    if (c < a.D)
        for (long long r = blockIdx.y * per + (threadIdx.x >> 6); r < r1; r += 4) {
            const float e = (float)reinterpret_cast<const T *>(a.dy)[r * a.ldy + c];
            dg += e * (((float)reinterpret_cast<const T *>(a.x)[r * a.ldx + c] - a.mean[r]) * a.rstd[r]);
            db += e;
        }
    sh[0][threadIdx.x] = dg;
    sh[1][threadIdx.x] = db;
    __syncthreads();
    if (threadIdx.x < 128) {
        const int k = threadIdx.x >> 6, l = threadIdx.x & 63;
        const float v = sh[k][l] + sh[k][64 + l] + sh[k][128 + l] + sh[k][192 + l];
        if (c < a.D) a.part[((long long)blockIdx.y * 2 + k) * a.D + c] = v;
    }
}
// dg, db = the workgroups' shares, always added in the same order.  16 columns
// to a workgroup and 64 threads to each: a few loads in flight per thread and
// no chain of waits (64 columns and 16 threads to each took 11 us for 512
// shares of 1024 columns).  From column `first` on.
__global__ __launch_bounds__(1024) void k_norm_join(const float *part, int n, int D, float *dg, float *db, int first) {
    __shared__ float sh[16][16];
    const int l = threadIdx.x & 15, w = threadIdx.x >> 4, k = blockIdx.y;
    const long long c = first + (long long)blockIdx.x * 16 + l;
    float *o = k ? db : dg;
    if (!o) return;
    float v = 0.f;
    if (c < D)
        for (int s = w; s < n; s += 8 * 64) {
            float t[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) t[q] = s + 64 * q < n ? part[((long long)(s + 64 * q) * 2 + k) * D + c] : 0.f;
#pragma unroll
            for (int q = 0; q < 8; ++q) v += t[q];
        }
    v += __shfl_xor(v, 16);
    v += __shfl_xor(v, 32);
    if ((threadIdx.x & 63) < 16) sh[threadIdx.x >> 6][l] = v;
    __syncthreads();
    if (threadIdx.x < 16 && c < D) {
        v = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) v += sh[i][l];
        o[c] = v;
    }
}

// ---- host ---------------------------------------------------------------
// Columns of one launch where `per` threads work on each: a launch has fewer
// than 2^32 threads in each direction, so very wide rows (above 2^25 columns in
// k_norm_join, 2^29 in k_norm_wide_sums) take several.
static long long columns_of(int per) { return (1ll << 31) / per; }
// The layout of rows of D elements: the first of these that holds their pieces
// of 16 bytes, 0 for wider ones.  A thread's pieces stay in registers, forward
// next to gamma and beta, backward next to gamma and the sums of dg and db, so
// that backward has at most 256 registers' worth of threads to a row.
static int layout(int D, int dtype) {
    const long long pieces = ((long long)D * (dtype == 0 ? 4 : 2) + 15) / 16;
    const int cap[] = {16, 32, 64, 128, 192, 256, 512, 1024, 2048, 4096};
    for (int i = 0; i < (dtype == 0 ? 10 : 9); ++i)
        if (pieces <= cap[i]) return i + 1;
    return 0;
}
// workgroups of the backward pass, each with a share of dg and db
static int backward_groups(long long rows, int D, int dtype) {
    const int lay = layout(D, dtype);
    if (!lay) return (int)std::min<long long>(64, std::max<long long>(1, rows / 16));
    const int slots = lay == 1 ? 16 : lay == 2 ? 8 : lay <= (dtype == 0 ? 6 : 5) ? 4 : 1;  // rows at once
    const int most = lay <= 3 || (dtype != 0 && lay == 6) ? 1024 : lay <= 7 ? 512 : 256;
    // Each share is 8 bytes a column, written and read, so a workgroup should have
    // several rows; but few workgroups wait for one row after the other.  128 of
    // them, 256 where each still has 8 rows, more where each has 16 (bf16 200 x
    // 16384: 16 workgroups 55 us, 128 36, 200 39; 600 x 16384: 32 75, 128 45, 256 49,
    // 512 76; 2000 x 4096: 128 30, 256 24, 512 29; 8000 x 1500: 128 31, 256 22, 512 23).
    const long long want = std::max({128ll, std::min(256ll, rows / 8), rows / 16});
    return (int)std::max<long long>(1, std::min({(long long)ceil_div(rows, slots), (long long)most, want}));
}

template <typename T, int TPR, int NP> static void launch_forward(const Args &a, hipStream_t s) {
    using L = Rows<T, TPR, NP>;
    // as many as a CU holds: each takes gamma and beta once (4096 workgroups read
    // 32000 rows of 1024 in bf16 in 64 us, for the sake of their 8 KiB)
    const unsigned grid = (unsigned)std::min<long long>(ceil_div(a.rows, L::ROWS), 256 * 2048 / L::THREADS);
    hipLaunchKernelGGL((k_norm<T, TPR, NP>), dim3(grid), dim3(L::THREADS), 0, s, a);
}
template <typename T, int TPR, int NP> static void launch_backward(const Args &a, int groups, hipStream_t s) {
    hipLaunchKernelGGL((k_norm_backward<T, TPR, NP>), dim3(groups), dim3(Rows<T, TPR, NP>::THREADS), 0, s, a);
}
template <typename T> static void run_forward(const Args &a, int lay, hipStream_t s) {
    switch (lay) {
        case 1: return launch_forward<T, 16, 1>(a, s);
        case 2: return launch_forward<T, 32, 1>(a, s);
        case 3: return launch_forward<T, 64, 1>(a, s);
        case 4: return launch_forward<T, 64, 2>(a, s);
        case 5: return launch_forward<T, 64, 3>(a, s);
        case 6: return launch_forward<T, 256, 1>(a, s);
        case 7: return launch_forward<T, 256, 2>(a, s);
        case 8: return launch_forward<T, 1024, 1>(a, s);
        case 9: return launch_forward<T, 1024, 2>(a, s);
    }
    if constexpr (sizeof(T) == 4)
        if (lay == 10) return launch_forward<T, 1024, 4>(a, s);
    hipLaunchKernelGGL(k_norm_wide<T>, dim3((unsigned)a.rows), dim3(1024), 0, s, a);
}
template <typename T> static void run_backward(const Args &a, int lay, int groups, hipStream_t s) {
    switch (lay) {
        case 1: return launch_backward<T, 16, 1>(a, groups, s);
        case 2: return launch_backward<T, 32, 1>(a, groups, s);
        case 3: return launch_backward<T, 64, 1>(a, groups, s);
        case 4: return launch_backward<T, 64, 2>(a, groups, s);
        case 7: return launch_backward<T, 256, 2>(a, groups, s);
        case 9: return launch_backward<T, 512, 4>(a, groups, s);
    }
    if constexpr (sizeof(T) == 4) {
        if (lay == 5 || lay == 6) return launch_backward<T, 64, 4>(a, groups, s);
        if (lay == 8) return launch_backward<T, 256, 4>(a, groups, s);
        if (lay == 10) return launch_backward<T, 512, 8>(a, groups, s);
    } else {
        if (lay == 5) return launch_backward<T, 64, 3>(a, groups, s);
        if (lay == 6) return launch_backward<T, 256, 1>(a, groups, s);
        if (lay == 8) return launch_backward<T, 512, 2>(a, groups, s);
    }
    // the sums first: dx may be written over dy
    if (a.part)
        for (long long c = 0, n = columns_of(4); c < a.D; c += n)
            hipLaunchKernelGGL(k_norm_wide_sums<T>, dim3((unsigned)ceil_div(std::min(n, a.D - c), 64), groups), dim3(256), 0,
                               s, a, (int)c);
    if (a.out && a.rows)
        hipLaunchKernelGGL(k_norm_wide_backward<T>, dim3((unsigned)a.rows), dim3(1024), 0, s, a);
}
template <typename T> static int run(const char *fn, const Args &a, int dtype, bool back, float *dg, float *db,
                                     hipStream_t s) {
    const int groups = backward_groups(a.rows, a.D, dtype), lay = layout(a.D, dtype);
    if (back)
        run_backward<T>(a, lay, groups, s);
    else
        run_forward<T>(a, lay, s);
    MDX_CHECK_LAUNCH(fn);
    if (back && a.part) {
        for (long long c = 0, n = columns_of(64); c < a.D; c += n)
            hipLaunchKernelGGL(k_norm_join, dim3((unsigned)ceil_div(std::min(n, a.D - c), 16), 2), dim3(1024), 0, s, a.part,
                               groups, a.D, dg, db, (int)c);
        MDX_CHECK_LAUNCH(fn);
    }
    return MDX_OK;
}
static int dispatch(const char *fn, const Args &a, int dtype, bool back, float *dg, float *db, hipStream_t s) {
    switch (dtype) {
        case 0: return run<float>(fn, a, dtype, back, dg, db, s);
        case 1: return run<_Float16>(fn, a, dtype, back, dg, db, s);
        default: return run<__bf16>(fn, a, dtype, back, dg, db, s);
    }
}
static int check(const char *fn, int64_t rows, int D, int dtype) {
    MDX_REQUIRE(dtype == 0 || dtype == 1 || dtype == 3, "%s: dtype must be 0 (f32), 1 (f16) or 3 (bf16)", fn);
    MDX_REQUIRE(rows >= 0 && D > 0, "%s: bad shape", fn);
    // a workgroup of 1024 threads for each row there, and fewer than 2^32 threads in a launch
    MDX_REQUIRE(layout(D, dtype) || rows < (1 << 22), "%s: at most 2^22 - 1 rows of this width", fn);
    return MDX_OK;
}

}  // namespace norm
}  // namespace mdx

using namespace mdx;

extern "C" int mdx_layer_norm(const void *x, int64_t ldx, const float *gamma, const float *beta, int64_t rows, int D,
                              float eps, int dtype, void *out, int64_t ldo, float *mean, float *rstd,
                              mdx_stream_t stream) {
    if (int rc = norm::check("mdx_layer_norm", rows, D, dtype)) return rc;
    if (rows == 0) return MDX_OK;
    MDX_REQUIRE(x && out, "mdx_layer_norm: null pointer");
    MDX_REQUIRE(ldx >= D && ldo >= D, "mdx_layer_norm: a row stride is below its row's length");
    MDX_REQUIRE(eps >= 0.f, "mdx_layer_norm: eps must not be negative");
    norm::Args a{};
    a.x = x; a.ldx = ldx;
    a.gamma = gamma; a.beta = beta;
    a.rows = rows; a.D = D; a.eps = eps;
    a.out = out; a.ldo = ldo;
    a.mean = mean; a.rstd = rstd;
    return norm::dispatch("mdx_layer_norm", a, dtype, false, nullptr, nullptr, as_stream(stream));
}

extern "C" int64_t mdx_layer_norm_backward_workspace_bytes(int64_t rows, int D, int dtype) {
    if (rows < 0 || D <= 0) return 0;
    return (int64_t)norm::backward_groups(rows, D, dtype) * 2 * D * 4;
}
extern "C" int mdx_layer_norm_backward(const void *grad, int64_t ldg, const void *x, int64_t ldx, const float *mean,
                                       const float *rstd, const float *gamma, int64_t rows, int D, int dtype, void *dx,
                                       int64_t lddx, float *dgamma, float *dbeta, void *workspace,
                                       int64_t workspace_bytes, mdx_stream_t stream) {
    if (int rc = norm::check("mdx_layer_norm_backward", rows, D, dtype)) return rc;
    MDX_REQUIRE(rows == 0 || (grad && x && mean && rstd), "mdx_layer_norm_backward: null pointer");
    MDX_REQUIRE(ldg >= D && ldx >= D && (!dx || lddx >= D),
                "mdx_layer_norm_backward: a row stride is below its row's length");
    const int64_t need = dgamma || dbeta ? mdx_layer_norm_backward_workspace_bytes(rows, D, dtype) : 0;
    MDX_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0,
                "mdx_layer_norm_backward: the workspace must be 16-byte aligned");
    MDX_REQUIRE(need == 0 || (workspace && workspace_bytes >= need),
                "mdx_layer_norm_backward: needs %lld bytes of workspace, got %lld", (long long)need,
                (long long)workspace_bytes);
    if (!need && (!dx || rows == 0)) return MDX_OK;
    norm::Args a{};
    a.x = x; a.ldx = ldx;
    a.dy = grad; a.ldy = ldg;
    a.gamma = gamma;
    a.rows = rows; a.D = D;
    a.out = dx; a.ldo = lddx;
    a.mean = const_cast<float *>(mean); a.rstd = const_cast<float *>(rstd);
    a.part = need ? reinterpret_cast<float *>(workspace) : nullptr;
    return norm::dispatch("mdx_layer_norm_backward", a, dtype, true, dgamma, dbeta, as_stream(stream));
}
