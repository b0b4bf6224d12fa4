// A projection shared by all rows with low-rank adapters that each row
// chooses, on gfx950, forward and backward.
//
// Rows are sorted by adapter first (a counting sort that keeps their order),
// so a tile of rows meets few adapters. Then
//   H = A xd        the rows' low-rank inputs, one small product per tile
//   Y = W x + b + s B H   one matrix product; a tile's own low-rank products
//                   go into its accumulators before the walk over the depth
// and backward
//   dH = s B^T dy,  dX = W^T dy + drop(A^T dH),  dA = dH^T xd,  dB = s H^T dy.
// Low-rank values H and dH stay float; where they meet a bf16 operand in the
// matrix units they are split into bf16 terms (kdec_frag.hpp).
#include "kdec_frag.hpp"
#include "kdec_internal.hpp"
#include "kdec_philox.hpp"

#include <climits>
#include <memory>

namespace kdec {
namespace {

constexpr int NT = 256;   // threads of a block
constexpr int ST = 1024;  // threads of the sort
constexpr int GM = 128, GN = 128;  // features and rows of a product tile

struct Adapter {
    const void *X, *W, *bias, *A, *B, *dY;
    long x_rs, dy_rs;
    const float* scale;
    const int *idx, *unit_off;
    int T, in, out, n, units, rank, R;  // R = units * rank
    Drop drop;
    bool dropping;
    const int *perm, *seg;  // sorted rows; adapter a's are [seg[a], seg[a+1]), those without any from seg[n]
    float *H, *dH;          // (T, R)
    bool vec_x, vec_w, vec_a, vec_b, vec_dy, vec_h;
};

__device__ inline int adapter_of(const Adapter& p, int row) {
    const int a = p.idx[row];
    return a >= 0 && a < p.n ? a : p.n;
}

// Block a places adapter a's rows (a = n: the rows without one): every thread
// counts a run of rows, the counts are scanned, and the rows written in order.
__global__ __launch_bounds__(ST) void adapter_sort_k(const int* idx, int T, int n, int* perm, int* seg) {
    __shared__ int less_sum[ST / 64], eq_sum[ST / 64];
    const int a = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (T + ST - 1) / ST;
    const int t0 = static_cast<int>(min(static_cast<long>(tid) * per, static_cast<long>(T)));
    const int t1 = static_cast<int>(min(static_cast<long>(t0) + per, static_cast<long>(T)));
    int less = 0, eq = 0;
    for (int t = t0; t < t1; ++t) {
        int id = idx[t];
        if (id < 0 || id >= n) id = n;
        less += id < a;
        eq += id == a;
    }
    for (int o = 32; o; o >>= 1) less += __shfl_xor(less, o);
    int before = eq;  // inclusive scan within the wave
    for (int o = 1; o < 64; o <<= 1) {
        const int v = __shfl_up(before, o);
        if (lane >= o) before += v;
    }
    if (lane == 63) {
        less_sum[wave] = less;
        eq_sum[wave] = before;
    }
    __syncthreads();
    int at = before - eq;
    for (int w = 0; w < ST / 64; ++w) {
        at += less_sum[w];
        if (w < wave) at += eq_sum[w];
    }
    if (tid == 0) {
        seg[a] = at;
        if (a == n) seg[n + 1] = T;
    }
    for (int t = t0; t < t1; ++t) {
        int id = idx[t];
        if (id < 0 || id >= n) id = n;
        if (id == a) perm[at++] = t;
    }
}

// Zeros the fragment's values that the dropout mask drops: columns col .. + 7
// (a multiple of 8) of a row. The kept values' factor is the caller's.
template <class T>
__device__ inline Frag<T> dropped(const Drop& d, int row, int col, Frag<T> f) {
    unsigned w[4];
    drop_words(d, static_cast<unsigned>(row), static_cast<unsigned>(col) >> 3, w);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (!kept(d, w, i)) f[i] = static_cast<T>(0.0f);
    return f;
}

// The sum of the four waves' accumulators over a 32 x 32 block, handed to
// f(row, column, sum) by all threads.
template <class F>
__device__ inline void join_waves(float (&buf)[4][32][33], const f32x16& acc, F f) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
#pragma unroll
    for (int r = 0; r < 16; ++r) buf[wave][acc_row(r, lane >> 5)][lane & 31] = acc[r];
    __syncthreads();
    for (int e = tid; e < 1024; e += NT) {
        const int m = e & 31, c = e >> 5;
        f(m, c, (buf[0][m][c] + buf[1][m][c]) + (buf[2][m][c] + buf[3][m][c]));
    }
    __syncthreads();
}

// H: 32 sorted rows by 32 of the R low-rank columns per block, the depth
// split over its waves; one product per adapter that the rows meet.
template <class T>
__global__ __launch_bounds__(NT) void adapter_h_k(Adapter p) {
    __shared__ float buf[4][32][33];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5;
    const int s0 = blockIdx.x * 32, m0 = blockIdx.y * 32, ns = min(32, p.T - s0);
    const int col = lane & 31, row = col < ns ? p.perm[s0 + col] : 0;
    const int m = m0 + col;
    const T* x = static_cast<const T*>(p.X) + row * p.x_rs;
    for (int s = s0; s < s0 + ns;) {
        const int a = adapter_of(p, p.perm[s]), end = min(p.seg[a + 1], s0 + ns);
        f32x16 acc = f32x16{};
        if (a < p.n) {
            const T* w = static_cast<const T*>(p.A) + (static_cast<long>(a) * p.R + (m < p.R ? m : 0)) * p.in;
            for (int k = 16 * wave; k < p.in; k += 64) {
                const int d = k + 8 * half;
                Frag<T> f = load8(x + d, col < ns ? min(8, p.in - d) : 0, p.vec_x);
                if (p.dropping) f = dropped<T>(p.drop, row, d, f);
                acc = mma32(load8(w + d, m < p.R ? min(8, p.in - d) : 0, p.vec_a), f, acc);
            }
        }
        join_waves(buf, acc, [&](int c, int t, float v) {
            if (t >= s - s0 && t < end - s0 && m0 + c < p.R)
                p.H[static_cast<long>(p.perm[s0 + t]) * p.R + m0 + c] = p.dropping ? v * p.drop.keep : v;
        });
        s = end;
    }
}

// dH: as H, over a unit's output rows; B holds them row by row, so a lane
// gathers its eight depths.
template <class T>
__global__ __launch_bounds__(NT) void adapter_dh_k(Adapter p) {
    __shared__ float buf[4][32][33];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5;
    const int jt = (p.rank + 31) / 32, unit = blockIdx.y / jt, m0 = 32 * (blockIdx.y % jt);
    const int s0 = blockIdx.x * 32, ns = min(32, p.T - s0);
    const int col = lane & 31, row = col < ns ? p.perm[s0 + col] : 0;
    const int m = m0 + col;
    const int u0 = min(max(p.unit_off[unit], 0), p.out), u1 = min(max(p.unit_off[unit + 1], u0), p.out);
    const T* y = static_cast<const T*>(p.dY) + row * p.dy_rs;
    for (int s = s0; s < s0 + ns;) {
        const int a = adapter_of(p, p.perm[s]), end = min(p.seg[a + 1], s0 + ns);
        f32x16 acc = f32x16{};
        float sc = 0.0f;
        if (a < p.n) {
            sc = p.scale[a];
            const T* w = static_cast<const T*>(p.B) + static_cast<long>(a) * p.out * p.rank + (m < p.rank ? m : 0);
            for (int k = (u0 & ~15) + 16 * wave; k < u1; k += 64) {
                const int d = k + 8 * half;
                Frag<T> f = load8(y + d, col < ns ? min(8, p.out - d) : 0, p.vec_dy), g;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const bool in = d + i >= u0 && d + i < u1;
                    g[i] = in && m < p.rank ? w[static_cast<long>(d + i) * p.rank] : static_cast<T>(0.0f);
                    if (!in) f[i] = static_cast<T>(0.0f);
                }
                acc = mma32(g, f, acc);
            }
        }
        join_waves(buf, acc, [&](int c, int t, float v) {
            if (t >= s - s0 && t < end - s0 && m0 + c < p.rank)
                p.dH[static_cast<long>(p.perm[s0 + t]) * p.R + unit * p.rank + m0 + c] = v * sc;
        });
        s = end;
    }
}

// The product tile's operands: M features (W's rows forward, its columns
// backward), N sorted rows of X or dY, depth K.
struct Product {
    int M, K;
    const void* Z;  // X or dY
    long z_rs;
    bool vec_z;
    void* Y;
    long y_rs;
    bool vec_y;
    int splits;
    float* part;  // (splits, T, M)
};

template <class T> constexpr int depth_of() { return sizeof(T) == 2 ? 64 : 32; }  // of a tile: 128 bytes

// One 128 x 128 tile: forward Y = W X (+ bias + s B H), backward
// dX = W^T dY (+ drop(A^T dH)). Features are the accumulators' rows, so a
// lane holds one token's run of features. Four waves of 64 x 64. Rows of W
// lie along the depth forward and across it backward, where the transposing
// LDS read turns them.
template <class T, bool BWD>
__global__ __launch_bounds__(NT, 1) void adapter_gemm_k(Adapter p, Product g) {
    constexpr int BK = depth_of<T>(), WC = (BWD ? GM : BK) / 8;
    typedef Tile<T, BWD ? GM : BK> Tw;
    typedef Tile<T, BK> Tz;
    constexpr int NZ = GN * BK / 8 / NT, NW = GM * BK / 8 / NT;
    __shared__ __align__(16) T sw[GM * BK];
    __shared__ __align__(16) T sz[GN * BK];
    __shared__ int srow[GN], sid[GN];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5, col = lane & 31;
    const int mt = (g.M + GM - 1) / GM;
    const int m0 = (blockIdx.x % mt) * GM, s0 = (blockIdx.x / mt) * GN, ns = min(GN, p.T - s0), split = blockIdx.y;
    if (tid < GN) {
        const int row = tid < ns ? p.perm[s0 + tid] : 0;
        srow[tid] = row;
        sid[tid] = tid < ns ? adapter_of(p, row) : p.n;
    }
    __syncthreads();
    const int wm = m0 + 64 * (wave & 1), wn = 64 * (wave >> 1);
    f32x16 acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x16{};

    // the rows' adapters; splits take them in turn
    int turn = 0;
    for (int s = s0; s < s0 + ns;) {
        const int a = sid[s - s0], end = min(p.seg[a + 1], s0 + ns), s_end = end - s0;
        const bool mine = a < p.n && turn++ % g.splits == split && s - s0 < wn + 64 && s_end > wn;
        s = end;
        if (!mine) continue;
        const float sc = BWD ? 1.0f : p.scale[a];
        const float* H = BWD ? p.dH : p.H;
        int u0 = 0, u1 = p.units;
        if (!BWD) {  // the units that meet the wave's features
            while (u0 + 1 < p.units && p.unit_off[u0 + 1] <= wm) ++u0;
            u1 = u0 + 1;
            while (u1 < p.units && p.unit_off[u1] < wm + 64) ++u1;
        }
        for (int u = u0; u < u1; ++u) {
            const int lo = BWD ? 0 : p.unit_off[u], hi = BWD ? g.M : p.unit_off[u + 1];
            f32x16 tmp[2][2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) tmp[i][j] = f32x16{};
            for (int k = 0; k < p.rank; k += 16) {
                const int d = k + 8 * half;
                Frag<T> w[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int m = wm + 32 * i + col;
                    const bool in = m >= lo && m < hi && m < g.M;
                    if (BWD) {  // A's columns
                        const T* q = static_cast<const T*>(p.A) + (static_cast<long>(a) * p.R + u * p.rank) * p.in + (in ? m : 0);
#pragma unroll
                        for (int x = 0; x < 8; ++x)
                            w[i][x] = in && d + x < p.rank ? q[static_cast<long>(d + x) * p.in] : static_cast<T>(0.0f);
                    } else {
                        const T* q = static_cast<const T*>(p.B) + (static_cast<long>(a) * p.out + (in ? m : 0)) * p.rank;
                        w[i] = load8(q + (d < p.rank ? d : 0), in ? min(8, p.rank - d) : 0, p.vec_b);
                    }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int t = wn + 32 * j + col;
                    const float* h = H + static_cast<long>(srow[t]) * p.R + u * p.rank;
                    f32x8 f = load8(h + (d < p.rank ? d : 0), t < ns ? min(8, p.rank - d) : 0, p.vec_h);
#pragma unroll
                    for (int x = 0; x < 8; ++x) f[x] *= sc;
                    const Terms<T, 2> v(f);
#pragma unroll
                    for (int x = 0; x < v.n; ++x)
#pragma unroll
                        for (int i = 0; i < 2; ++i) tmp[i][j] = mma32(w[i], v.t[x], tmp[i][j]);
                }
            }
            // only this adapter's rows take the product, whatever another's would be
#pragma unroll
            for (int j = 0; j < 2; ++j)
                if (sid[wn + 32 * j + col] == a)
#pragma unroll
                    for (int i = 0; i < 2; ++i)
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[i][j][r] += tmp[i][j][r];
        }
    }
    if (BWD && p.dropping) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    unsigned w[4];
                    drop_words(p.drop, static_cast<unsigned>(srow[wn + 32 * j + col]),
                               static_cast<unsigned>(wm + 32 * i + 8 * q) >> 3, w);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const unsigned v = half ? w[2 + (x >> 1)] : w[x >> 1];
                        const bool keep = ((x & 1) ? v >> 16 : v & 0xFFFFu) >= p.drop.thr;
                        acc[i][j][4 * q + x] = keep ? acc[i][j][4 * q + x] * p.drop.keep : 0.0f;
                    }
                }
    }

    const int steps = (g.K + BK - 1) / BK;
    const int c0 = static_cast<int>(static_cast<long>(steps) * split / g.splits);
    const int c1 = static_cast<int>(static_cast<long>(steps) * (split + 1) / g.splits);
    Frag<T> fw[NW], fz[NZ];
    const auto load = [&](int c) {
        const int k0 = c * BK;
#pragma unroll
        for (int i = 0; i < NZ; ++i) {
            const int e = tid + i * NT, t = e / (BK / 8), d = k0 + 8 * (e % (BK / 8));
            fz[i] = load8(static_cast<const T*>(g.Z) + srow[t] * g.z_rs + d, t < ns ? min(8, g.K - d) : 0, g.vec_z);
        }
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const int e = tid + i * NT, r = e / WC, d = 8 * (e % WC);
            if (BWD) {
                const bool in = k0 + r < g.K;
                fw[i] = load8(static_cast<const T*>(p.W) + static_cast<long>(in ? k0 + r : 0) * g.M + m0 + d,
                              in ? min(8, g.M - m0 - d) : 0, p.vec_w);
            } else {
                const bool in = m0 + r < g.M;
                fw[i] = load8(static_cast<const T*>(p.W) + static_cast<long>(in ? m0 + r : 0) * g.K + k0 + d,
                              in ? min(8, g.K - k0 - d) : 0, p.vec_w);
            }
        }
    };
    if (c0 < c1) load(c0);
    for (int c = c0; c < c1; ++c) {
#pragma unroll
        for (int i = 0; i < NZ; ++i) {
            const int e = tid + i * NT;
            Tz::put8(sz, e / (BK / 8), e % (BK / 8), fz[i]);
        }
#pragma unroll
        for (int i = 0; i < NW; ++i) {
            const int e = tid + i * NT;
            Tw::put8(sw, e / WC, e % WC, fw[i]);
        }
        __syncthreads();
        if (c + 1 < c1) load(c + 1);
#pragma unroll
        for (int k = 0; k < BK / 16; ++k) {
            Frag<T> w[2], z[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int m = 64 * (wave & 1) + 32 * i;
                if constexpr (BWD) w[i] = lds_cols<GM, false>(sw, 16 * k, m);
                else w[i] = lds_rows<T, BK>(sw, m, k);
                z[i] = lds_rows<T, BK>(sz, wn + 32 * i, k);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = mma32(w[i], z[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int t = wn + 32 * j + col;
        if (t >= ns) continue;
        const long row = srow[t];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int m = wm + 32 * i + 8 * q + 4 * half;
                float v[4];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    v[x] = acc[i][j][4 * q + x];
                    if (!BWD && p.bias && m + x < g.M) v[x] += static_cast<float>(static_cast<const T*>(p.bias)[m + x]);
                }
                if (g.splits > 1)
                    store4(g.part + (split * static_cast<long>(p.T) + row) * g.M + m, g.M - m, g.M % 4 == 0, v[0], v[1], v[2], v[3]);
                else
                    store4(static_cast<T*>(g.Y) + row * g.y_rs + m, g.M - m, g.vec_y, v[0], v[1], v[2], v[3]);
            }
    }
}

// The splits' sums in their order, rounded once.
template <class T>
__global__ __launch_bounds__(NT) void adapter_join_k(const float* part, int splits, long n, int M, T* Y, long y_rs) {
    const long e = static_cast<long>(blockIdx.x) * NT + threadIdx.x;
    if (e >= n) return;
    float s = 0.0f;
    for (int i = 0; i < splits; ++i) s += part[i * n + e];
    const long row = e / M;
    Y[row * y_rs + (e - row * M)] = static_cast<T>(s);
}

// Sums over an adapter's rows: C[m, c] = f sum_t P[t, m] Z[t, c] for 32
// columns m of the float matrix P (H or dH, width R) and 128 columns c of X or
// dY. dA = dH^T drop(X): all of P's columns. dB^T = s H^T dY: the columns of
// the unit that c lies in. Steps of 32 rows through shared memory.
template <class T, bool DB>
__global__ __launch_bounds__(NT) void adapter_outer_k(Adapter p, const float* P, const T* Z, long z_rs, int C, bool vec_z,
                                                      float* out, float beta, int mt) {
    constexpr int NTERM = Terms<T, 3>::n;
    __shared__ __align__(16) T sz[32 * 128];
    __shared__ __align__(16) T sp[NTERM][32 * 64];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5, col = lane & 31;
    const int ct = (C + 127) / 128;
    int b = blockIdx.x;
    const int c0 = (b % ct) * 128;
    b /= ct;
    const int m0 = (b % mt) * 32, a = b / mt;
    const int s0 = p.seg[a], s1 = p.seg[a + 1];
    const int cols = DB ? p.rank : p.R;  // P's columns that a block's m counts
    const float f = DB ? p.scale[a] : p.dropping ? p.drop.keep : 1.0f;
    int u0 = 0, u1 = 1;
    if (DB) {
        while (u0 + 1 < p.units && p.unit_off[u0 + 1] <= c0) ++u0;
        u1 = u0 + 1;
        while (u1 < p.units && p.unit_off[u1] < c0 + 128) ++u1;
    }
    for (int u = u0; u < u1; ++u) {
        const float* base = P + (DB ? u * p.rank : 0);
        f32x16 acc = f32x16{};
        for (int s = s0; s < s1; s += 32) {
            for (int e = tid; e < 32 * 16; e += NT) {
                const int t = e >> 4, d = c0 + 8 * (e & 15), row = s + t < s1 ? p.perm[s + t] : 0;
                Frag<T> z = load8(Z + row * z_rs + d, s + t < s1 ? min(8, C - d) : 0, vec_z);
                if (!DB && p.dropping) z = dropped<T>(p.drop, row, d, z);
                Tile<T, 128>::put8(sz, t, e & 15, z);
            }
            if (tid < 32 * 4) {
                const int t = tid >> 2, d = m0 + 8 * (tid & 3), row = s + t < s1 ? p.perm[s + t] : 0;
                const float* q = base + static_cast<long>(row) * p.R + (d < cols ? d : 0);
                const Terms<T, 3> v(load8(q, s + t < s1 ? min(8, cols - d) : 0, false));
#pragma unroll
                for (int x = 0; x < NTERM; ++x) Tile<T, 64>::put8(sp[x], t, tid & 3, v.t[x]);
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const Frag<T> z = lds_cols<128, false>(sz, 16 * k, 32 * wave);
#pragma unroll
                for (int x = 0; x < NTERM; ++x) acc = mma32(lds_cols<64, false>(sp[x], 16 * k, 0), z, acc);
            }
            __syncthreads();
        }
        const int c = c0 + 32 * wave + col;
        if (c >= C || (DB && (c < p.unit_off[u] || c >= p.unit_off[u + 1]))) continue;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int m = m0 + acc_row(r, half);
            if (m >= cols) continue;
            float* o = DB ? out + (static_cast<long>(a) * C + c) * p.rank + m : out + (static_cast<long>(a) * p.R + m) * C + c;
            *o = beta == 0.0f ? f * acc[r] : beta * *o + f * acc[r];
        }
    }
}

// ─── host ───

bool aligned16(const void* p, long stride_bytes) {
    return reinterpret_cast<size_t>(p) % 16 == 0 && stride_bytes % 16 == 0;
}

int check(kdec_ctx* ctx, const char* who, int dtype, int T, int in, int out, int adapters, int units, int rank, float prob,
          long seed, long offset, Adapter& p) {
    const auto bad = [&](const char* why) { return fail(ctx, KDEC_EINVAL, std::string(who) + ": " + why); };
    if (dtype != KDEC_F32 && dtype != KDEC_BF16) return bad("unknown type");
    if (T < 0 || in <= 0 || out <= 0 || adapters < 0) return bad("bad sizes");
    if (units < 1 || units > 4096) return bad("units outside 1..4096");
    if (rank < 1 || rank > 128) return bad("rank outside 1..128");
    if (T > INT_MAX - 256 || in > INT_MAX - 256 || out > INT_MAX - 256 || adapters > (1 << 20)) return bad("sizes too large");
    if (!make_drop(prob, seed, offset, p.drop)) return bad("p must be at least 0 and below 1");
    p.dropping = p.drop.thr != 0;
    return KDEC_OK;
}

// Launches f(type value) for the call's type.
template <class F> int typed(int dtype, F f) { return dtype == KDEC_F32 ? f(float{}) : f(bf16{}); }

void sort_rows(kdec_ctx* ctx, const Adapter& p, int* perm, int* seg) {
    hipLaunchKernelGGL(adapter_sort_k, dim3(p.n + 1), dim3(ST), 0, ctx->stream, p.idx, p.T, p.n, perm, seg);
}

template <class T, bool BWD>
int product(kdec_ctx* ctx, const Adapter& p, Product g) {
    const long tiles = cdiv(g.M, GM) * cdiv(p.T, GN);
    if (tiles >= INT_MAX) return fail(ctx, KDEC_EINVAL, "kdec_adapter: too many rows");
    hipLaunchKernelGGL((adapter_gemm_k<T, BWD>), dim3(static_cast<unsigned>(tiles), g.splits), dim3(NT), 0, ctx->stream, p, g);
    if (g.splits > 1) {
        const long n = static_cast<long>(p.T) * g.M;
        hipLaunchKernelGGL(adapter_join_k<T>, dim3(static_cast<unsigned>(cdiv(n, NT))), dim3(NT), 0, ctx->stream, g.part, g.splits,
                           n, g.M, static_cast<T*>(g.Y), g.y_rs);
    }
    return KDEC_OK;
}

size_t up(size_t n) { return (n + 255) & ~size_t(255); }

}  // namespace
}  // namespace kdec

using namespace kdec;

extern "C" {

int kdec_adapter_fwd(kdec_ctx* ctx, int dtype, const void* X, long x_rs, const void* W, const void* bias, const void* A,
                     const void* B, const float* scale, const int* idx, const int* unit_off, int T, int in, int out,
                     int adapters, int units, int rank, float prob, long seed, long offset, float* H, void* Y, long y_rs) {
    if (!ctx) return KDEC_EINVAL;
    Adapter p{};
    if (int rc = check(ctx, "kdec_adapter_fwd", dtype, T, in, out, adapters, units, rank, prob, seed, offset, p)) return rc;
    if (T == 0) return KDEC_OK;
    KDEC_CHECK(ctx, X && W && Y && idx && unit_off && (adapters == 0 || (A && B && scale)), "kdec_adapter_fwd: null tensor");
    KDEC_CHECK(ctx, T == 1 || y_rs >= out, "kdec_adapter_fwd: row stride of Y too small");
    const size_t es = dtype == KDEC_F32 ? 4 : 2;
    const int el = static_cast<int>(16 / es), R = units * rank;
    p.X = X; p.W = W; p.bias = bias; p.A = A; p.B = B; p.x_rs = x_rs;
    p.scale = scale; p.idx = idx; p.unit_off = unit_off;
    p.T = T; p.in = in; p.out = out; p.n = adapters; p.units = units; p.rank = rank; p.R = R;
    p.vec_x = in % el == 0 && aligned16(X, x_rs * es);
    p.vec_w = in % el == 0 && aligned16(W, 0);
    p.vec_a = in % el == 0 && aligned16(A, 0);
    p.vec_b = rank % 8 == 0 && aligned16(B, 0);
    ProfScope ps(ctx, "adapter", 2.0 * T * in * out, 0.0);
    const size_t perm_b = up(T * 4ul), seg_b = up((adapters + 2ul) * 4), h_b = H ? 0 : up(static_cast<size_t>(T) * R * 4);
    Workspace ws(ctx, perm_b + seg_b + h_b);
    if (!ws.p) return KDEC_ENOMEM;
    int *perm = ws.as<int>(), *seg = reinterpret_cast<int*>(ws.as<char>() + perm_b);
    p.perm = perm;
    p.seg = seg;
    p.H = H ? H : reinterpret_cast<float*>(ws.as<char>() + perm_b + seg_b);
    p.vec_h = rank % 8 == 0 && aligned16(p.H, 0);
    sort_rows(ctx, p, perm, seg);
    return typed(dtype, [&](auto t) {
        typedef decltype(t) E;
        hipLaunchKernelGGL(adapter_h_k<E>, dim3(static_cast<unsigned>(cdiv(T, 32)), static_cast<unsigned>(cdiv(R, 32))), dim3(NT), 0,
                           ctx->stream, p);
        Product g{out, in, X, x_rs, p.vec_x, Y, y_rs,
                  out % 4 == 0 && reinterpret_cast<size_t>(Y) % (4 * es) == 0 && (y_rs * es) % (4 * es) == 0, 1, nullptr};
        if (int rc = product<E, false>(ctx, p, g)) return rc;
        return launch_check(ctx, "kdec_adapter_fwd");
    });
}

int kdec_adapter_bwd(kdec_ctx* ctx, int dtype, const void* X, long x_rs, const void* W, const void* A, const void* B,
                     const float* scale, const int* idx, const int* unit_off, int T, int in, int out, int adapters, int units,
                     int rank, float prob, long seed, long offset, const float* H, const void* dY, long dy_rs, void* dX,
                     long dx_rs, float* dA, float* dB, float beta) {
    if (!ctx) return KDEC_EINVAL;
    Adapter p{};
    if (int rc = check(ctx, "kdec_adapter_bwd", dtype, T, in, out, adapters, units, rank, prob, seed, offset, p)) return rc;
    KDEC_CHECK(ctx, !dA == !dB, "kdec_adapter_bwd: dA and dB go together");
    KDEC_CHECK(ctx, T == 0 || (X && W && H && dY && idx && unit_off), "kdec_adapter_bwd: null tensor");
    KDEC_CHECK(ctx, unit_off && (adapters == 0 || (A && B && scale)), "kdec_adapter_bwd: null tensor");
    KDEC_CHECK(ctx, !dX || T <= 1 || dx_rs >= in, "kdec_adapter_bwd: row stride of dX too small");
    if ((T == 0 || !dX) && (adapters == 0 || !dA)) return KDEC_OK;
    const size_t es = dtype == KDEC_F32 ? 4 : 2;
    const int el = static_cast<int>(16 / es), R = units * rank;
    p.X = X; p.W = W; p.A = A; p.B = B; p.dY = dY; p.x_rs = x_rs; p.dy_rs = dy_rs;
    p.scale = scale; p.idx = idx; p.unit_off = unit_off;
    p.T = T; p.in = in; p.out = out; p.n = adapters; p.units = units; p.rank = rank; p.R = R;
    p.vec_x = in % el == 0 && aligned16(X, x_rs * es);
    p.vec_w = in % el == 0 && aligned16(W, 0);
    p.vec_a = in % el == 0 && aligned16(A, 0);
    p.vec_b = rank % 8 == 0 && aligned16(B, 0);
    p.vec_dy = out % el == 0 && aligned16(dY, dy_rs * es);
    ProfScope ps(ctx, "adapter", 2.0 * T * in * out, 0.0);
    // Few tiles over a long depth: the depth split over blocks, to no fewer
    // than 512 deep each.
    const long tiles = cdiv(in, GM) * cdiv(T, GN);
    long splits = dX && T > 0 ? cdiv(2L * ctx->num_cus, tiles) : 1;
    if (splits > out / 512) splits = out / 512;
    if (splits < 1) splits = 1;
    const size_t perm_b = up(T * 4ul), seg_b = up((adapters + 2ul) * 4), h_b = up(static_cast<size_t>(T) * R * 4);
    Workspace ws(ctx, perm_b + seg_b + h_b + (splits > 1 ? static_cast<size_t>(splits) * T * in * 4 : 0));
    if (!ws.p) return KDEC_ENOMEM;
    int *perm = ws.as<int>(), *seg = reinterpret_cast<int*>(ws.as<char>() + perm_b);
    p.perm = perm;
    p.seg = seg;
    p.H = const_cast<float*>(H);
    p.dH = reinterpret_cast<float*>(ws.as<char>() + perm_b + seg_b);
    p.vec_h = rank % 8 == 0;
    sort_rows(ctx, p, perm, seg);
    return typed(dtype, [&](auto t) {
        typedef decltype(t) E;
        if (T > 0) {
            const long jt = cdiv(rank, 32);
            hipLaunchKernelGGL(adapter_dh_k<E>, dim3(static_cast<unsigned>(cdiv(T, 32)), static_cast<unsigned>(units * jt)), dim3(NT),
                               0, ctx->stream, p);
        }
        if (T > 0 && dX) {
            Product g{in, out, dY, dy_rs, p.vec_dy, dX, dx_rs,
                      in % 4 == 0 && reinterpret_cast<size_t>(dX) % (4 * es) == 0 && (dx_rs * es) % (4 * es) == 0,
                      static_cast<int>(splits), reinterpret_cast<float*>(ws.as<char>() + perm_b + seg_b + h_b)};
            if (int rc = product<E, true>(ctx, p, g)) return rc;
        }
        if (dA && adapters > 0) {
            const long at = cdiv(R, 32), bt = cdiv(rank, 32);
            const long ab = cdiv(in, 128) * at * adapters, bb = cdiv(out, 128) * bt * adapters;
            KDEC_CHECK(ctx, ab < INT_MAX && bb < INT_MAX, "kdec_adapter_bwd: too many adapters");
            hipLaunchKernelGGL((adapter_outer_k<E, false>), dim3(static_cast<unsigned>(ab)), dim3(NT), 0, ctx->stream, p, p.dH,
                               static_cast<const E*>(X), x_rs, in, p.vec_x, dA, beta, static_cast<int>(at));
            hipLaunchKernelGGL((adapter_outer_k<E, true>), dim3(static_cast<unsigned>(bb)), dim3(NT), 0, ctx->stream, p, p.H,
                               static_cast<const E*>(dY), dy_rs, out, p.vec_dy, dB, beta, static_cast<int>(bt));
        }
        return launch_check(ctx, "kdec_adapter_bwd");
    });
}

}  // extern "C"
