// A projection shared by all rows with low-rank adapters that each row
// chooses, on gfx950, forward and backward.
//
// With many rows they are sorted by adapter first (a counting sort that keeps
// their order) and cut into pieces of one adapter each. Then
//   H = s A xd       the rows' low-rank inputs, one small product per piece
//   Y = W x + b + B H  one matrix product; a tile's own low-rank products
//                    go into its accumulators before the walk over the depth
// and backward
//   dH = s B^T dy,  dX = W^T dy + drop(A^T dH),  dA = dH^T xd,  dB = H^T dy.
// Low-rank values H and dH stay float; where they meet a bf16 operand in the
// matrix units they are split into bf16 terms (kdec_frag.hpp). Few rows go
// without the sort: a row's H is a block's work, and a block of the product
// holds all rows.
#include "kdec_frag.hpp"
#include "kdec_internal.hpp"
#include "kdec_philox.hpp"

#include <climits>
#include <memory>

namespace kdec {
namespace {

constexpr int NT = 256;            // threads of the gradients' blocks
constexpr int LT = 512;            // threads of the low-rank kernels' blocks, 8 waves
constexpr int ST = 1024;           // threads of the sort
constexpr int PIECE = 32;          // sorted rows of a piece
constexpr int CHUNK = 256;         // least sorted rows of a chunk, the adapters' gradients' unit of work
constexpr int CHUNKS = 512;        // cuts of the rows: each holds a gradient of its own until they are added
constexpr int FEW = 64;            // rows that one block of the product holds whole

// Sorted rows [start, start + count) of one adapter (n: none).
struct Piece {
    int start, count, adapter, pad;
};

struct Adapter {
    const void *X, *W, *bias, *A, *B, *dY;
    long x_rs, dy_rs;
    const float* scale;
    const int *idx, *unit_off;
    int T, in, out, n, units, rank, R;  // R = units * rank
    Drop drop;
    bool dropping;
    const int* perm;              // sorted rows
    const Piece *pieces, *chunks;
    float *H, *dH;                // (T, R), with the adapters' scales
    bool vec_x, vec_w, vec_a, vec_b, vec_dy, vec_h;
};

__device__ inline int adapter_of(const Adapter& p, int row) {
    const int a = p.idx[row];
    return a >= 0 && a < p.n ? a : p.n;
}

// The unit that holds output row m: how many of the offsets 1 .. units - 1 are
// not past it, 64 at a time (all lanes of the wave take part).
__device__ inline int unit_at(const int* off, int units, int m) {
    const int lane = threadIdx.x & 63;
    int u = 0;
    for (int b = 1; b < units; b += 64)
        u += __builtin_popcountll(__builtin_amdgcn_ballot_w64(b + lane < units && off[b + lane] <= m));
    return u;
}

// Block a places adapter a's rows (a = n: the rows without one): every wave
// counts a run of rows, and from the counts writes its rows in order. Its
// pieces (and chunks) are the windows of PIECE (`chunk`) sorted places that its
// rows meet. They start at table entry start / window + a,
// which no other adapter's reach: an adapter of c rows meets at most
// c / window + 1 windows; entries up to the next adapter's first are empty.
__global__ __launch_bounds__(ST) void adapter_sort_k(const int* idx, int T, int n, int chunk, int* perm, Piece* pieces, Piece* chunks) {
    constexpr int NW = ST / 64, AHEAD = 8;
    __shared__ int less_sum[NW], eq_sum[NW];
    const int a = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = ((T + NW - 1) / NW + 63) / 64 * 64;  // rows of a wave, 64 at a time
    const int t0 = static_cast<int>(min(static_cast<long>(wave) * per, static_cast<long>(T)));
    const int t1 = static_cast<int>(min(static_cast<long>(t0) + per, static_cast<long>(T)));
    const auto each = [&](auto f) {  // f(row, its adapter or n; -1 past the rows)
        for (int t = t0; t < t1; t += 64 * AHEAD) {
            int id[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int row = t + 64 * i + lane;
                id[i] = row < t1 ? idx[row] : -1;
                if (row < t1 && (id[i] < 0 || id[i] >= n)) id[i] = n;
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) f(t + 64 * i + lane, id[i]);
        }
    };
    int less = 0, eq = 0;
    each([&](int, int id) {
        less += __builtin_popcountll(__builtin_amdgcn_ballot_w64(id >= 0 && id < a));
        eq += __builtin_popcountll(__builtin_amdgcn_ballot_w64(id == a));
    });
    if (lane == 0) {
        less_sum[wave] = less;
        eq_sum[wave] = eq;
    }
    __syncthreads();
    int at = 0, start = 0, count = 0;
    for (int w = 0; w < NW; ++w) {
        start += less_sum[w];
        count += eq_sum[w];
        if (w < wave) at += eq_sum[w];
    }
    at += start;
    const auto table = [&](Piece* to, int window) {
        const int first = start / window, next = (start + count) / window + a + 1;
        for (int i = first + a + tid; i < next; i += ST) {
            const int w = i - a, s = max(start, w * window);
            to[i] = Piece{s, max(min(start + count, (w + 1) * window) - s, 0), a, 0};
        }
    };
    table(pieces, PIECE);
    table(chunks, chunk);
    each([&](int row, int id) {
        const unsigned long long hit = __builtin_amdgcn_ballot_w64(id == a);
        if (id == a) perm[at + __builtin_popcountll(hit & ((1ull << lane) - 1))] = row;
        at += __builtin_popcountll(hit);
    });
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

// The sum of eight waves' accumulators over a 32 x 32 block, handed to
// f(row, column, sum) by all threads, rows running fastest.
typedef float Join8[32][33];
template <class F>
__device__ inline void join8(Join8* buf, const f32x16& acc, F f) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
#pragma unroll
    for (int r = 0; r < 16; ++r) buf[wave][acc_row(r, lane >> 5)][lane & 31] = acc[r];
    __syncthreads();
    for (int e = tid; e < 1024; e += LT) {
        const int m = e & 31, c = e >> 5;
        float s = buf[0][m][c];
#pragma unroll
        for (int w = 1; w < 8; ++w) s += buf[w][m][c];
        f(m, c, s);
    }
    __syncthreads();
}

// H: a piece's rows (or, unsorted, one row) by 32 MT of the R low-rank columns
// per block, the depth split over its eight waves, four steps' loads in flight.
template <class T, int MT>
__global__ __launch_bounds__(LT) void adapter_h_k(Adapter p) {
    __shared__ Join8 buf[8];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5, col = lane & 31;
    const int m0 = blockIdx.y * 32 * MT;
    int start = 0, count = 1, a, row;
    if (p.pieces) {
        const Piece pc = p.pieces[blockIdx.x];
        start = pc.start;
        count = pc.count;
        a = pc.adapter;
        if (!count) return;
        row = p.perm[start + min(col, count - 1)];
    } else {
        row = blockIdx.x;
        a = adapter_of(p, row);
    }
    const auto row_of = [&](int c) { return p.pieces ? p.perm[start + c] : static_cast<int>(blockIdx.x); };
    f32x16 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x16{};
    float f = 0.0f;
    if (a < p.n) {
        f = p.scale[a] * (p.dropping ? p.drop.keep : 1.0f);
        const T* x = static_cast<const T*>(p.X) + row * p.x_rs;
        const T* w[MT];
#pragma unroll
        for (int i = 0; i < MT; ++i)
            w[i] = static_cast<const T*>(p.A) + (static_cast<long>(a) * p.R + min(m0 + 32 * i + col, p.R - 1)) * p.in;
        for (int k = 16 * wave; k < p.in; k += 512) {
            Frag<T> z[4], g[4][MT];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const int d = k + 128 * s + 8 * half, n = min(8, p.in - d);
                z[s] = load8(x + (n > 0 ? d : 0), col < count ? n : 0, p.vec_x);
#pragma unroll
                for (int i = 0; i < MT; ++i) g[s][i] = load8(w[i] + (n > 0 ? d : 0), m0 + 32 * i + col < p.R ? n : 0, p.vec_a);
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                if (k + 128 * s >= p.in) break;
                if (p.dropping) z[s] = dropped<T>(p.drop, row, k + 128 * s + 8 * half, z[s]);
#pragma unroll
                for (int i = 0; i < MT; ++i) acc[i] = mma32(g[s][i], z[s], acc[i]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i)
        join8(buf, acc[i], [&](int m, int c, float v) {
            if (c < count && m0 + 32 * i + m < p.R) p.H[static_cast<long>(row_of(c)) * p.R + m0 + 32 * i + m] = v * f;
        });
}

// dH: a piece's rows by 32 low-rank columns of one unit per block. The
// depth is the unit's output rows, RT at a time per wave with four steps'
// loads in flight; B's rows go through
// the wave's shared memory, from which the product reads their columns.
template <class T>
__global__ __launch_bounds__(LT) void adapter_dh_k(Adapter p) {
    constexpr int RT = sizeof(T) == 2 ? 32 : 16, DPB = 64, NB = RT * 4 / 64, AHEAD = 4;
    __shared__ __align__(16) char smem[8 * sizeof(Join8)];
    static_assert(sizeof(smem) >= 8 * RT * DPB * sizeof(T), "the waves are joined in the tiles' place");
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5, col = lane & 31;
    const Piece pc = p.pieces[blockIdx.x];
    if (!pc.count) return;
    const int jt = (p.rank + 31) / 32, unit = blockIdx.y / jt, m0 = 32 * (blockIdx.y % jt), a = pc.adapter;
    const int u0 = min(max(p.unit_off[unit], 0), p.out), u1 = min(max(p.unit_off[unit + 1], u0), p.out);
    const int row = p.perm[pc.start + min(col, pc.count - 1)];
    T* tile = reinterpret_cast<T*>(smem) + wave * RT * DPB;
    f32x16 acc = f32x16{};
    float f = 0.0f;
    if (a < p.n) {
        f = p.scale[a];
        const T* y = static_cast<const T*>(p.dY) + row * p.dy_rs;
        const T* b = static_cast<const T*>(p.B) + static_cast<long>(a) * p.out * p.rank + m0;
        Frag<T> z[AHEAD][RT / 16], w[AHEAD][NB];
        const auto load = [&](int r0, Frag<T> (&z)[RT / 16], Frag<T> (&w)[NB]) __attribute__((always_inline)) {
#pragma unroll
            for (int c = 0; c < RT / 16; ++c) {
                const int d = r0 + 16 * c + 8 * half;
                z[c] = load8(y + min(d, p.out), col < pc.count ? min(8, p.out - d) : 0, p.vec_dy);
            }
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int e = lane + 64 * i, r = r0 + (e >> 2), j = 8 * (e & 3);
                const bool in = r >= u0 && r < u1 && m0 + j < p.rank;
                w[i] = load8(b + (in ? static_cast<long>(r) * p.rank + j : 0), in ? min(8, p.rank - m0 - j) : 0, p.vec_b);
            }
        };
        const auto step = [&](int r0, Frag<T> (&z)[RT / 16], const Frag<T> (&w)[NB]) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int e = lane + 64 * i;
                Tile<T, DPB>::put8(tile, e >> 2, e & 3, w[i]);
            }
            if (r0 < u0 || r0 + RT > u1) {  // other units' outputs, whatever they hold
#pragma unroll
                for (int c = 0; c < RT / 16; ++c)
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int d = r0 + 16 * c + 8 * half + i;
                        if (d < u0 || d >= u1) z[c][i] = static_cast<T>(0.0f);
                    }
            }
#pragma unroll
            for (int c = 0; c < RT / 16; ++c) acc = mma32(lds_cols<DPB, false>(tile, 16 * c, 0), z[c], acc);
        };
        const int first = (u0 & ~7) + RT * wave;
#pragma unroll
        for (int s = 0; s < AHEAD; ++s)
            if (first + 8 * RT * s < u1) load(first + 8 * RT * s, z[s], w[s]);
        for (int r0 = first; r0 < u1; r0 += 8 * RT * AHEAD)
#pragma unroll
            for (int s = 0; s < AHEAD; ++s) {
                const int r = r0 + 8 * RT * s;
                if (r >= u1) break;
                step(r, z[s], w[s]);
                if (r + 8 * RT * AHEAD < u1) load(r + 8 * RT * AHEAD, z[s], w[s]);
            }
    }
    __syncthreads();
    join8(reinterpret_cast<Join8*>(smem), acc, [&](int c, int t, float v) {
        if (t < pc.count && m0 + c < p.rank)
            p.dH[static_cast<long>(p.perm[pc.start + t]) * p.R + unit * p.rank + m0 + c] = v * f;
    });
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

// The low-rank products of 32 MB of a wave's features (from wm) and its 32 NB
// rows (a lane each: its row and adapter), into acc: forward B H, backward
// A^T dH. Rows of other adapters and features of other units take part with
// zeros, which values that are not finite would make NaN: such values of either
// side are left out, and `wild` gets the rows that they belong to. Adapters and
// units are taken in turn by `turns` takers of which this is number `turn`.
template <class T, bool BWD, int MB, int NB>
__device__ inline void low_rank(const Adapter& p, int M, int wm, int u0, int u1, int row, int id, int turn, int turns,
                                f32x16 (&acc)[MB][NB], unsigned long long& wild) {
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
    const float* H = BWD ? p.dH : p.H;
    unsigned long long left = __builtin_amdgcn_ballot_w64(id < p.n);
    int rows[NB], ids[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        rows[j] = __shfl(row, 32 * j + col);
        ids[j] = __shfl(id, 32 * j + col);
    }
    int u = u0 + turn;  // the next unit that is this taker's
    while (left) {
        const int a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        const unsigned long long mine = __builtin_amdgcn_ballot_w64(id == a);
        left &= ~mine;
        for (; u < u1; u += turns) {
            const int lo = BWD ? 0 : p.unit_off[u], hi = BWD ? M : p.unit_off[u + 1];
            for (int k = 0; k < p.rank; k += 16) {
                const int d = k + 8 * half, n = min(8, p.rank - d), dd = n > 0 ? d : 0;
                Frag<T> w[2];
                f32x8 h[NB];
                bool bad = false;
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    h[j] = load8(H + static_cast<long>(rows[j]) * p.R + u * p.rank + dd, ids[j] == a ? n : 0, p.vec_h);
                    bad |= not_finite(h[j]);
                }
                if (__builtin_amdgcn_ballot_w64(bad)) {
#pragma unroll
                    for (int j = 0; j < NB; ++j) h[j] = finite_part(h[j]);
                    wild |= mine;
                    asm volatile("");  // a branch
                }
#pragma unroll
                for (int i0 = 0; i0 < MB; i0 += 2) {  // 64 features at a time, which the registers leave room for
                    bad = false;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int m = wm + 32 * (i0 + i) + col;
                        const bool in = m >= lo && m < hi && m < M;
                        if (BWD) {  // A's columns
                            const T* q = static_cast<const T*>(p.A) + (static_cast<long>(a) * p.R + u * p.rank) * p.in + (in ? m : 0);
#pragma unroll
                            for (int x = 0; x < 8; ++x)
                                w[i][x] = in && x < n ? q[static_cast<long>(d + x) * p.in] : static_cast<T>(0.0f);
                        } else {
                            const T* q = static_cast<const T*>(p.B) + (static_cast<long>(a) * p.out + (in ? m : 0)) * p.rank;
                            w[i] = load8(q + dd, in ? n : 0, p.vec_b);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) bad |= not_finite(w[i]);
                    if (__builtin_amdgcn_ballot_w64(bad)) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) w[i] = finite_part(w[i]);
                        wild |= mine;
                        asm volatile("");  // a branch
                    }
#pragma unroll
                    for (int j = 0; j < NB; ++j) {
                        if (!(mine >> (32 * j) & 0xFFFFFFFFull)) continue;
                        const Terms<T, 2> v(h[j]);
#pragma unroll
                        for (int x = 0; x < v.n; ++x)
#pragma unroll
                            for (int i = 0; i < 2; ++i) acc[i0 + i][j] = mma32(w[i], v.t[x], acc[i0 + i][j]);
                    }
                    if (MB > 2) __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        u -= u1 - u0;
    }
}

// What low_rank left out of the `wild` rows: their low-rank sums over a wave's
// `features` from wm, one by one, of which those that are not finite are added
// to what the wave has written. (Splits that share such a sum all add it, which
// changes neither an infinity nor NaN.)
template <class T, bool BWD, class O>
__device__ inline void wild_sums(const Adapter& p, int M, int wm, int features, int u0, int u1, int row, int id,
                                 unsigned long long wild, O* Y, long y_rs) {
    const int lane = threadIdx.x & 63;
    __threadfence();  // a lane takes what others wrote
    for (; wild; wild &= wild - 1) {
        const int l = __builtin_ctzll(wild);
        const int t = __builtin_amdgcn_readlane(row, l), a = __builtin_amdgcn_readlane(id, l);
        for (int m = wm + lane; m < min(wm + features, M); m += 64) {
            float low = 0.0f;
            for (int u = u0; u < u1; ++u) {
                if (!BWD && (m < p.unit_off[u] || m >= p.unit_off[u + 1])) continue;
                const float* h = (BWD ? p.dH : p.H) + static_cast<long>(t) * p.R + u * p.rank;
                const T* w = BWD ? static_cast<const T*>(p.A) + (static_cast<long>(a) * p.R + u * p.rank) * p.in + m
                                 : static_cast<const T*>(p.B) + (static_cast<long>(a) * p.out + m) * p.rank;
                for (int j = 0; j < p.rank; ++j) low = __builtin_fmaf(static_cast<float>(w[BWD ? static_cast<long>(j) * p.in : j]), h[j], low);
                if (!__builtin_amdgcn_ballot_w64(low == low)) break;  // NaN whatever follows
            }
            if (BWD && p.dropping) {
                unsigned w[4];
                drop_words(p.drop, static_cast<unsigned>(t), static_cast<unsigned>(m) >> 3, w);
                unsigned v = w[0];
#pragma unroll
                for (int i = 1; i < 4; ++i) v = (m >> 1 & 3) == i ? w[i] : v;
                if (((m & 1) ? v >> 16 : v & 0xFFFFu) < p.drop.thr) low = 0.0f;
            }
            O* y = Y + t * y_rs + m;
            if (!(__builtin_fabsf(low) < __builtin_inff())) *y = static_cast<O>(static_cast<float>(*y) + low);
        }
    }
}

// One tile of features by rows: forward Y = W X (+ bias + B H), backward
// dX = W^T dY (+ drop(A^T dH)). Features are the accumulators' rows, so a lane
// holds one token's run of features. Rows of W lie along the depth forward
// and across it backward, where the transposing LDS read turns them. Tiles
// are copied straight to shared memory (DIRECT), or go through registers where
// alignment or size rule that out. BIG: 256 x 256 by eight waves of 128 x 64,
// which copies half the bytes per product; else 128 x 128 by four waves of
// 64 x 64, two blocks per CU. Two buffers each.
template <class T, bool BWD, bool DIRECT, bool BIG>
__global__ __launch_bounds__(BIG ? 512 : 256, DIRECT ? 2 : 1) void adapter_gemm_k(Adapter p, Product g) {
    constexpr int GM = BIG ? 256 : 128, GN = GM, NT = 2 * GM, MB = BIG ? 4 : 2;
    constexpr int BK = depth_of<T>(), WC = (BWD ? GM : BK) / 8, WR = BWD ? BK : GM;
    typedef Tile<T, BWD ? GM : BK> Tw;
    typedef Tile<T, BK> Tz;
    constexpr int NZ = GN * BK / 8 / NT, NW = GM * BK / 8 / NT;
    __shared__ __align__(256) T sw0[GM * BK], sw1[GM * BK], sz0[GN * BK], sz1[GN * BK];
    __shared__ int srow[GN], sid[GN];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5, col = lane & 31;
    // Blocks go to the eight XCDs in turn: each takes a run of row tiles with
    // all their features, so its L2 holds few rows of X and one step of W.
    int tile = blockIdx.x;
    if (gridDim.x % 8 == 0) tile = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    const int mt = (g.M + GM - 1) / GM;
    const int m0 = (tile % mt) * GM, s0 = (tile / mt) * GN, ns = min(GN, p.T - s0), split = blockIdx.y;
    if (tid < GN) {
        const int row = tid < ns ? p.perm[s0 + tid] : 0;
        srow[tid] = row;
        sid[tid] = tid < ns ? adapter_of(p, row) : p.n;
    }
    __syncthreads();
    const int wf = 32 * MB * (wave & 1), wm = m0 + wf, wn = 64 * (wave >> 1);  // the wave's features and rows
    const int steps = (g.K + BK - 1) / BK;
    const int c0 = static_cast<int>(static_cast<long>(steps) * split / g.splits);
    const int c1 = static_cast<int>(static_cast<long>(steps) * (split + 1) / g.splits);
    const T* W = static_cast<const T*>(p.W);
    const T* Z = static_cast<const T*>(g.Z);

    // direct copies: a thread's units of both tiles
    Copy<T, BWD ? GM : BK, WR, NT> cw;
    constexpr int NU = Tz::NU, NZU = GN * NU / NT;
    unsigned oz[NZU];
    __amdgpu_buffer_rsrc_t rz = rows_rsrc<T>(Z, 0, 0, 0);
    const auto z_offsets = [&](int depth) __attribute__((always_inline)) {  // columns of the tile that are there
#pragma unroll
        for (int i = 0; i < NZU; ++i) {
            const int u = tid + i * NT, r = u / NU, c = Tz::U * ((u % NU) ^ Tz::swz(r));
            oz[i] = r < ns && c < depth ? static_cast<unsigned>((srow[r] * g.z_rs + c) * static_cast<long>(sizeof(T))) : 0xFFFFFFF0u;
        }
    };
    if (DIRECT) {
        cw.init(BWD ? g.M : g.K, BWD ? g.M - m0 : g.K - c0 * BK, tid);
        z_offsets(g.K - c0 * BK);
        rz = uniform_rsrc(Z, static_cast<int>(((p.T - 1) * g.z_rs + g.K) * static_cast<long>(sizeof(T))));
    }
    Frag<T> fw[DIRECT ? 1 : NW], fz[DIRECT ? 1 : NZ];
    const auto load = [&](int c, T* tw, T* tz) __attribute__((always_inline)) {
        const int k0 = c * BK;
        if constexpr (DIRECT) {
            if (c > c0 && k0 + BK > g.K) {  // the last, narrower step
                if (!BWD) cw.init(g.K, g.K - k0, tid);
                z_offsets(g.K - k0);
            }
            if (BWD) cw.load(tw, W + static_cast<long>(k0) * g.M + m0, g.M, g.K - k0, min(GM, g.M - m0), wave);
            else cw.load(tw, W + static_cast<long>(m0) * g.K + k0, g.K, g.M - m0, min(BK, g.K - k0), wave);
#pragma unroll
            for (int i = 0; i < NZU; ++i)
                copy16(rz, tz + (64 * wave + i * NT) * Tz::U,
                       static_cast<int>(oz[i] == 0xFFFFFFF0u ? oz[i] : oz[i] + static_cast<unsigned>(k0 * sizeof(T))));
        } else {
#pragma unroll
            for (int i = 0; i < NZ; ++i) {
                const int e = tid + i * NT, t = e / (BK / 8), d = k0 + 8 * (e % (BK / 8));
                fz[i] = load8(Z + srow[t] * g.z_rs + min(d, g.K), t < ns ? min(8, g.K - d) : 0, g.vec_z);
            }
#pragma unroll
            for (int i = 0; i < NW; ++i) {
                const int e = tid + i * NT, r = e / WC, d = 8 * (e % WC);
                const bool in = BWD ? k0 + r < g.K : m0 + r < g.M;
                const long at = BWD ? static_cast<long>(k0 + r) * g.M + m0 + d : static_cast<long>(m0 + r) * g.K + k0 + d;
                const int n = BWD ? g.M - m0 - d : g.K - k0 - d;
                fw[i] = load8(W + (in && n > 0 ? at : 0), in ? min(8, n) : 0, p.vec_w);
            }
        }
    };
    const auto landed = [&](T* tw, T* tz) __attribute__((always_inline)) {
        if constexpr (DIRECT) {
            wait_loads<0>();
        } else {
#pragma unroll
            for (int i = 0; i < NZ; ++i) Tz::put8(tz, (tid + i * NT) / (BK / 8), (tid + i * NT) % (BK / 8), fz[i]);
#pragma unroll
            for (int i = 0; i < NW; ++i) Tw::put8(tw, (tid + i * NT) / WC, (tid + i * NT) % WC, fw[i]);
        }
    };
    f32x16 acc[MB][2];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x16{};
    if (c0 < c1) load(c0, sw0, sz0);
    const int u0 = BWD ? 0 : unit_at(p.unit_off, p.units, wm);
    const int u1 = BWD ? p.units : unit_at(p.unit_off, p.units, min(wm + 32 * MB - 1, g.M - 1)) + 1;
    unsigned long long wild = 0;
    low_rank<T, BWD>(p, g.M, wm, u0, u1, srow[wn + lane], sid[wn + lane], split, g.splits, acc, wild);
    if (DIRECT && BIG) {  // formed again rather than held meanwhile
        asm volatile("" ::: "memory");
        z_offsets(g.K - c0 * BK);
    }
    if (BWD && p.dropping) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int i = 0; i < MB; ++i)
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
                    __builtin_amdgcn_sched_barrier(0);  // one mask's registers at a time
                }
    }
    const auto operands = [&](int k, const T* tw, const T* tz, Frag<T> (&w)[MB], Frag<T> (&z)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            if constexpr (BWD) w[i] = lds_cols<GM, false>(tw, 16 * k, wf + 32 * i);
            else w[i] = lds_rows<T, BK>(tw, wf + 32 * i, k);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) z[j] = lds_rows<T, BK>(tz, wn + 32 * j, k);
    };
    const auto products = [&](const Frag<T> (&w)[MB], const Frag<T> (&z)[2]) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) acc[i][j] = mma32(w[i], z[j], acc[i][j]);
    };
    if (c0 < c1) {
        landed(sw0, sz0);
        lds_barrier();
    }
    if constexpr (BIG) {
        // A step is four products deep. Each one's operands are read under the
        // one before, across the barrier too: before a step's last products
        // the next tile is awaited, and the tile after it sent for, to the
        // place of this step's, whose operands all are in registers by then.
        Frag<T> w[2][MB], z[2][2];
        if (c0 < c1) {
            if (c0 + 1 < c1) load(c0 + 1, sw1, sz1);
            operands(0, sw0, sz0, w[0], z[0]);
        }
        const auto walk = [&](int c, T* tw, T* tz, T* nw, T* nz) __attribute__((always_inline)) {
#pragma unroll
            for (int k = 0; k < 3; ++k) {
                operands(k + 1, tw, tz, w[(k + 1) & 1], z[(k + 1) & 1]);
                __builtin_amdgcn_sched_barrier(0);
                products(w[k & 1], z[k & 1]);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (c + 1 < c1) {
                landed(nw, nz);
                lds_barrier();
                if (c + 2 < c1) load(c + 2, tw, tz);
                operands(0, nw, nz, w[0], z[0]);
                __builtin_amdgcn_sched_barrier(0);
            }
            products(w[1], z[1]);
        };
        for (int c = c0; c < c1; c += 2) {
            walk(c, sw0, sz0, sw1, sz1);
            if (c + 1 < c1) walk(c + 1, sw1, sz1, sw0, sz0);
        }
    } else {
        const auto walk = [&](int c, const T* tw, const T* tz, T* nw, T* nz) __attribute__((always_inline)) {
            if (c + 1 < c1) load(c + 1, nw, nz);
#pragma unroll
            for (int k = 0; k < BK / 16; ++k) {
                Frag<T> w[MB], z[2];
                operands(k, tw, tz, w, z);
                products(w, z);
            }
            if (c + 1 < c1) landed(nw, nz);
            lds_barrier();
        };
        for (int c = c0; c < c1; c += 2) {
            walk(c, sw0, sz0, sw1, sz1);
            if (c + 1 < c1) walk(c + 1, sw1, sz1, sw0, sz0);
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int t = wn + 32 * j + col;
        if (t >= ns) continue;
        const long row = srow[t];
#pragma unroll
        for (int i = 0; i < MB; ++i)
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
    if (wild) {
        const int row = srow[wn + lane], id = sid[wn + lane];
        if (g.splits > 1)
            wild_sums<T, BWD>(p, g.M, wm, 32 * MB, u0, u1, row, id, wild, g.part + split * static_cast<long>(p.T) * g.M, g.M);
        else
            wild_sums<T, BWD>(p, g.M, wm, 32 * MB, u0, u1, row, id, wild, static_cast<T*>(g.Y), g.y_rs);
    }
}

// The splits' sums, rounded once: 64 values per block, its sixteen waves
// taking the splits in turn and their sums added in order.
template <class T>
__global__ __launch_bounds__(1024) void adapter_join_k(const float* part, int splits, long n, int M, T* Y, long y_rs) {
    __shared__ float sum[16][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long e = static_cast<long>(blockIdx.x) * 64 + lane;
    float s = 0.0f;
    if (e < n)
#pragma unroll 4
        for (int i = wave; i < splits; i += 16) s += part[i * n + e];
    sum[wave][lane] = s;
    __syncthreads();
    if (wave || e >= n) return;
    for (int w = 1; w < 16; ++w) s += sum[w][lane];
    const long row = e / M;
    Y[row * y_rs + (e - row * M)] = static_cast<T>(s);
}

// The same for few rows and 32 features: two of the taker's pairs of adapter
// and unit at a time, the loads of both in flight.
template <class T, int NB>
__device__ inline void low_rank_few(const Adapter& p, int M, int m0, int u0, int u1, int id, int turn, int turns, f32x16 (&acc)[NB],
                                    unsigned long long& wild) {
    const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31, m = m0 + col;
    unsigned long long left = __builtin_amdgcn_ballot_w64(id < p.n);
    int rows[NB], ids[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
        rows[j] = min(32 * j + col, p.T - 1);
        ids[j] = __shfl(id, 32 * j + col);
    }
    int a = -1, u = u0 + turn;
    unsigned long long mine = 0;
    const auto next = [&]() __attribute__((always_inline)) {  // moves to the taker's next pair
        if (a >= 0) u += turns;
        while (a < 0 || u >= u1) {
            if (a >= 0) u -= u1 - u0;
            if (!left) return false;
            a = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
            mine = __builtin_amdgcn_ballot_w64(id == a);
            left &= ~mine;
        }
        return true;
    };
    for (bool more = next(); more;) {
        int as[2], us[2];
        unsigned long long mines[2];
        as[0] = as[1] = a, us[0] = us[1] = u, mines[0] = mine, mines[1] = 0;
        more = next();
        if (more) {
            as[1] = a, us[1] = u, mines[1] = mine;
            more = next();
        }
        bool in[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) in[i] = m >= p.unit_off[us[i]] && m < p.unit_off[us[i] + 1] && m < M;
        for (int k = 0; k < p.rank; k += 16) {
            const int d = k + 8 * half, n = min(8, p.rank - d), dd = n > 0 ? d : 0;
            Frag<T> w[2];
            f32x8 h[2][NB];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                w[i] = load8(static_cast<const T*>(p.B) + (static_cast<long>(as[i]) * p.out + (in[i] ? m : 0)) * p.rank + dd, in[i] ? n : 0,
                             p.vec_b);
#pragma unroll
                for (int j = 0; j < NB; ++j)
                    h[i][j] = load8(p.H + static_cast<long>(rows[j]) * p.R + us[i] * p.rank + dd, ids[j] == as[i] ? n : 0, p.vec_h);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                bool bad = not_finite(w[i]);
#pragma unroll
                for (int j = 0; j < NB; ++j) bad |= not_finite(h[i][j]);
                if (__builtin_amdgcn_ballot_w64(bad)) {
                    w[i] = finite_part(w[i]);
#pragma unroll
                    for (int j = 0; j < NB; ++j) h[i][j] = finite_part(h[i][j]);
                    wild |= mines[i];
                    asm volatile("");  // a branch
                }
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    if (!(mines[i] >> (32 * j) & 0xFFFFFFFFull)) continue;
                    const Terms<T, 2> v(h[i][j]);
#pragma unroll
                    for (int x = 0; x < v.n; ++x) acc[j] = mma32(w[i], v.t[x], acc[j]);
                }
            }
        }
    }
}

// Up to 64 rows, unsorted: a block forms 32 features of all of them, its eight
// waves taking the depth (and then the adapters) in turn. W is read once, four
// steps' loads in flight.
template <class T, int NB>
__global__ __launch_bounds__(LT) void adapter_few_k(Adapter p, Product g) {
    __shared__ Join8 buf[8];
    __shared__ unsigned long long swild[8];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5, col = lane & 31;
    const int m0 = blockIdx.x * 32, m = m0 + col;
    const int id = lane < p.T ? adapter_of(p, lane) : p.n;
    const T* w = static_cast<const T*>(p.W) + static_cast<long>(min(m, g.M - 1)) * g.K;
    const T* x[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) x[j] = static_cast<const T*>(g.Z) + min(32 * j + col, p.T - 1) * g.z_rs;
    f32x16 acc[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) acc[j] = f32x16{};
    for (int k = 16 * wave; k < g.K; k += 512) {
        Frag<T> f[4], z[4][NB];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int d = k + 128 * s + 8 * half, n = min(8, g.K - d), dd = n > 0 ? d : 0;
            f[s] = load8(w + dd, m < g.M ? n : 0, p.vec_w);
#pragma unroll
            for (int j = 0; j < NB; ++j) z[s][j] = load8(x[j] + dd, 32 * j + col < p.T ? n : 0, g.vec_z);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (k + 128 * s >= g.K) break;
#pragma unroll
            for (int j = 0; j < NB; ++j) acc[j] = mma32(f[s], z[s][j], acc[j]);
        }
    }
    const int u0 = unit_at(p.unit_off, p.units, m0), u1 = unit_at(p.unit_off, p.units, min(m0 + 31, g.M - 1)) + 1;
    unsigned long long wild = 0;
    low_rank_few<T, NB>(p, g.M, m0, u0, u1, id, wave, 8, acc, wild);
    if (lane == 0) swild[wave] = wild;
#pragma unroll
    for (int j = 0; j < NB; ++j)
        join8(buf, acc[j], [&](int r, int c, float v) {
            const int t = 32 * j + c;
            if (t >= p.T || m0 + r >= g.M) return;
            if (p.bias) v += static_cast<float>(static_cast<const T*>(p.bias)[m0 + r]);
            static_cast<T*>(g.Y)[t * g.y_rs + m0 + r] = static_cast<T>(v);
        });
#pragma unroll
    for (int w = 0; w < 8; ++w) wild |= swild[w];
    if (!wild) return;  // all waves or none
    __threadfence();
    __syncthreads();
    if (!wave) wild_sums<T, false>(p, g.M, m0, 32, u0, u1, lane, id, wild, static_cast<T*>(g.Y), g.y_rs);
}

// Sums over a chunk's rows: C[m, c] = f sum_t P[t, m] Z[t, c] for 32 columns m
// of the float matrix P (H or dH, width R) and 128 columns c of X or dY.
// dA = dH^T drop(X): all of P's columns. dB^T = H^T dY: the columns of the
// unit that c lies in. Steps of 64 rows through shared memory, the next
// step's loads in flight. Where every adapter is one chunk (T <= CHUNK) the
// sums are the gradients; else they go to `part` (chunks, the gradient's
// adapter) and adapter_grad_k adds them.
template <class T, bool DB>
__global__ __launch_bounds__(NT) void adapter_outer_k(Adapter p, const float* P, const T* Z, long z_rs, int C, bool vec_z,
                                                      float* out, float beta, float* part, int mt) {
    constexpr int NTERM = Terms<T, 3, true>::n, ROWS = 64, NZ = ROWS * 16 / NT;
    __shared__ __align__(16) T sz[ROWS * 128];
    __shared__ __align__(16) T sp[NTERM][ROWS * 64];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5, col = lane & 31;
    const int ct = (C + 127) / 128;
    const int c0 = (blockIdx.x % ct) * 128, m0 = (blockIdx.x / ct % mt) * 32;
    const int chunk = blockIdx.x / ct / mt;
    const Piece pc = p.chunks[chunk];
    const int a = pc.adapter;
    if (a >= p.n || (part && !pc.count)) return;
    if (!part && chunk > 0 && p.chunks[chunk - 1].adapter == a) return;  // the adapter's empty last entry
    const int cols = DB ? p.rank : p.R;  // P's columns that a block's m counts
    const float f = !DB && p.dropping ? p.drop.keep : 1.0f;
    const int u0 = DB ? unit_at(p.unit_off, p.units, c0) : 0;
    const int u1 = DB ? unit_at(p.unit_off, p.units, min(c0 + 127, C - 1)) + 1 : 1;
    for (int u = u0; u < u1; ++u) {
        const float* base = P + (DB ? u * p.rank : 0);
        f32x16 acc = f32x16{};
        Frag<T> z[NZ];
        f32x8 h;
        int rows[NZ];
        const auto load = [&](int s) {
#pragma unroll
            for (int i = 0; i < NZ; ++i) {
                const int e = tid + i * NT, t = s + (e >> 4), d = c0 + 8 * (e & 15);
                rows[i] = t < pc.count ? p.perm[pc.start + t] : 0;
                z[i] = load8(Z + rows[i] * z_rs + min(d, C), t < pc.count ? min(8, C - d) : 0, vec_z);
            }
            const int t = s + (tid >> 2), d = m0 + 8 * (tid & 3), row = t < pc.count ? p.perm[pc.start + t] : 0;
            h = load8(base + static_cast<long>(row) * p.R + min(d, cols), t < pc.count ? min(8, cols - d) : 0, p.vec_h);
        };
        if (pc.count) load(0);
        for (int s = 0; s < pc.count; s += ROWS) {
#pragma unroll
            for (int i = 0; i < NZ; ++i) {
                const int e = tid + i * NT;
                if (!DB && p.dropping) z[i] = dropped<T>(p.drop, rows[i], c0 + 8 * (e & 15), z[i]);
                Tile<T, 128>::put8(sz, e >> 4, e & 15, z[i]);
            }
            const Terms<T, 3, true> v(h);
#pragma unroll
            for (int x = 0; x < NTERM; ++x) Tile<T, 64>::put8(sp[x], tid >> 2, tid & 3, v.t[x]);
            __syncthreads();
            if (s + ROWS < pc.count) load(s + ROWS);
#pragma unroll
            for (int k = 0; k < ROWS / 16; ++k) {
                Frag<T> w = lds_cols<128, false>(sz, 16 * k, 32 * wave);
#pragma unroll
                for (int x = 0; x < NTERM; ++x) {
                    acc = mma32(lds_cols<64, false>(sp[x], 16 * k, 0), w, acc);
                    // values that are not finite meet P's first term alone
                    if (NTERM > 1 && x == 0 && __builtin_amdgcn_ballot_w64(not_finite(w))) w = finite_part(w);
                }
            }
            __syncthreads();
        }
        const int c = c0 + 32 * wave + col;
        if (c >= C || (DB && (c < p.unit_off[u] || c >= p.unit_off[u + 1]))) continue;
        const long size = DB ? static_cast<long>(C) * p.rank : static_cast<long>(p.R) * C;
        float* to = part ? part + chunk * size : out + a * size;
        const bool add = !part && beta != 0.0f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int m = m0 + 8 * q + 4 * half;
            if (DB && p.vec_h && !add) {  // four of a row
                store4(to + static_cast<long>(c) * p.rank + m, cols - m, true, acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
                continue;
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                if (m + x >= cols) continue;
                float* o = DB ? to + static_cast<long>(c) * p.rank + m + x : to + static_cast<long>(m + x) * C + c;
                *o = add ? beta * *o + f * acc[4 * q + x] : f * acc[4 * q + x];
            }
        }
    }
}

// The gradients of up to 64 rows: an adapter has few of them, and what counts
// is writing its gradients (dB of 16 voices, 35000 outputs of rank 16: 36 MB in
// 18 us). Four values a thread, the rows in turn.
// dA[m, c] = sum_t dH[t, m] drop(X)[t, c], dB[c, m] = sum_t H[t, u(c) rank + m] dY[t, c].
template <class T, bool DB>
__global__ __launch_bounds__(NT) void adapter_outer_few_k(Adapter p, const float* P, const T* Z, long z_rs, int C, bool vec,
                                                          float* out, float beta) {
    const int chunk = blockIdx.y;
    const Piece pc = p.chunks[chunk];
    const int a = pc.adapter;
    if (a >= p.n || (chunk > 0 && p.chunks[chunk - 1].adapter == a)) return;  // (the adapter's empty last entry)
    const int width = DB ? p.rank : C, q = (width + 3) / 4;  // a row of the gradient, in fours
    const long n = static_cast<long>(DB ? C : p.R) * q;
    const long e = static_cast<long>(blockIdx.x) * NT + threadIdx.x;
    const int r = static_cast<int>(min(e, n - 1) / q), x = 4 * static_cast<int>(e - static_cast<long>(r) * q);
    int u = 0;
    if (DB) {  // the wave's first row's unit, and on from there
        u = unit_at(p.unit_off, p.units, __builtin_amdgcn_readfirstlane(r));
        while (u + 1 < p.units && p.unit_off[u + 1] <= r) ++u;
    }
    if (e >= n) return;
    float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int t = 0; t < pc.count; ++t) {
        const int row = p.perm[pc.start + t];
        float v[4], f;
        if (DB) {
            const float* h = P + static_cast<long>(row) * p.R + u * p.rank + x;
            f = static_cast<float>(Z[row * z_rs + r]);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = x + i < width ? h[i] : 0.0f;
        } else {
            f = P[static_cast<long>(row) * p.R + r];
            unsigned w[4];
            if (p.dropping) drop_words(p.drop, static_cast<unsigned>(row), static_cast<unsigned>(x) >> 3, w);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[i] = x + i < width ? static_cast<float>(Z[row * z_rs + x + i]) : 0.0f;
                if (p.dropping) v[i] = kept(p.drop, w, (x & 7) + i) ? v[i] * p.drop.keep : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = __builtin_fmaf(f, v[i], s[i]);
    }
    float* o = out + (static_cast<long>(a) * (DB ? C : p.R) + r) * width + x;
    if (vec && beta == 0.0f) {
        *reinterpret_cast<f32x4*>(o) = f32x4{s[0], s[1], s[2], s[3]};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (x + i < width) o[i] = beta == 0.0f ? s[i] : beta * o[i] + s[i];
}

// An adapter's chunks' sums in their order; adapters without rows get zeros.
__global__ __launch_bounds__(NT) void adapter_grad_k(const Piece* chunks, int table, const float* part, long size, float* out,
                                                     float beta, int a0) {
    __shared__ int range[2];
    const int a = a0 + blockIdx.y;
    if (threadIdx.x == 0) {  // the adapter's entries: [first, next), found by their adapter
        int lo = 0, hi = table;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (chunks[mid].adapter < a) lo = mid + 1;
            else hi = mid;
        }
        range[0] = lo;
        while (lo < table && chunks[lo].adapter == a && chunks[lo].count) ++lo;
        range[1] = lo;
    }
    __syncthreads();
    const long e = static_cast<long>(blockIdx.x) * NT + threadIdx.x;
    if (e >= size) return;
    float s = 0.0f;
#pragma unroll 4
    for (int i = range[0]; i < range[1]; ++i) s += part[i * size + e];
    float* o = out + a * size + e;
    *o = beta == 0.0f ? s : beta * *o + s;
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
    if (T > INT_MAX / 2 || in > (1 << 24) || out > (1 << 24) || adapters > (1 << 20)) return bad("sizes too large");
    if (!make_drop(prob, seed, offset, p.drop)) return bad("p must be at least 0 and below 1");
    p.dropping = p.drop.thr != 0;
    return KDEC_OK;
}

size_t up(size_t n) { return (n + 255) & ~size_t(255); }

// The sort's workspace: rows, pieces, chunks.
struct Sorted {
    size_t perm, pieces, chunks;
    int chunk;  // rows of a chunk
    long n_pieces, n_chunks;
    Sorted(int T, int adapters)
        : perm(up(T * 4ul)), chunk(static_cast<int>(cdiv(T > 0 ? T : 1, static_cast<long>(CHUNK) * CHUNKS)) * CHUNK),
          n_pieces(T / PIECE + adapters + 1), n_chunks(T / chunk + adapters + 1) {
        pieces = up(n_pieces * sizeof(Piece));
        chunks = up(n_chunks * sizeof(Piece));
    }
    size_t bytes() const { return perm + pieces + chunks; }
    void sort(kdec_ctx* ctx, Adapter& p, char* ws) const {
        int* rows = reinterpret_cast<int*>(ws);
        Piece *a = reinterpret_cast<Piece*>(ws + perm), *b = reinterpret_cast<Piece*>(ws + perm + pieces);
        hipLaunchKernelGGL(adapter_sort_k, dim3(p.n + 1), dim3(ST), 0, ctx->stream, p.idx, p.T, p.n, chunk, rows, a, b);
        p.perm = rows;
        p.pieces = a;
        p.chunks = b;
    }
};

template <class T>
void low_inputs(kdec_ctx* ctx, const Adapter& p, long pieces) {
    const unsigned x = static_cast<unsigned>(p.pieces ? pieces : p.T);
    if (p.R > 32)
        hipLaunchKernelGGL((adapter_h_k<T, 2>), dim3(x, static_cast<unsigned>(cdiv(p.R, 64))), dim3(LT), 0, ctx->stream, p);
    else
        hipLaunchKernelGGL((adapter_h_k<T, 1>), dim3(x, 1), dim3(LT), 0, ctx->stream, p);
}

template <class T, bool BWD>
int product(kdec_ctx* ctx, const Adapter& p, Product g) {
    const long tiles = cdiv(g.M, 128) * cdiv(p.T, 128), big = cdiv(g.M, 256) * cdiv(p.T, 256);
    if (tiles >= INT_MAX) return fail(ctx, KDEC_EINVAL, "kdec_adapter: too many rows");
    const long bytes = ((p.T - 1) * g.z_rs + g.K) * static_cast<long>(sizeof(T));
    const long reach = 256L * (BWD ? g.M : g.K) * static_cast<long>(sizeof(T));  // of a tile's offsets in W
    const dim3 grid(static_cast<unsigned>(tiles), g.splits);
    if (!(p.vec_w && g.vec_z && g.z_rs >= 0 && bytes < 0xFFFF0000L && reach < (1L << 30)))
        hipLaunchKernelGGL((adapter_gemm_k<T, BWD, false, false>), grid, dim3(256), 0, ctx->stream, p, g);
    // Big tiles where they reach seven CUs of eight (1024 -> 4096, forward:
    // 3500 rows 54 us for the small ones' 62, 2048 rows, half the CUs, 51 for 40).
    else if (sizeof(T) == 2 && g.splits == 1 && 8 * big >= 7 * ctx->num_cus)
        hipLaunchKernelGGL((adapter_gemm_k<bf16, BWD, true, true>), dim3(static_cast<unsigned>(big)), dim3(512), 0, ctx->stream, p, g);
    else
        hipLaunchKernelGGL((adapter_gemm_k<T, BWD, true, false>), grid, dim3(256), 0, ctx->stream, p, g);
    if (g.splits > 1) {
        const long n = static_cast<long>(p.T) * g.M;
        hipLaunchKernelGGL(adapter_join_k<T>, dim3(static_cast<unsigned>(cdiv(n, 64))), dim3(1024), 0, ctx->stream, g.part, g.splits,
                           n, g.M, static_cast<T*>(g.Y), g.y_rs);
    }
    return KDEC_OK;
}

template <class T>
int forward(kdec_ctx* ctx, const Adapter& p, const Product& g, long pieces) {
    low_inputs<T>(ctx, p, pieces);
    if (!p.pieces) {
        const dim3 grid(static_cast<unsigned>(cdiv(g.M, 32)));
        if (p.T <= 32) hipLaunchKernelGGL((adapter_few_k<T, 1>), grid, dim3(LT), 0, ctx->stream, p, g);
        else hipLaunchKernelGGL((adapter_few_k<T, 2>), grid, dim3(LT), 0, ctx->stream, p, g);
    } else if (int rc = product<T, false>(ctx, p, g)) {
        return rc;
    }
    return launch_check(ctx, "kdec_adapter_fwd");
}

struct Grads {
    float *dA, *dB, beta, *part_a, *part_b;  // parts: null where every adapter is one chunk
    long n_chunks;
};

template <class T, bool DB>
int grads(kdec_ctx* ctx, const Adapter& p, const Grads& gr, const float* P, const void* Z, long z_rs, int C, bool vec_z, float* out,
          float* part, long size) {
    if (p.T <= FEW && gr.n_chunks <= 65535) {
        const int width = DB ? p.rank : C;
        const long n = static_cast<long>(DB ? C : p.R) * cdiv(width, 4);
        if (cdiv(n, NT) >= INT_MAX) return fail(ctx, KDEC_EINVAL, "kdec_adapter_bwd: too many adapters");
        hipLaunchKernelGGL((adapter_outer_few_k<T, DB>), dim3(static_cast<unsigned>(cdiv(n, NT)), static_cast<unsigned>(gr.n_chunks)),
                           dim3(NT), 0, ctx->stream, p, P, static_cast<const T*>(Z), z_rs, C, width % 4 == 0 && aligned16(out, 0), out,
                           gr.beta);
        return KDEC_OK;
    }
    const long mt = cdiv(DB ? p.rank : p.R, 32), blocks = cdiv(C, 128) * mt * gr.n_chunks;
    if (blocks >= INT_MAX || cdiv(size, NT) >= INT_MAX) return fail(ctx, KDEC_EINVAL, "kdec_adapter_bwd: too many adapters");
    hipLaunchKernelGGL((adapter_outer_k<T, DB>), dim3(static_cast<unsigned>(blocks)), dim3(NT), 0, ctx->stream, p, P,
                       static_cast<const T*>(Z), z_rs, C, vec_z, out, gr.beta, part, static_cast<int>(mt));
    if (part)
        for (int a = 0; a < p.n; a += 65535)  // the grid's second dimension ends there
            hipLaunchKernelGGL(adapter_grad_k, dim3(static_cast<unsigned>(cdiv(size, NT)), static_cast<unsigned>(p.n - a < 65535 ? p.n - a : 65535)),
                               dim3(NT), 0, ctx->stream, p.chunks, static_cast<int>(gr.n_chunks), part, size, out, gr.beta, a);
    return KDEC_OK;
}

template <class T>
int backward(kdec_ctx* ctx, const Adapter& p, const Product& g, const Grads& gr, long pieces) {
    if (p.T > 0)
        hipLaunchKernelGGL(adapter_dh_k<T>, dim3(static_cast<unsigned>(pieces), static_cast<unsigned>(p.units * cdiv(p.rank, 32))),
                           dim3(LT), 0, ctx->stream, p);
    if (p.T > 0 && g.Y)
        if (int rc = product<T, true>(ctx, p, g)) return rc;
    if (gr.dA && p.n > 0) {
        if (int rc = grads<T, false>(ctx, p, gr, p.dH, p.X, p.x_rs, p.in, p.vec_x, gr.dA, gr.part_a, static_cast<long>(p.R) * p.in))
            return rc;
        if (int rc = grads<T, true>(ctx, p, gr, p.H, p.dY, p.dy_rs, p.out, p.vec_dy, gr.dB, gr.part_b,
                                    static_cast<long>(p.out) * p.rank))
            return rc;
    }
    return launch_check(ctx, "kdec_adapter_bwd");
}

// Whether four values of a row of Y can be stored at once.
bool stores4(const void* Y, long rs, int cols, size_t es) {
    return cols % 4 == 0 && reinterpret_cast<size_t>(Y) % (4 * es) == 0 && (rs * es) % (4 * es) == 0;
}

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
    const Sorted sorted(T, adapters);
    const size_t h_b = H ? 0 : up(static_cast<size_t>(T) * R * 4);
    Workspace ws(ctx, sorted.bytes() + h_b);
    if (!ws.p) return KDEC_ENOMEM;
    p.H = H ? H : reinterpret_cast<float*>(ws.as<char>() + sorted.bytes());
    p.vec_h = rank % 8 == 0 && aligned16(p.H, 0);
    // (bf16, 1024 -> 1536, 12 adapters: 8 rows 14 us for 29 sorted, 64 rows 16 for 36)
    if (T > FEW) sorted.sort(ctx, p, ws.as<char>());
    const Product g{out, in, X, x_rs, p.vec_x, Y, y_rs, stores4(Y, y_rs, out, es), 1, nullptr};
    return dtype == KDEC_F32 ? forward<float>(ctx, p, g, sorted.n_pieces) : forward<bf16>(ctx, p, g, sorted.n_pieces);
}

int kdec_adapter_bwd(kdec_ctx* ctx, int dtype, const void* X, long x_rs, const void* W, const void* A, const void* B,
                     const float* scale, const int* idx, const int* unit_off, int T, int in, int out, int adapters, int units,
                     int rank, float prob, long seed, long offset, const float* H, const void* dY, long dy_rs, void* dX,
                     long dx_rs, float* dA, float* dB, float beta) {
    if (!ctx) return KDEC_EINVAL;
    Adapter p{};
    if (int rc = check(ctx, "kdec_adapter_bwd", dtype, T, in, out, adapters, units, rank, prob, seed, offset, p)) return rc;
    KDEC_CHECK(ctx, !dA == !dB, "kdec_adapter_bwd: dA and dB go together");
    KDEC_CHECK(ctx, T == 0 || (X && W && H && dY && idx), "kdec_adapter_bwd: null tensor");
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
    // than 64 deep each (from 256 on: two blocks' sums cost more to join).
    const long tiles = cdiv(in, 128) * cdiv(T, 128);
    long splits = dX && T > 0 ? cdiv(2L * ctx->num_cus, tiles) : 1;
    if (splits > out / 64) splits = out < 256 ? 1 : out / 64;
    if (splits < 1) splits = 1;
    const Sorted sorted(T, adapters);
    const size_t h_b = up(static_cast<size_t>(T) * R * 4), s_b = splits > 1 ? up(static_cast<size_t>(splits) * T * in * 4) : 0;
    const bool parts = dA && T > sorted.chunk;
    const size_t a_b = parts ? up(static_cast<size_t>(sorted.n_chunks) * R * in * 4) : 0;
    const size_t b_b = parts ? up(static_cast<size_t>(sorted.n_chunks) * out * rank * 4) : 0;
    Workspace ws(ctx, sorted.bytes() + h_b + s_b + a_b + b_b);
    if (!ws.p) return KDEC_ENOMEM;
    char* at = ws.as<char>() + sorted.bytes();
    p.H = const_cast<float*>(H);
    p.dH = reinterpret_cast<float*>(at);
    p.vec_h = rank % 8 == 0 && aligned16(H, 0) && aligned16(dB, 0);
    sorted.sort(ctx, p, ws.as<char>());
    const Product g{in, out, dY, dy_rs, p.vec_dy, dX, dx_rs, dX && stores4(dX, dx_rs, in, es), static_cast<int>(splits),
                    reinterpret_cast<float*>(at + h_b)};
    const Grads gr{dA, dB, beta, parts ? reinterpret_cast<float*>(at + h_b + s_b) : nullptr,
                   parts ? reinterpret_cast<float*>(at + h_b + s_b + a_b) : nullptr, sorted.n_chunks};
    return dtype == KDEC_F32 ? backward<float>(ctx, p, g, gr, sorted.n_pieces) : backward<bf16>(ctx, p, g, gr, sorted.n_pieces);
}

}  // extern "C"
