// The norms before and after a block with its gate and residual, in one pass
// each way on gfx950:
//
//   u = N_post(z) (or z),  r = x_scale x + scale g u,  y = N_pre(r)
//
// N is the RMS or the layer norm of a row with weight and bias. A row lies in
// the registers of 1 to 8 waves, eight neighbouring columns a lane at a time,
// so that each tensor is read once and statistics are formed from the values
// (the layer norm's variance around its mean). r enters the second norm
// unrounded.
//
// The backward forms r again from x and z with the kept statistics (reading r
// instead would cost the same and bring its rounding into the gradients):
//   e = dy w2;  d = dr + s2 (e - [mean e] - r^ mean(e r^));  dx = x_scale d
//   du = scale g d;  dg = scale u d;  f = du w1
//   dz = s1 (f - [mean f] - z^ mean(f z^))
// and sums dw1 = du z^, db1 = du, dw2 = dy r^, db2 = dy, and dg of a column's
// gate over the rows: every block over its rows in registers, a second kernel
// over the blocks in their order.
//
// Bound by memory where rows are many: 8192 x 2048, bf16, a gate for each row,
// forward 38 us for 168 MB (4.5 TB/s; a large copy reaches 5.1), backward 54 and 5
// for 268; 2050 x 5120 forward 18.6 for 84 MB; 4093 x 768, float, layer norms,
// 12.7 for 50 MB, then 21 and 4 for 75. Past 4096 columns the backward waits for its
// rows, one at a time: 2048 x 5120 with a gate for each row 61 and 5 us for 168 MB,
// 1024 x 8192 47 and 5 for 134. 16 rows of 1024 take 3.6 us, a launch and three
// reductions.
#include "kdec_frag.hpp"
#include "kdec_internal.hpp"

#include <climits>
#include <cmath>
#include <type_traits>

namespace kdec {
namespace {

constexpr int MOST = 8192;  // columns that a row's registers hold

struct Rows {
    const void* p;
    long rs;
};

struct Norm {
    Rows x, z, gate;  // gate: rs 0 for one row of gates
    const void *w1, *b1, *w2, *b2;
    int T, C;
    bool post, pre, layer, vec;
    float eps, scale, x_scale;
    float* stats;  // (T, 4): mean and 1 / deviation of z's norm, of r's
    void *r, *y;
    long r_rs, y_rs;
};

// A row's waves and a block's rows: W is 1 or 2, with 4 or 2 rows a block, or 0
// for one row in as many waves as the block has.
template <int W>
struct Block {
    static constexpr int R = W ? 4 / W : 1, MAX = W ? 256 : 512;
    __device__ static inline int waves() { return W ? W : blockDim.x >> 6; }
};

// The sum over a wave's lanes, in all of them.
__device__ inline float wave_sum(float x) {
    const auto add = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
        x += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), decltype(ctrl)::value, decltype(rows)::value, 15, false));
    };
    typedef std::integral_constant<int, 15> All;
    add(std::integral_constant<int, 0x111>{}, All{});  // lanes of 16 to the right by 1, 2, 4, 8
    add(std::integral_constant<int, 0x112>{}, All{});
    add(std::integral_constant<int, 0x114>{}, All{});
    add(std::integral_constant<int, 0x118>{}, All{});
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 10>{});  // the 16's last lane to the next 16
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 12>{});  // lane 31 to the upper half
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}

// Two sums over a row's lanes, the same in all of them. Waves of a row meet in
// shared memory, in two buffers in turn so that one barrier a sum is enough.
typedef float Meet[2][2][8];  // buffer, sum, wave of the row (or row and wave)
template <int W>
__device__ inline void row_sums(float& a, float& b, Meet& red, int& turn) {
    a = wave_sum(a);
    b = wave_sum(b);
    if (W == 1) return;
    const int wave = threadIdx.x >> 6, n = W ? W : blockDim.x >> 6, first = W ? wave / W * W : 0;
    if ((threadIdx.x & 63) == 0) {
        red[turn][0][wave] = a;
        red[turn][1][wave] = b;
    }
    __syncthreads();
    a = red[turn][0][first];
    b = red[turn][1][first];
    if constexpr (W == 2) {
        a += red[turn][0][first + 1];
        b += red[turn][1][first + 1];
    } else {
#pragma unroll
        for (int i = 1; i < 8; ++i) {  // past the row's waves the sums stay as they are
            a += i < n ? red[turn][0][i] : 0.0f;
            b += i < n ? red[turn][1][i] : 0.0f;
        }
    }
    turn ^= 1;
}

// Eight columns of a tensor's row, from byte offset `off` of it: zeros past the
// row's end or where the tensor is absent, without a branch around the load, so
// that a row's tensors are on their way together. Rows of other widths than
// multiples of 8 (or that start elsewhere) take eight loads: 4093 x 1021, bf16,
// forward 27 us and backward 37 where 1024 columns take 10.8 and 15, float 43 and 63
// for 14 and 22.
template <class T>
struct Raw {
    Frag<T> f;
    __device__ inline f32x8 floats() const {
        f32x8 r;
#pragma unroll
        for (int i = 0; i < 8; ++i) r[i] = static_cast<float>(f[i]);
        return r;
    }
};
template <class T, bool VEC>
__device__ inline Raw<T> load_raw(const Rows& t, long row, int C, int c) {
    const __amdgpu_buffer_rsrc_t r = uniform_rsrc(static_cast<const T*>(t.p) + row * t.rs, t.p ? C * static_cast<int>(sizeof(T)) : 0);
    Raw<T> x;
    if constexpr (VEC) {
        x.f = buffer_load8(r, c * static_cast<int>(sizeof(T)), T{});
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(T) == 2)
                x.f[i] = __builtin_bit_cast(bf16, static_cast<unsigned short>(__builtin_amdgcn_raw_buffer_load_b16(r, 2 * (c + i), 0, 0)));
            else
                x.f[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, 4 * (c + i), 0, 0));
        }
    }
    return x;
}
// The same of a vector of C, `none` where it is absent.
template <class T, bool VEC>
__device__ inline Raw<T> load_vector(const void* p, int C, int c, float none) {
    if (p) return load_raw<T, VEC>(Rows{p, 0}, 0, C, c);
    Raw<T> x;
#pragma unroll
    for (int i = 0; i < 8; ++i) x.f[i] = static_cast<T>(none);
    return x;
}
template <class T, bool VEC>
__device__ inline void store8(T* p, int n, const f32x8& v) {
    Frag<T> f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<T>(v[i]);
    if constexpr (VEC) {
        if (n > 0) *reinterpret_cast<Frag<T>*>(p) = f;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) p[i] = f[i];
    }
}

// A row's mean (0 for the RMS norm) and 1 / sqrt(mean square around it + eps).
template <int V, int W>
__device__ inline void moments(const Norm& p, const f32x8 (&u)[V], const int (&n)[V], Meet& red, int& turn, float& mean, float& rstd) {
    float s = 0.0f, none = 0.0f;
    mean = 0.0f;
    if (p.layer) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) s += u[v][i];  // zeros past the row's end
        row_sums<W>(s, none, red, turn);
        mean = s / static_cast<float>(p.C);
        s = none = 0.0f;
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float d = u[v][i] - mean;
            s = i < n[v] ? __builtin_fmaf(d, d, s) : s;
        }
    row_sums<W>(s, none, red, turn);
    rstd = 1.0f / sqrtf(s / static_cast<float>(p.C) + p.eps);
}

template <class T, int V, int W, bool VEC>
__global__ __launch_bounds__(Block<W>::MAX) void resnorm_k(Norm p) {
    __shared__ Meet red;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, waves = Block<W>::waves();
    const long row = static_cast<long>(blockIdx.x) * Block<W>::R + wave / waves;
    const bool live = row < p.T;
    const long at = live ? row : p.T - 1;
    int c[V], n[V], turn = 0;
    f32x8 x[V], u[V], g[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        c[v] = 512 * (v * waves + wave % waves) + 8 * lane;
        n[v] = max(min(8, p.C - c[v]), 0);
        x[v] = load_raw<T, VEC>(p.x, at, p.C, c[v]).floats();
        u[v] = load_raw<T, VEC>(p.z, at, p.C, c[v]).floats();
        g[v] = load_raw<T, VEC>(p.gate, at, p.C, c[v]).floats();
    }
    float m1 = 0.0f, s1 = 0.0f, m2 = 0.0f, s2 = 0.0f;
    if (p.z.p) {
        if (p.post) {
            Raw<T> w[V], b[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                w[v] = load_vector<T, VEC>(p.w1, p.C, c[v], 1.0f);
                b[v] = load_vector<T, VEC>(p.b1, p.C, c[v], 0.0f);
            }
            moments<V, W>(p, u, n, red, turn, m1, s1);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const f32x8 wf = w[v].floats(), bf = b[v].floats();
#pragma unroll
                for (int i = 0; i < 8; ++i) u[v][i] = __builtin_fmaf((u[v][i] - m1) * s1, wf[i], bf[i]);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float a = p.gate.p ? p.scale * g[v][i] : p.scale;
                x[v][i] = i < n[v] ? __builtin_fmaf(a, u[v][i], p.x_scale * x[v][i]) : 0.0f;
            }
            if (live) store8<T, VEC>(static_cast<T*>(p.r) + at * p.r_rs + c[v], n[v], x[v]);
        }
    }
    if (p.pre) {
        Raw<T> w[V], b[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            w[v] = load_vector<T, VEC>(p.w2, p.C, c[v], 1.0f);
            b[v] = load_vector<T, VEC>(p.b2, p.C, c[v], 0.0f);
        }
        moments<V, W>(p, x, n, red, turn, m2, s2);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const f32x8 wf = w[v].floats(), bf = b[v].floats();
            f32x8 y;
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = __builtin_fmaf((x[v][i] - m2) * s2, wf[i], bf[i]);
            if (live) store8<T, VEC>(static_cast<T*>(p.y) + at * p.y_rs + c[v], n[v], y);
        }
    }
    if (p.stats && live && lane == 0 && wave % waves == 0) *reinterpret_cast<f32x4*>(p.stats + 4 * at) = f32x4{m1, s1, m2, s2};
}

struct Back {
    Norm n;
    Rows dr, dy;
    void *dx, *dz, *dgate;  // dgate: (T, C) of the tensors' type
    float* part;            // (blocks, SUMS, C), the sums in use first
    int sums, at[5];        // where dw1, db1, dw2, db2 and the columns' dgate are among them, -1: not in use
};

// A row's tensors, and its kept statistics, as they are loaded.
template <class T, int V>
struct Row {
    Raw<T> x[V], z[V], g[V], dr[V], dy[V];
    f32x4 st;
};

// Blocks take rows in turn, the next row's tensors on their way.
template <class T, int V, int W, bool VEC>
__global__ __launch_bounds__(Block<W>::MAX) void resnorm_bwd_k(Back b) {
    constexpr int R = Block<W>::R;
    __shared__ Meet red;
    __shared__ float join[R > 1 ? R - 1 : 1][R > 1 ? 64 * W * 8 : 1];
    const Norm& p = b.n;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, waves = Block<W>::waves();
    int c[V], n[V], turn = 0;
    Raw<T> w1[V], b1[V], w2[V];
    f32x8 sum[5][V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        c[v] = 512 * (v * waves + wave % waves) + 8 * lane;
        n[v] = max(min(8, p.C - c[v]), 0);
        if (V == 1) {
            w1[v] = load_vector<T, VEC>(p.w1, p.C, c[v], 1.0f);
            b1[v] = load_vector<T, VEC>(p.b1, p.C, c[v], 0.0f);
            w2[v] = load_vector<T, VEC>(p.w2, p.C, c[v], 1.0f);
        }
#pragma unroll
        for (int k = 0; k < 5; ++k) sum[k][v] = f32x8{};
    }
    // A vector's columns: held over the rows, where the registers hold them.
    const auto vec = [&](const Raw<T>& held, const void* from, int v, float none) __attribute__((always_inline)) {
        return V == 1 ? held.floats() : load_vector<T, VEC>(from, p.C, c[v], none).floats();
    };
    const float over = 1.0f / static_cast<float>(p.C);
    const auto load = [&](long row0, Row<T, V>& o) __attribute__((always_inline)) {
        const long at = min(row0 + wave / waves, p.T - 1L);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            o.x[v] = load_raw<T, VEC>(p.x, at, p.C, c[v]);
            o.z[v] = load_raw<T, VEC>(p.z, at, p.C, c[v]);
            o.dr[v] = load_raw<T, VEC>(b.dr, at, p.C, c[v]);
            o.dy[v] = load_raw<T, VEC>(b.dy, at, p.C, c[v]);
            o.g[v] = load_raw<T, VEC>(p.gate, at, p.C, c[v]);
        }
        o.st = *reinterpret_cast<const f32x4*>(p.stats + 4 * at);
    };
    const auto take = [&](long row0, const Row<T, V>& o) __attribute__((always_inline)) {
        const long row = row0 + wave / waves;
        const bool live = row < p.T;
        const long at = live ? row : p.T - 1;
        f32x8 rh[V], zh[V], d[V];
        const f32x4 st = o.st;
        const auto gate = [&](int v) __attribute__((always_inline)) {
            f32x8 g = o.g[v].floats();
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] = p.gate.p ? p.scale * g[i] : p.scale;
            return g;
        };
        // the normalised rows
#pragma unroll
        for (int v = 0; v < V; ++v) {
            rh[v] = o.x[v].floats();
            zh[v] = o.z[v].floats();
            if (p.z.p) {
                const f32x8 g = gate(v), w = vec(w1[v], p.w1, v, 1.0f), bias = vec(b1[v], p.b1, v, 0.0f);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float u = zh[v][i];
                    if (p.post) {
                        zh[v][i] = (u - st[0]) * st[1];
                        u = __builtin_fmaf(zh[v][i], w[i], bias[i]);
                    }
                    rh[v][i] = __builtin_fmaf(g[i], u, p.x_scale * rh[v][i]);
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) rh[v][i] = (rh[v][i] - st[2]) * st[3];
            d[v] = o.dr[v].floats();
        }
        if (p.pre) {
            float e1 = 0.0f, e2 = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const f32x8 w = vec(w2[v], p.w2, v, 1.0f), dy = o.dy[v].floats();
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (live) {
                        sum[2][v][i] = __builtin_fmaf(dy[i], rh[v][i], sum[2][v][i]);
                        sum[3][v][i] += dy[i];
                    }
                    const float e = dy[i] * w[i];  // zero past the row's end
                    e1 += e;
                    e2 = i < n[v] ? __builtin_fmaf(e, rh[v][i], e2) : e2;
                }
            }
            row_sums<W>(e1, e2, red, turn);
            e1 = p.layer ? e1 * over : 0.0f;
            e2 *= over;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const f32x8 w = vec(w2[v], p.w2, v, 1.0f), dy = o.dy[v].floats();
#pragma unroll
                for (int i = 0; i < 8; ++i) d[v][i] += st[3] * (dy[i] * w[i] - e1 - rh[v][i] * e2);
            }
        }
        if (live)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                f32x8 x;
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = p.x_scale * d[v][i];
                store8<T, VEC>(static_cast<T*>(b.dx) + at * p.C + c[v], n[v], x);
            }
        if (!p.z.p) return;
        float f1 = 0.0f, f2 = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const f32x8 g = gate(v), w = vec(w1[v], p.w1, v, 1.0f);
            if (p.gate.p) {  // scale u d
                const f32x8 bias = vec(b1[v], p.b1, v, 0.0f);
                f32x8 x;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    x[i] = p.scale * (p.post ? __builtin_fmaf(zh[v][i], w[i], bias[i]) : zh[v][i]) * d[v][i];
                if (b.dgate) {
                    if (live) store8<T, VEC>(static_cast<T*>(b.dgate) + at * p.C + c[v], n[v], x);
                } else if (live) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum[4][v][i] += x[i];
                }
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                d[v][i] *= g[i];  // du
                if (p.post) {
                    if (live) {
                        sum[0][v][i] = __builtin_fmaf(d[v][i], zh[v][i], sum[0][v][i]);
                        sum[1][v][i] += d[v][i];
                    }
                    d[v][i] = i < n[v] ? d[v][i] * w[i] : 0.0f;
                    f1 += d[v][i];
                    f2 = i < n[v] ? __builtin_fmaf(d[v][i], zh[v][i], f2) : f2;
                }
            }
        }
        if (p.post) {
            row_sums<W>(f1, f2, red, turn);
            f1 = p.layer ? f1 * over : 0.0f;
            f2 *= over;
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) d[v][i] = st[1] * (d[v][i] - f1 - zh[v][i] * f2);
        }
        if (live)
#pragma unroll
            for (int v = 0; v < V; ++v) store8<T, VEC>(static_cast<T*>(b.dz) + at * p.C + c[v], n[v], d[v]);
    };
    const long step = static_cast<long>(gridDim.x) * R;
    long row0 = static_cast<long>(blockIdx.x) * R;
    Row<T, V> cur;
    if constexpr (V == 1) {
        Row<T, V> next;
        load(row0, cur);
        for (; row0 < p.T; row0 += step) {
            load(row0 + step, next);
            take(row0, cur);
            cur = next;
        }
    } else {  // two rows at once do not fit the registers
        for (; row0 < p.T; row0 += step) {
            load(row0, cur);
            take(row0, cur);
        }
    }
    // the block's rows together, then its share of every sum
#pragma unroll
    for (int k = 0; k < 5; ++k) {
        if (b.at[k] < 0) continue;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if constexpr (R > 1) {
                const int slot = wave / W, place = 8 * (threadIdx.x % (64 * W));
                __syncthreads();
                if (slot > 0)
#pragma unroll
                    for (int i = 0; i < 8; ++i) join[slot - 1][place + i] = sum[k][v][i];
                __syncthreads();
                if (slot > 0) continue;
                for (int s = 0; s < R - 1; ++s)
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum[k][v][i] += join[s][place + i];
            }
            float* to = b.part + (static_cast<long>(blockIdx.x) * b.sums + b.at[k]) * p.C + c[v];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n[v]) to[i] = sum[k][v][i];
        }
    }
}

// The blocks' shares: out k's columns, sixteen waves each a stretch of the
// blocks, their sums in order.
struct Outs {
    float* p[5];
};
constexpr int JW = 16;
__global__ __launch_bounds__(64 * JW) void resnorm_join_k(const float* part, int blocks, int sums, int C, Outs out) {
    __shared__ float s[JW][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), k = blockIdx.y;
    const int c = blockIdx.x * 64 + lane;
    float a = 0.0f;
    const int b0 = blocks * wave / JW, b1 = blocks * (wave + 1) / JW;
    if (c < C) {
        const float* from = part + static_cast<long>(k) * C + c;
        const long step = static_cast<long>(sums) * C;
#pragma unroll 8
        for (int i = b0; i < b1; ++i) a += from[i * step];
    }
    s[wave][lane] = a;
    __syncthreads();
    if (wave > 0 || c >= C) return;
    for (int w = 1; w < JW; ++w) a += s[w][lane];
    out.p[k][c] = a;
}

// A row's registers and waves: 512 columns a wave and register block.
struct Shape {
    int V, W, rows, threads;
};
Shape shape(int C) {
    const int V = C <= 4096 ? 1 : 2, W = static_cast<int>(cdiv(C, 512 * V)), rows = W <= 2 ? 4 / W : 1;
    return Shape{V, W, rows, 64 * W * rows};
}
template <class F>
void by_shape(const Shape& s, bool vec, F f) {
    const auto go = [&](auto V, auto W) {
        if (vec) f(V, W, std::true_type{});
        else f(V, W, std::false_type{});
    };
    typedef std::integral_constant<int, 0> Any;
    typedef std::integral_constant<int, 1> One;
    typedef std::integral_constant<int, 2> Two;
    if (s.V == 2) go(Two{}, Any{});
    else if (s.W == 1) go(One{}, One{});
    else if (s.W == 2) go(One{}, Two{});
    else go(One{}, Any{});
}

bool wide(const void* p, long rs, int es) { return reinterpret_cast<size_t>(p) % 16 == 0 && rs * es % 16 == 0; }

int fill(kdec_ctx* ctx, const char* who, int dtype, int layer, const void* X, long x_rs, const void* Z, long z_rs, const void* gate,
         long gate_rs, int post, const void* w1, const void* b1, int pre, const void* w2, const void* b2, float eps, float scale,
         float x_scale, int T, int C, Norm& p) {
    const auto bad = [&](const char* why) { return fail(ctx, KDEC_EINVAL, std::string(who) + ": " + why); };
    if (dtype != KDEC_F32 && dtype != KDEC_BF16) return bad("unknown type");
    if (T < 0 || C < 1 || C > MOST) return bad("columns outside 1..8192, or rows negative");
    if (!(eps > 0.0f && eps < HUGE_VALF)) return bad("eps must be positive");
    if (T > 0 && !X) return bad("null tensor");
    if (T > 0 && !Z && (post || gate)) return bad("a norm or a gate without the block's output");
    if (T > 0 && !Z && !pre) return bad("nothing to do");
    const int es = dtype == KDEC_F32 ? 4 : 2;
    p = Norm{};
    p.x = Rows{X, x_rs};
    p.z = Rows{Z, z_rs};
    p.gate = Rows{gate, gate_rs};
    p.w1 = post ? w1 : nullptr;
    p.b1 = post ? b1 : nullptr;
    p.w2 = pre ? w2 : nullptr;
    p.b2 = pre ? b2 : nullptr;
    p.T = T;
    p.C = C;
    p.post = post != 0;
    p.pre = pre != 0;
    p.layer = layer != 0;
    p.eps = eps;
    p.scale = scale;
    p.x_scale = Z ? x_scale : 1.0f;
    p.vec = C % 8 == 0 && wide(X, x_rs, es) && wide(Z, z_rs, es) && wide(gate, gate_rs, es) && wide(p.w1, 0, es) && wide(p.b1, 0, es) &&
            wide(p.w2, 0, es) && wide(p.b2, 0, es);
    return KDEC_OK;
}

}  // namespace
}  // namespace kdec

using namespace kdec;

extern "C" {

int kdec_resnorm_fwd(kdec_ctx* ctx, int dtype, int layer, const void* X, long x_rs, const void* Z, long z_rs, const void* gate,
                     long gate_rs, int post, const void* w1, const void* b1, int pre, const void* w2, const void* b2, float eps,
                     float scale, float x_scale, int T, int C, void* R, long r_rs, void* Y, long y_rs, float* stats) {
    if (!ctx) return KDEC_EINVAL;
    const DeviceScope device(ctx);
    Norm p;
    if (int rc = fill(ctx, "kdec_resnorm_fwd", dtype, layer, X, x_rs, Z, z_rs, gate, gate_rs, post, w1, b1, pre, w2, b2, eps, scale, x_scale,
                      T, C, p))
        return rc;
    if (T == 0) return KDEC_OK;
    KDEC_CHECK(ctx, (R || !Z) && (Y || !pre), "kdec_resnorm_fwd: null output");
    KDEC_CHECK(ctx, T == 1 || ((!Z || r_rs >= C) && (!pre || y_rs >= C)), "kdec_resnorm_fwd: row stride of an output too small");
    KDEC_CHECK(ctx, reinterpret_cast<size_t>(stats) % 16 == 0, "kdec_resnorm_fwd: statistics must be aligned to 16 bytes");
    const int es = dtype == KDEC_F32 ? 4 : 2;
    p.vec = p.vec && (!Z || wide(R, r_rs, es)) && (!pre || wide(Y, y_rs, es));
    p.r = R;
    p.r_rs = r_rs;
    p.y = Y;
    p.y_rs = y_rs;
    p.stats = stats;
    ProfScope ps(ctx, "resnorm", 0.0, static_cast<double>(es) * T * C * (1 + (Z ? 2 : 0) + (pre ? 1 : 0) + (gate && gate_rs ? 1 : 0)));
    const Shape sh = shape(C);
    KDEC_CHECK(ctx, grid_holds(cdiv(T, sh.rows), sh.threads), "kdec_resnorm_fwd: too many rows");
    const auto run = [&](auto ty) {
        typedef decltype(ty) E;
        by_shape(sh, p.vec, [&](auto v, auto w, auto vec) {
            hipLaunchKernelGGL((resnorm_k<E, decltype(v)::value, decltype(w)::value, decltype(vec)::value>),
                               dim3(static_cast<unsigned>(cdiv(T, sh.rows))), dim3(sh.threads), 0, ctx->stream, p);
        });
    };
    if (dtype == KDEC_F32) run(0.0f);
    else run(bf16{});
    return launch_check(ctx, "kdec_resnorm_fwd");
}

int kdec_resnorm_bwd(kdec_ctx* ctx, int dtype, int layer, const void* X, long x_rs, const void* Z, long z_rs, const void* gate,
                     long gate_rs, int post, const void* w1, const void* b1, int pre, const void* w2, const void* b2, float eps,
                     float scale, float x_scale, int T, int C, const float* stats, const void* dR, long dr_rs, const void* dY, long dy_rs,
                     void* dX, void* dZ, void* dgate, float* dw1, float* db1, float* dw2, float* db2) {
    if (!ctx) return KDEC_EINVAL;
    const DeviceScope device(ctx);
    Back b{};
    if (int rc = fill(ctx, "kdec_resnorm_bwd", dtype, layer, X, x_rs, Z, z_rs, gate, gate_rs, post, w1, b1, pre, w2, b2, eps, scale, x_scale,
                      T, C, b.n))
        return rc;
    KDEC_CHECK(ctx, T == 0 || (stats && dX && (dZ || !Z) && (dY || !pre)), "kdec_resnorm_bwd: null tensor");
    KDEC_CHECK(ctx, !gate == !dgate, "kdec_resnorm_bwd: a gate and its gradient come together");
    KDEC_CHECK(ctx, (!(dw1 || db1) || post) && (!(dw2 || db2) || pre), "kdec_resnorm_bwd: the gradient of a norm that is not there");
    KDEC_CHECK(ctx, reinterpret_cast<size_t>(stats) % 16 == 0, "kdec_resnorm_bwd: statistics must be aligned to 16 bytes");
    const int es = dtype == KDEC_F32 ? 4 : 2;
    const bool by_row = gate && gate_rs != 0;
    b.n.stats = const_cast<float*>(stats);
    b.dr = Rows{dR, dr_rs};
    b.dy = Rows{dY, dy_rs};
    b.n.vec = b.n.vec && wide(dR, dr_rs, es) && wide(dY, dy_rs, es) && wide(dX, C, es) && wide(dZ, C, es) &&
              (!by_row || wide(dgate, C, es));
    b.dx = dX;
    b.dz = dZ;
    b.dgate = by_row ? dgate : nullptr;
    float* const given[5] = {dw1, db1, dw2, db2, by_row ? nullptr : static_cast<float*>(dgate)};
    Outs outs{};
    for (int k = 0; k < 5; ++k) {
        b.at[k] = given[k] ? b.sums : -1;
        if (given[k]) outs.p[b.sums++] = given[k];
    }
    ProfScope ps(ctx, "resnorm", 0.0, static_cast<double>(es) * T * C * (3 + (Z ? 2 : 0) + (pre ? 1 : 0) + (by_row ? 2 : 0)));
    const Shape sh = shape(C);
    // Two blocks a CU, one of more than four waves: their sums are so much more to
    // write and read (bf16, forward and backward, one block a CU, two, four: 8192 x
    // 2048 112 us, 98, 102; 16000 x 1024 98, 85; 4096 x 4096 94, 102; 2048 x 5120 91,
    // 101, 117).
    long blocks = (sh.threads > 256 ? 1L : 2L) * ctx->num_cus;
    if (blocks > cdiv(T, sh.rows)) blocks = cdiv(T, sh.rows);
    Workspace ws(ctx, static_cast<size_t>(blocks) * b.sums * C * sizeof(float));
    if (!ws.p) return KDEC_ENOMEM;
    b.part = ws.as<float>();
    const auto run = [&](auto ty) {
        typedef decltype(ty) E;
        by_shape(sh, b.n.vec, [&](auto v, auto w, auto vec) {
            hipLaunchKernelGGL((resnorm_bwd_k<E, decltype(v)::value, decltype(w)::value, decltype(vec)::value>),
                               dim3(static_cast<unsigned>(blocks)), dim3(sh.threads), 0, ctx->stream, b);
        });
    };
    if (T > 0) {
        if (dtype == KDEC_F32) run(0.0f);
        else run(bf16{});
    }
    if (b.sums)
        hipLaunchKernelGGL(resnorm_join_k, dim3(static_cast<unsigned>(cdiv(C, 64)), static_cast<unsigned>(b.sums)), dim3(64 * JW), 0,
                           ctx->stream, b.part, static_cast<int>(blocks), b.sums, C, outs);
    return launch_check(ctx, "kdec_resnorm_bwd");
}

}  // extern "C"
