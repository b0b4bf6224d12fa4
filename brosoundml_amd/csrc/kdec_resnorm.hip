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
#include "kdec_frag.hpp"
#include "kdec_internal.hpp"

#include <climits>

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

// W waves hold a row, R rows are in a block.
template <int W>
struct Block {
    static constexpr int R = W >= 4 ? 1 : 4 / W, NT = 64 * W * R;
};

__device__ inline float wave_sum(float x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// Two sums over a row's lanes, the same in all of them. Waves of a row meet in
// shared memory, in two buffers in turn so that one barrier a sum is enough.
template <int W>
__device__ inline void row_sums(float& a, float& b, float (*red)[2][2 * W], int& turn) {
    a = wave_sum(a);
    b = wave_sum(b);
    if (W == 1) return;
    const int wave = threadIdx.x >> 6, slot = wave / W, w = wave % W;
    float* at = red[slot][turn];
    if ((threadIdx.x & 63) == 0) {
        at[2 * w] = a;
        at[2 * w + 1] = b;
    }
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        a += at[2 * i];
        b += at[2 * i + 1];
    }
    turn ^= 1;
}

template <class T>
__device__ inline f32x8 floats8(const T* p, int n, bool vec) {
    const Frag<T> f = load8(p, n, vec);
    f32x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = static_cast<float>(f[i]);
    return r;
}
template <class T>
__device__ inline f32x8 vector8(const void* p, int c, int n, bool vec, float none) {
    if (p) return floats8(static_cast<const T*>(p) + c, n, vec);
    f32x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = none;
    return r;
}
template <class T>
__device__ inline void store8(T* p, int n, bool vec, const f32x8& v) {
    Frag<T> f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<T>(v[i]);
    if (vec) {
        if (n > 0) *reinterpret_cast<Frag<T>*>(p) = f;
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = f[i];
}

// A row's mean (0 for the RMS norm) and 1 / sqrt(mean square around it + eps).
template <int V, int W>
__device__ inline void moments(const Norm& p, const f32x8 (&u)[V], const int (&n)[V], float (*red)[2][2 * W], int& turn, float& mean,
                               float& rstd) {
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

template <class T, int V, int W>
__global__ __launch_bounds__(Block<W>::NT) void resnorm_k(Norm p) {
    constexpr int R = Block<W>::R;
    __shared__ float red[R][2][2 * W];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const long row = static_cast<long>(blockIdx.x) * R + wave / W;
    const bool live = row < p.T;
    const long at = live ? row : p.T - 1;
    int c[V], n[V], turn = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        c[v] = 512 * (v * W + wave % W) + 8 * lane;
        n[v] = max(min(8, p.C - c[v]), 0);
    }
    f32x8 x[V], u[V];
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = floats8(static_cast<const T*>(p.x.p) + at * p.x.rs + c[v], n[v], p.vec);
    float m1 = 0.0f, s1 = 0.0f, m2 = 0.0f, s2 = 0.0f;
    if (p.z.p) {
#pragma unroll
        for (int v = 0; v < V; ++v) u[v] = floats8(static_cast<const T*>(p.z.p) + at * p.z.rs + c[v], n[v], p.vec);
        if (p.post) {
            moments<V, W>(p, u, n, red, turn, m1, s1);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const f32x8 w = vector8<T>(p.w1, c[v], n[v], p.vec, 1.0f), b = vector8<T>(p.b1, c[v], n[v], p.vec, 0.0f);
#pragma unroll
                for (int i = 0; i < 8; ++i) u[v][i] = __builtin_fmaf((u[v][i] - m1) * s1, w[i], b[i]);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const f32x8 g = p.gate.p ? vector8<T>(static_cast<const T*>(p.gate.p) + at * p.gate.rs, c[v], n[v], p.vec, 1.0f)
                                     : vector8<T>(nullptr, 0, 0, false, 1.0f);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[v][i] = i < n[v] ? __builtin_fmaf(p.scale * g[i], u[v][i], p.x_scale * x[v][i]) : 0.0f;
            if (live) store8(static_cast<T*>(p.r) + at * p.r_rs + c[v], n[v], p.vec, x[v]);
        }
    }
    if (p.pre) {
        moments<V, W>(p, x, n, red, turn, m2, s2);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const f32x8 w = vector8<T>(p.w2, c[v], n[v], p.vec, 1.0f), b = vector8<T>(p.b2, c[v], n[v], p.vec, 0.0f);
            f32x8 y;
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = __builtin_fmaf((x[v][i] - m2) * s2, w[i], b[i]);
            if (live) store8(static_cast<T*>(p.y) + at * p.y_rs + c[v], n[v], p.vec, y);
        }
    }
    if (p.stats && live && lane == 0 && wave % W == 0) *reinterpret_cast<f32x4*>(p.stats + 4 * at) = f32x4{m1, s1, m2, s2};
}

struct Back {
    Norm n;
    Rows dr, dy;
    void *dx, *dz, *dgate;  // dgate: (T, C) of the tensors' type
    float* part;            // (blocks, SUMS, C), the sums in use first
    int sums, at[5];        // where dw1, db1, dw2, db2 and the columns' dgate are among them, -1: not in use
};

template <class T, int V, int W>
__global__ __launch_bounds__(Block<W>::NT) void resnorm_bwd_k(Back b) {
    constexpr int R = Block<W>::R;
    __shared__ float red[R][2][2 * W];
    __shared__ float join[R > 1 ? R - 1 : 1][R > 1 ? 64 * W * 8 : 1];
    const Norm& p = b.n;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    int c[V], n[V], turn = 0;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        c[v] = 512 * (v * W + wave % W) + 8 * lane;
        n[v] = max(min(8, p.C - c[v]), 0);
    }
    f32x8 sum[5][V];
#pragma unroll
    for (int k = 0; k < 5; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) sum[k][v] = f32x8{};
    const float over = 1.0f / static_cast<float>(p.C);
    for (long row0 = static_cast<long>(blockIdx.x) * R; row0 < p.T; row0 += static_cast<long>(gridDim.x) * R) {
        const long row = row0 + wave / W;
        const bool live = row < p.T;
        const long at = live ? row : p.T - 1;
        const auto load = [&](const Rows& t, int v) __attribute__((always_inline)) {
            return floats8(static_cast<const T*>(t.p) + at * t.rs + c[v], live ? n[v] : 0, p.vec);
        };
        f32x8 rh[V], zh[V], d[V], dy[V];
        const f32x4 st = *reinterpret_cast<const f32x4*>(p.stats + 4 * at);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            rh[v] = load(p.x, v);
            zh[v] = p.z.p ? load(p.z, v) : f32x8{};
            d[v] = b.dr.p ? load(b.dr, v) : f32x8{};
            dy[v] = p.pre ? load(b.dy, v) : f32x8{};
        }
        const auto gate = [&](int v) __attribute__((always_inline)) {
            f32x8 g = p.gate.p ? load(p.gate, v) : vector8<T>(nullptr, 0, 0, false, 1.0f);
#pragma unroll
            for (int i = 0; i < 8; ++i) g[i] *= p.scale;
            return g;
        };
        // the normalised rows
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (p.z.p) {
                const f32x8 w = p.post ? vector8<T>(p.w1, c[v], n[v], p.vec, 1.0f) : f32x8{};
                const f32x8 bias = p.post ? vector8<T>(p.b1, c[v], n[v], p.vec, 0.0f) : f32x8{};
                const f32x8 g = gate(v);
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
        }
        if (p.pre) {
            float e1 = 0.0f, e2 = 0.0f;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const f32x8 w = vector8<T>(p.w2, c[v], n[v], p.vec, 1.0f);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (i < n[v] && live) {
                        sum[2][v][i] = __builtin_fmaf(dy[v][i], rh[v][i], sum[2][v][i]);
                        sum[3][v][i] += dy[v][i];
                    }
                    dy[v][i] = i < n[v] ? dy[v][i] * w[i] : 0.0f;
                    e1 += dy[v][i];
                    e2 = i < n[v] ? __builtin_fmaf(dy[v][i], rh[v][i], e2) : e2;
                }
            }
            row_sums<W>(e1, e2, red, turn);
            e1 = p.layer ? e1 * over : 0.0f;
            e2 *= over;
#pragma unroll
            for (int v = 0; v < V; ++v)
#pragma unroll
                for (int i = 0; i < 8; ++i) d[v][i] += st[3] * (dy[v][i] - e1 - rh[v][i] * e2);
        }
        if (live)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                f32x8 o;
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = p.x_scale * d[v][i];
                store8(static_cast<T*>(b.dx) + at * p.C + c[v], n[v], p.vec, o);
            }
        if (!p.z.p) continue;
        float f1 = 0.0f, f2 = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const f32x8 w = p.post ? vector8<T>(p.w1, c[v], n[v], p.vec, 1.0f) : f32x8{};
            if (p.gate.p) {  // scale u d
                const f32x8 bias = p.post ? vector8<T>(p.b1, c[v], n[v], p.vec, 0.0f) : f32x8{};
                f32x8 o;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    o[i] = p.scale * (p.post ? __builtin_fmaf(zh[v][i], w[i], bias[i]) : zh[v][i]) * d[v][i];
                if (b.dgate) {
                    if (live) store8(static_cast<T*>(b.dgate) + at * p.C + c[v], n[v], p.vec, o);
                } else if (live) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) sum[4][v][i] += i < n[v] ? o[i] : 0.0f;
                }
            }
            const f32x8 g = gate(v);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                d[v][i] = i < n[v] ? d[v][i] * g[i] : 0.0f;  // du
                if (p.post) {
                    if (i < n[v] && live) {
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
            for (int v = 0; v < V; ++v) store8(static_cast<T*>(b.dz) + at * p.C + c[v], n[v], p.vec, d[v]);
    }
    // the block's rows together, then its share of every sum
#pragma unroll
    for (int k = 0; k < 5; ++k) {
        if (b.at[k] < 0) continue;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            if (R > 1) {
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

// Waves and columns a lane of a row: as few waves as hold it in a register
// block of 8 V columns a lane.
template <class T, class F>
int by_width(int C, F f) {
    if (C <= 512) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{});
    if (C <= 1024) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 2>{});
    if (C <= 2048) return f(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
    if (C <= 4096) return f(std::integral_constant<int, 2>{}, std::integral_constant<int, 4>{});
    return f(std::integral_constant<int, 2>{}, std::integral_constant<int, 8>{});
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
    const auto run = [&](auto ty) {
        typedef decltype(ty) E;
        return by_width<E>(C, [&](auto v, auto w) {
            constexpr int V = decltype(v)::value, W = decltype(w)::value;
            hipLaunchKernelGGL((resnorm_k<E, V, W>), dim3(static_cast<unsigned>(cdiv(T, Block<W>::R))), dim3(Block<W>::NT), 0, ctx->stream,
                               p);
            return KDEC_OK;
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
    const auto run = [&](auto ty) {
        typedef decltype(ty) E;
        return by_width<E>(C, [&](auto v, auto w) {
            constexpr int V = decltype(v)::value, W = decltype(w)::value, R = Block<W>::R;
            long blocks = cdiv(T, R);
            if (blocks > 2L * ctx->num_cus) blocks = 2L * ctx->num_cus;
            Workspace ws(ctx, static_cast<size_t>(blocks) * b.sums * C * sizeof(float));
            if (!ws.p) return KDEC_ENOMEM;
            b.part = ws.as<float>();
            if (T > 0)
                hipLaunchKernelGGL((resnorm_bwd_k<E, V, W>), dim3(static_cast<unsigned>(blocks)), dim3(Block<W>::NT), 0, ctx->stream, b);
            if (b.sums)
                hipLaunchKernelGGL(resnorm_join_k, dim3(static_cast<unsigned>(cdiv(C, 64)), static_cast<unsigned>(b.sums)), dim3(64 * JW), 0,
                                   ctx->stream, b.part, static_cast<int>(blocks), b.sums, C, outs);
            return KDEC_OK;
        });
    };
    if (int rc = dtype == KDEC_F32 ? run(0.0f) : run(bf16{})) return rc;
    return launch_check(ctx, "kdec_resnorm_bwd");
}

}  // extern "C"
