// Attention of packed documents on gfx950, forward and backward.
//
// Every row sees one contiguous run of keys [lo, hi): its document's, cut at
// its own position or at the document's prefix where the mask is causal. So
// a mask is two comparisons per score, a tile of keys that all rows of a
// block see takes none, and a block walks the keys from its rows' least lo to
// their greatest hi.
//
// One pass over the keys with the running maximum m and sum l of the
// softmax, in log2 units: p = 2^(t - m), with l and the output scaled by
// 2^(m_old - m) when the maximum moves. The scores are formed transposed,
// S^T = K Q^T, so that a lane holds one row's scores (row statistics need one
// exchange between the two lane halves) and the registers of S^T are, as they
// stand, the operand of O^T = V^T P (kdec_frag.hpp); V^T is read from the
// row-major tile with the transposing LDS read.
//
// Entries: the rows of the heads that share a key head, entry e = row * G +
// head within the group, so keys and values are staged once for the group.
#include "kdec_frag.hpp"
#include "kdec_internal.hpp"

#include <climits>
#include <cmath>
#include <memory>
#include <type_traits>

namespace kdec {
namespace {

constexpr int AT = 256;        // threads of a block
constexpr int BM = 128;        // entries of a block, 32 per wave
constexpr int BN = 64;         // keys of a tile
constexpr int RN = 32;         // keys of a wave's tile in the few-rows kernel
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

struct Docs {
    const int *q_off, *k_off, *k_len, *prefix;
    int docs, causal, Tq, Tk;
};

struct Attn {
    const void *Q, *K, *V;
    long q_rs, q_hs, k_rs, k_hs, v_rs, v_hs;
    Docs m;
    const float* slopes;
    float scale, cap;
    int Hq, Hkv, G, D, E;  // G = Hq / Hkv, E = Tq * G entries per key head
    bool vec;              // the inputs take 16-byte loads
    void* O;
    long o_rs, o_hs;
    bool vec_o;
    float* lse;
    int splits;
    float *part_o, *part_ml;  // (splits, Hkv, E, D) and (splits, Hkv, E, 2)
};

struct Row {
    int lo, hi, pos;  // keys [lo, hi), the key row at the row's own position
};

// The document whose query rows hold i (the last whose offset is not past
// it), or -1.
__device__ inline int doc_of(const int* off, int docs, int i) {
    int a = 0, b = docs;
    while (a < b) {
        const int mid = (a + b) >> 1;
        if (off[mid] <= i) a = mid + 1;
        else b = mid;
    }
    return a - 1;
}

struct Doc {
    int q0, lq, k0, lk, prefix;
};
__device__ inline Doc doc_at(const Docs& m, int d) {
    Doc r;
    r.q0 = min(max(m.q_off[d], 0), m.Tq);
    r.lq = max(min(m.q_off[d + 1], m.Tq) - r.q0, 0);
    r.k0 = min(max(m.k_off[d], 0), m.Tk);
    const int slot = max(min(m.k_off[d + 1], m.Tk) - r.k0, 0);
    r.lk = m.k_len ? min(max(m.k_len[d], 0), slot) : slot;
    r.prefix = m.prefix ? min(max(m.prefix[d], 0), r.lk) : 0;
    return r;
}

__device__ inline Row row_at(const Docs& m, int i) {
    Row r{INT_MAX, INT_MIN, 0};
    const int d = doc_of(m.q_off, m.docs, i);
    if (d < 0 || i >= m.q_off[d + 1]) return r;
    const Doc c = doc_at(m, d);
    const int p = i - c.q0 + c.lk - c.lq;  // position of its last key
    const int n = m.causal ? min(max(max(p + 1, c.prefix), 0), c.lk) : c.lk;
    if (n <= 0) return r;
    r.lo = c.k0;
    r.hi = c.k0 + n;
    r.pos = c.k0 + p;
    return r;
}

__device__ inline float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// tanh for scores in float: 1 - 2 / (1 + e^2x) away from zero; near it, where
// that difference loses its digits, the odd series (next term 62/2835 x^9,
// below 2^-25 of x up to 0.15).
__device__ inline float tanh_(float x) {
    const float big = 1.0f - 2.0f * __builtin_amdgcn_rcpf(1.0f + exp2_(2.0f * LOG2E * x));
    const float q = x * x;
    const float small = x * (1.0f + q * (-1.0f / 3 + q * (2.0f / 15 + q * (-17.0f / 315))));
    return __builtin_fabsf(x) < 0.15f ? small : big;
}

// A score in the softmax's units from the raw product. Without cap and bias
// the units are the products' own and `unit` = scale * log2(e); with either,
// log2 and unit = 1. dt: the capped score's derivative by the scaled product.
struct ScoreRule {
    float scale, cap, inv_cap, unit, slope;
    template <bool MODS>
    __device__ inline float of(float s, int dist, float& dt) const {
        dt = 1.0f;
        if (!MODS) return s;
        float t = s * scale;
        if (cap > 0.0f) {
            const float th = tanh_(t * inv_cap);
            t = cap * th;
            dt = 1.0f - th * th;
        }
        return (t - slope * static_cast<float>(dist)) * LOG2E;
    }
};
template <bool MODS>
__device__ inline ScoreRule score_rule(const Attn& a, int head) {
    ScoreRule r;
    r.scale = a.scale;
    r.cap = a.cap;
    r.inv_cap = a.cap > 0.0f ? 1.0f / a.cap : 0.0f;
    r.unit = MODS ? 1.0f : a.scale * LOG2E;
    r.slope = MODS && a.slopes ? a.slopes[head] : 0.0f;
    return r;
}

// Running softmax state of one lane's column over a score accumulator's 16
// rows (keys j0 + acc_row): s becomes the probabilities, and the column's
// output scale is returned.
struct Soft {
    float m = -__builtin_inff(), l = 0.0f;
};

template <class T, int DP>
struct Tiles {
    static constexpr int LS = DP + 16 / static_cast<int>(sizeof(T));  // row stride: 16 bytes past the row
    static constexpr int CH = DP / 8;                                 // 8-element chunks of a row
};

// One thread's share of a tile of ROWS rows, held between the global loads
// and the stores to shared memory.
template <class T, int DP, int ROWS, int NT>
struct Stage {
    static constexpr int N = ROWS * (DP / 8) / NT;
    Frag<T> f[N];
};

// Rows j0 .. of a key-side tensor (base of the key head) into a stage; rows
// at or past `end` are zeros.
template <class T, int DP, int ROWS, int NT>
__device__ inline void load_keys(Stage<T, DP, ROWS, NT>& st, const T* base, long rs, int j0, int end, int D, bool vec,
                                 int tid) {
#pragma unroll
    for (int i = 0; i < st.N; ++i) {
        const int c = tid + i * NT, row = c / (DP / 8), d = 8 * (c % (DP / 8));
        const int j = j0 + row;
        st.f[i] = load8(base + static_cast<long>(j < end ? j : 0) * rs + d, j < end ? min(8, D - d) : 0, vec);
    }
}
template <class T, int DP, int ROWS, int NT>
__device__ inline void store_tile(const Stage<T, DP, ROWS, NT>& st, T* tile, int tid) {
    constexpr int LS = Tiles<T, DP>::LS;
#pragma unroll
    for (int i = 0; i < st.N; ++i) {
        const int c = tid + i * NT, row = c / (DP / 8), d = 8 * (c % (DP / 8));
        *reinterpret_cast<Frag<T>*>(tile + row * LS + d) = st.f[i];
    }
}
// Values that are not finite become zeros: a product with a probability that
// the mask made zero would be NaN. Marks their rows in bad (when given).
template <class T, int DP, int ROWS, int NT>
__device__ inline void clean(Stage<T, DP, ROWS, NT>& st, unsigned* bad, int tid) {
#pragma unroll
    for (int i = 0; i < st.N; ++i)
        if (any_nonfinite<T>(st.f[i])) {
            st.f[i] = finite_or_zero<T>(st.f[i]);
            const int row = (tid + i * NT) / (DP / 8);
            if (bad) atomicOr(&bad[row >> 5], 1u << (row & 31));
        }
}

// Whether [lo, hi) holds a marked key of the 64 at j0.
__device__ inline bool sees_bad(int lo, int hi, int j0, unsigned long long bad) {
    const int a = min(max(lo - j0, 0), 64), b = min(max(hi - j0, 0), 64);
    if (b <= a) return false;
    const unsigned long long upto = b == 64 ? ~0ull : (1ull << b) - 1;
    return (upto & ~((1ull << a) - 1) & bad) != 0;
}

// One step of the running softmax of a lane's column over N score blocks of
// 32 keys from j0. Scores become probabilities; acc is rescaled when the
// wave's maxima move.
template <bool MODS, int N, int ND>
__device__ inline void soft_step(const ScoreRule& rule, const Row& row, bool masked, int j0, int half,
                                 f32x16 (&s)[N], f32x16 (&acc)[ND], Soft& st) {
    float mx = -__builtin_inff();
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int j = j0 + 32 * n + acc_row(r, half);
            float dt, t = rule.of<MODS>(s[n][r], abs(row.pos - j), dt);
            if (masked) t = (j >= row.lo && j < row.hi) ? t : -__builtin_inff();
            s[n][r] = t;
            mx = fmaxf(mx, t);
        }
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float m = fmaxf(st.m, mx);
    const float m0 = (m == -__builtin_inff() ? 0.0f : m) * rule.unit;
    float sum = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float p = exp2_(__builtin_fmaf(s[n][r], rule.unit, -m0));
            s[n][r] = p;
            sum += p;
        }
    if (__any(m != st.m)) {
        const float f = exp2_(__builtin_fmaf(st.m, rule.unit, -m0));
        st.l *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] *= f;
        st.m = m;
    }
    st.l += sum;
}

// A column's output and lse, or its unfinished state where the keys are split.
template <class T, int DP, bool MODS>
__device__ inline void finish(const Attn& a, int kvh, int e, int row, int head, int split, const ScoreRule& rule,
                              int half, const f32x16 (&acc)[DP / 32], float m, float l) {
    if (a.splits > 1) {
        const long at = (static_cast<long>(split) * a.Hkv + kvh) * a.E + e;
        float* o = a.part_o + at * a.D;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * dt + 8 * g + 4 * half;
                store4(o + d, a.D - d, a.D % 4 == 0, acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2],
                       acc[dt][4 * g + 3]);
            }
        if (!half) {
            a.part_ml[2 * at] = m * rule.unit;
            a.part_ml[2 * at + 1] = l;
        }
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* o = static_cast<T*>(a.O) + row * a.o_rs + head * a.o_hs;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * dt + 8 * g + 4 * half;
            store4(o + d, a.D - d, a.vec_o, acc[dt][4 * g] * inv, acc[dt][4 * g + 1] * inv, acc[dt][4 * g + 2] * inv,
                   acc[dt][4 * g + 3] * inv);
        }
    if (!half)
        a.lse[static_cast<long>(head) * a.m.Tq + row] = l == 0.0f ? -__builtin_inff() : m * rule.unit * LN2 + logf(l);
}

// Forward: a block holds 128 entries of one key head (32 per wave) and walks
// the keys that its rows see in tiles of 64, staged in shared memory with the
// next tile's loads in flight.
template <class T, int DP, bool MODS>
__global__ __launch_bounds__(AT, sizeof(T) == 2 ? 2 : 1) void attn_fwd_k(Attn a) {
    constexpr int LS = Tiles<T, DP>::LS, NC = DP / 16, ND = DP / 32;
    __shared__ __align__(16) T sk[BN * LS];
    __shared__ __align__(16) T sv[BN * LS];
    __shared__ unsigned bad[2][2];
    __shared__ int red[4][4];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5;
    const int kvh = blockIdx.x % a.Hkv;
    int tile = blockIdx.x / a.Hkv;
    if (a.m.causal) tile = gridDim.x / a.Hkv - 1 - tile;  // the longest walks first
    const int e = tile * BM + wave * 32 + (lane & 31);
    const bool valid = e < a.E;
    const int row = valid ? e / a.G : 0, head = kvh * a.G + (valid ? e - row * a.G : 0);
    const Row me = valid ? row_at(a.m, row) : Row{INT_MAX, INT_MIN, 0};

    // the wave's and the block's keys, and those that every row sees
    int lo = me.lo, hi = me.hi, full_lo = valid ? me.lo : INT_MIN, full_hi = valid ? me.hi : INT_MAX;
    for (int o = 16; o; o >>= 1) {
        lo = min(lo, __shfl_xor(lo, o));
        hi = max(hi, __shfl_xor(hi, o));
        full_lo = max(full_lo, __shfl_xor(full_lo, o));
        full_hi = min(full_hi, __shfl_xor(full_hi, o));
    }
    if (lane == 0) {
        red[wave][0] = lo;
        red[wave][1] = hi;
        red[wave][2] = full_lo;
        red[wave][3] = full_hi;
    }
    if (tid < 4) bad[tid >> 1][tid & 1] = 0;
    const int wlo = __builtin_amdgcn_readfirstlane(lo), whi = __builtin_amdgcn_readfirstlane(hi);
    __syncthreads();
    int blo = min(min(red[0][0], red[1][0]), min(red[2][0], red[3][0]));
    int bhi = max(max(red[0][1], red[1][1]), max(red[2][1], red[3][1]));
    full_lo = __builtin_amdgcn_readfirstlane(max(max(red[0][2], red[1][2]), max(red[2][2], red[3][2])));
    full_hi = __builtin_amdgcn_readfirstlane(min(min(red[0][3], red[1][3]), min(red[2][3], red[3][3])));
    blo = __builtin_amdgcn_readfirstlane(blo);
    bhi = __builtin_amdgcn_readfirstlane(bhi);
    const int tiles = bhi > blo ? (bhi - blo + BN - 1) / BN : 0;
    const int split = blockIdx.y;
    const int t0 = static_cast<int>(static_cast<long>(tiles) * split / a.splits);
    const int t1 = static_cast<int>(static_cast<long>(tiles) * (split + 1) / a.splits);

    const ScoreRule rule = score_rule<MODS>(a, head);
    Frag<T> q[NC];
    const T* qp = static_cast<const T*>(a.Q) + row * a.q_rs + head * a.q_hs;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int d = 16 * c + 8 * half;
        q[c] = load8(qp + d, valid ? min(8, a.D - d) : 0, a.vec);
    }
    const T* kb = static_cast<const T*>(a.K) + kvh * a.k_hs;
    const T* vb = static_cast<const T*>(a.V) + kvh * a.v_hs;
    Stage<T, DP, BN, AT> ks, vs;
    if (t0 < t1) {
        load_keys(ks, kb, a.k_rs, blo + t0 * BN, bhi, a.D, a.vec, tid);
        load_keys(vs, vb, a.v_rs, blo + t0 * BN, bhi, a.D, a.vec, tid);
    }
    f32x16 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
    Soft st;
    bool poison = false;
    for (int t = t0; t < t1; ++t) {
        const int j0 = blo + t * BN;
        const bool masked = !(j0 >= full_lo && j0 + BN <= full_hi);
        if (masked) clean(vs, bad[t & 1], tid);
        store_tile(ks, sk, tid);
        store_tile(vs, sv, tid);
        __syncthreads();
        if (t + 1 < t1) {
            load_keys(ks, kb, a.k_rs, j0 + BN, bhi, a.D, a.vec, tid);
            load_keys(vs, vb, a.v_rs, j0 + BN, bhi, a.D, a.vec, tid);
        }
        if (tid < 2) bad[(t + 1) & 1][tid] = 0;
        if (wlo < j0 + BN && whi > j0) {
            f32x16 s[2];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                s[n] = f32x16{};
#pragma unroll
                for (int c = 0; c < NC; ++c) s[n] = mma32(lds_rows(sk, LS, 32 * n, c), q[c], s[n]);
            }
            soft_step<MODS>(rule, me, masked, j0, half, s, acc, st);
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const Frag<T> p = acc_frag<T>(s[n], c);
#pragma unroll
                    for (int d = 0; d < ND; ++d) acc[d] = mma32(lds_cols(sv, LS, 32 * n, 32 * d, c), p, acc[d]);
                }
            if (masked) {
                const unsigned long long b = bad[t & 1][0] | static_cast<unsigned long long>(bad[t & 1][1]) << 32;
                poison |= sees_bad(me.lo, me.hi, j0, b);
            }
        }
        __syncthreads();
    }
    if (!valid) return;
    float l = st.l + __shfl_xor(st.l, 32);
    if (poison) l = __builtin_nanf("");
    finish<T, DP, MODS>(a, kvh, e, row, head, split, rule, half, acc, st.m, l);
}

// Forward of few rows over long keys: a block holds the heads of one row that
// share a key head (up to 32) and its waves take the keys in turn, 32 at a
// time, each with a softmax state of its own; the four are joined at the end.
// Keys go from memory into the product's registers, values through the wave's
// own shared memory for their transpose, so no wave waits for another.
template <class T, int DP, bool MODS>
__global__ __launch_bounds__(AT, 1) void attn_rows_k(Attn a, int chunks) {
    constexpr int LS = Tiles<T, DP>::LS, NC = DP / 16, ND = DP / 32;
    constexpr int JE = 8;  // columns joined at a time
    __shared__ __align__(16) T sv[4][RN * LS];
    __shared__ float sml[4][2][32];
    __shared__ float so[4][JE][DP + 1];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5;
    int b = blockIdx.x;
    const int kvh = b % a.Hkv;
    b /= a.Hkv;
    const int chunk = b % chunks, row = b / chunks;
    const int nh = min(32, a.G - 32 * chunk);  // heads of this block
    const bool valid = (lane & 31) < nh;
    const int g = 32 * chunk + (valid ? (lane & 31) : 0), head = kvh * a.G + g, e = row * a.G + g;
    const Row me = row_at(a.m, row);
    const int keys = me.hi > me.lo ? me.hi - me.lo : 0;
    const int tiles = (keys + RN - 1) / RN, split = blockIdx.y;
    const int t0 = static_cast<int>(static_cast<long>(tiles) * split / a.splits);
    const int t1 = static_cast<int>(static_cast<long>(tiles) * (split + 1) / a.splits);

    const ScoreRule rule = score_rule<MODS>(a, head);
    Frag<T> q[NC], k[NC];
    const T* qp = static_cast<const T*>(a.Q) + row * a.q_rs + head * a.q_hs;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int d = 16 * c + 8 * half;
        q[c] = load8(qp + d, valid ? min(8, a.D - d) : 0, a.vec);
    }
    const T* kb = static_cast<const T*>(a.K) + kvh * a.k_hs;
    const T* vb = static_cast<const T*>(a.V) + kvh * a.v_hs;
    Stage<T, DP, RN, 64> vs;
    const auto load = [&](int t) {
        const int j0 = me.lo + t * RN, j = j0 + (lane & 31);
        const T* p = kb + static_cast<long>(j < me.hi ? j : me.lo) * a.k_rs;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = 16 * c + 8 * half;
            k[c] = load8(p + d, j < me.hi ? min(8, a.D - d) : 0, a.vec);
        }
        load_keys(vs, vb, a.v_rs, j0, me.hi, a.D, a.vec, lane);
    };
    f32x16 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
    Soft st;
    if (t0 + wave < t1) load(t0 + wave);
    for (int t = t0 + wave; t < t1; t += 4) {
        const int j0 = me.lo + t * RN;
        f32x16 s[1];
        s[0] = f32x16{};
#pragma unroll
        for (int c = 0; c < NC; ++c) s[0] = mma32(k[c], q[c], s[0]);
        store_tile(vs, sv[wave], lane);
        if (t + 4 < t1) load(t + 4);
        soft_step<MODS>(rule, me, j0 + RN > me.hi, j0, half, s, acc, st);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const Frag<T> p = acc_frag<T>(s[0], c);
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[d] = mma32(lds_cols(sv[wave], LS, 0, 32 * d, c), p, acc[d]);
        }
    }
    // join the waves: their states' common maximum, then the sums in order
    float l = st.l + __shfl_xor(st.l, 32);
    if (!half) {
        sml[wave][0][lane] = st.m;
        sml[wave][1][lane] = l;
    }
    __syncthreads();
    const int col = lane & 31;
    float m = fmaxf(fmaxf(sml[0][0][col], sml[1][0][col]), fmaxf(sml[2][0][col], sml[3][0][col]));
    const float m0 = (m == -__builtin_inff() ? 0.0f : m) * rule.unit;
    const float f = exp2_(__builtin_fmaf(st.m, rule.unit, -m0));
    l = 0.0f;
    for (int w = 0; w < 4; ++w) l += sml[w][1][col] * exp2_(__builtin_fmaf(sml[w][0][col], rule.unit, -m0));
    for (int j = 0; j < nh; j += JE) {
        if (col >= j && col < j + JE)
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) so[wave][col - j][32 * d + acc_row(r, half)] = acc[d][r] * f;
        __syncthreads();
        // every wave takes the columns that fall to it: sums in the waves' order
        if ((wave == ((j / JE) & 3)) && col >= j && col < j + JE)
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int c = 32 * d + acc_row(r, half);
                    acc[d][r] = ((so[0][col - j][c] + so[1][col - j][c]) + so[2][col - j][c]) + so[3][col - j][c];
                }
        __syncthreads();
    }
    if (valid && wave == ((col / JE) & 3))
        finish<T, DP, MODS>(a, kvh, e, row, head, split, rule, half, acc, m, l);
}

// Joins the splits of an entry: one wave per entry, lanes over the output.
template <class T>
__global__ __launch_bounds__(AT) void attn_join_k(Attn a) {
    const int lane = threadIdx.x & 63;
    const long w = static_cast<long>(blockIdx.x) * (AT / 64) + (threadIdx.x >> 6);
    const long n = static_cast<long>(a.Hkv) * a.E;
    if (w >= n) return;
    const int kvh = static_cast<int>(w / a.E), e = static_cast<int>(w - static_cast<long>(kvh) * a.E);
    const int row = e / a.G, head = kvh * a.G + e - row * a.G;
    float m = -__builtin_inff();
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_ml[2 * (s * n + w)]);
    const float m0 = m == -__builtin_inff() ? 0.0f : m;
    float l = 0.0f, o[2] = {0.0f, 0.0f};
    for (int s = 0; s < a.splits; ++s) {
        const float f = exp2_(a.part_ml[2 * (s * n + w)] - m0);
        l += f * a.part_ml[2 * (s * n + w) + 1];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int d = lane + 64 * i;
            if (d < a.D) o[i] += f * a.part_o[(s * n + w) * a.D + d];
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = static_cast<T*>(a.O) + row * a.o_rs + head * a.o_hs;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = lane + 64 * i;
        if (d < a.D) out[d] = static_cast<T>(o[i] * inv);
    }
    if (lane == 0)
        a.lse[static_cast<long>(head) * a.m.Tq + row] = l == 0.0f ? -__builtin_inff() : m * LN2 + logf(l);
}

// ─── backward ───

struct AttnBwd {
    Attn f;  // the forward's arguments (O and lse its outputs)
    const void* dO;
    long do_rs, do_hs;
    void *dQ, *dK, *dV;
    long dq_rs, dq_hs, dk_rs, dk_hs, dv_rs, dv_hs;
    bool vec_dq, vec_dk, vec_dv;
    Row* rows;      // (Tq)
    float2* stat;   // (Hq, Tq): lse in log2 units, delta = dO . O
};

// delta = dO . O and lse in log2 units of every row and head, and the rows'
// keys. A row without keys gets lse = +inf, so that its probabilities are
// zeros; one whose delta is not finite gets NaN, which then marks every
// gradient that the row reaches. 16 lanes per row and head.
template <class T>
__global__ __launch_bounds__(AT) void attn_stat_k(AttnBwd b) {
    const Attn& a = b.f;
    const int lane = threadIdx.x & 15;
    const long w = static_cast<long>(blockIdx.x) * (AT / 16) + (threadIdx.x >> 4);
    if (w >= static_cast<long>(a.m.Tq) * a.Hq) return;
    const int row = static_cast<int>(w / a.Hq), head = static_cast<int>(w - static_cast<long>(row) * a.Hq);
    const int d = 8 * lane, n = min(8, a.D - d);
    const Frag<T> o = load8(static_cast<const T*>(a.O) + row * a.o_rs + head * a.o_hs + d, n, a.vec);
    const Frag<T> g = load8(static_cast<const T*>(b.dO) + row * b.do_rs + head * b.do_hs + d, n, a.vec);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += static_cast<float>(o[i]) * static_cast<float>(g[i]);
    for (int x = 8; x; x >>= 1) s += __shfl_xor(s, x);
    if (lane) return;
    const float lse = a.lse[static_cast<long>(head) * a.m.Tq + row];
    float l2 = lse == -__builtin_inff() ? __builtin_inff() : lse * LOG2E;
    if (lse != -__builtin_inff() && !(__builtin_fabsf(s) < __builtin_inff())) l2 = __builtin_nanf("");
    b.stat[static_cast<long>(head) * a.m.Tq + row] = make_float2(l2, lse == -__builtin_inff() ? 0.0f : s);
    if (head == 0) b.rows[row] = row_at(a.m, row);
}

// The score gradient of one element, dS without the factor `scale`, from the
// raw product s and dp = dO . V; p is returned for dV.
template <bool MODS>
__device__ inline float dscore(const ScoreRule& rule, float s, float dp, float lse2, float delta, int dist,
                               bool seen, float& p) {
    float dt;
    const float t = rule.of<MODS>(s, dist, dt);
    p = seen ? exp2_(__builtin_fmaf(t, rule.unit, -lse2)) : 0.0f;
    return seen ? p * (dp - delta) * dt : 0.0f;
}

// dQ: the forward's walk over the keys, with dQ^T = K^T dS^T in place of the
// output.
template <class T, int DP, bool MODS>
__global__ __launch_bounds__(AT, 1) void attn_dq_k(AttnBwd b) {
    constexpr int LS = Tiles<T, DP>::LS, NC = DP / 16, ND = DP / 32;
    __shared__ __align__(16) T sk[BN * LS];
    __shared__ __align__(16) T sv[BN * LS];
    __shared__ int red[4][4];
    const Attn& a = b.f;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5;
    const int kvh = blockIdx.x % a.Hkv;
    int tile = blockIdx.x / a.Hkv;
    if (a.m.causal) tile = gridDim.x / a.Hkv - 1 - tile;
    const int e = tile * BM + wave * 32 + (lane & 31);
    const bool valid = e < a.E;
    const int row = valid ? e / a.G : 0, head = kvh * a.G + (valid ? e - row * a.G : 0);
    const Row me = valid ? b.rows[row] : Row{INT_MAX, INT_MIN, 0};
    int lo = me.lo, hi = me.hi, full_lo = valid ? me.lo : INT_MIN, full_hi = valid ? me.hi : INT_MAX;
    for (int o = 16; o; o >>= 1) {
        lo = min(lo, __shfl_xor(lo, o));
        hi = max(hi, __shfl_xor(hi, o));
        full_lo = max(full_lo, __shfl_xor(full_lo, o));
        full_hi = min(full_hi, __shfl_xor(full_hi, o));
    }
    if (lane == 0) {
        red[wave][0] = lo;
        red[wave][1] = hi;
        red[wave][2] = full_lo;
        red[wave][3] = full_hi;
    }
    const int wlo = __builtin_amdgcn_readfirstlane(lo), whi = __builtin_amdgcn_readfirstlane(hi);
    __syncthreads();
    int blo = min(min(red[0][0], red[1][0]), min(red[2][0], red[3][0]));
    int bhi = max(max(red[0][1], red[1][1]), max(red[2][1], red[3][1]));
    full_lo = __builtin_amdgcn_readfirstlane(max(max(red[0][2], red[1][2]), max(red[2][2], red[3][2])));
    full_hi = __builtin_amdgcn_readfirstlane(min(min(red[0][3], red[1][3]), min(red[2][3], red[3][3])));
    blo = __builtin_amdgcn_readfirstlane(blo);
    bhi = __builtin_amdgcn_readfirstlane(bhi);
    const int tiles = bhi > blo ? (bhi - blo + BN - 1) / BN : 0;

    const ScoreRule rule = score_rule<MODS>(a, head);
    const float2 stat = valid ? b.stat[static_cast<long>(head) * a.m.Tq + row] : make_float2(__builtin_inff(), 0.0f);
    Frag<T> q[NC], g[NC];
    const T* qp = static_cast<const T*>(a.Q) + row * a.q_rs + head * a.q_hs;
    const T* gp = static_cast<const T*>(b.dO) + row * b.do_rs + head * b.do_hs;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int d = 16 * c + 8 * half, n = valid ? min(8, a.D - d) : 0;
        q[c] = load8(qp + d, n, a.vec);
        g[c] = load8(gp + d, n, a.vec);
    }
    const T* kb = static_cast<const T*>(a.K) + kvh * a.k_hs;
    const T* vb = static_cast<const T*>(a.V) + kvh * a.v_hs;
    Stage<T, DP, BN, AT> ks, vs;
    if (tiles) {
        load_keys(ks, kb, a.k_rs, blo, bhi, a.D, a.vec, tid);
        load_keys(vs, vb, a.v_rs, blo, bhi, a.D, a.vec, tid);
    }
    f32x16 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
    for (int t = 0; t < tiles; ++t) {
        const int j0 = blo + t * BN;
        const bool masked = !(j0 >= full_lo && j0 + BN <= full_hi);
        if (masked) clean(ks, nullptr, tid);  // a zero of dS times such a key
        store_tile(ks, sk, tid);
        store_tile(vs, sv, tid);
        __syncthreads();
        if (t + 1 < tiles) {
            load_keys(ks, kb, a.k_rs, j0 + BN, bhi, a.D, a.vec, tid);
            load_keys(vs, vb, a.v_rs, j0 + BN, bhi, a.D, a.vec, tid);
        }
        if (wlo < j0 + BN && whi > j0) {
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    s = mma32(lds_rows(sk, LS, 32 * n, c), q[c], s);
                    dp = mma32(lds_rows(sv, LS, 32 * n, c), g[c], dp);
                }
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int j = j0 + 32 * n + acc_row(r, half);
                    const bool seen = !masked || (j >= me.lo && j < me.hi);
                    float p;
                    s[r] = dscore<MODS>(rule, s[r], dp[r], stat.x, stat.y, abs(me.pos - j), seen, p);
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const Frag<T> ds = acc_frag<T>(s, c);
#pragma unroll
                    for (int d = 0; d < ND; ++d) acc[d] = mma32(lds_cols(sk, LS, 32 * n, 32 * d, c), ds, acc[d]);
                }
            }
        }
        __syncthreads();
    }
    if (!valid) return;
    T* o = static_cast<T*>(b.dQ) + row * b.dq_rs + head * b.dq_hs;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) {
            const int d = 32 * dt + 8 * g4 + 4 * half;
            store4(o + d, a.D - d, b.vec_dq, acc[dt][4 * g4] * a.scale, acc[dt][4 * g4 + 1] * a.scale,
                   acc[dt][4 * g4 + 2] * a.scale, acc[dt][4 * g4 + 3] * a.scale);
        }
}

// dK and dV: a block holds 128 keys of one key head (32 per wave, keys and
// values in registers) and walks the entries that see them in tiles of 32,
// their queries and output gradients staged in shared memory. All heads of
// the group are entries of the same walk, so the sums over shared heads need
// no joining. Scores are S = Q K^T here, a lane holding one key's column.
template <class T, int DP, bool MODS>
__global__ __launch_bounds__(AT, 1) void attn_dkv_k(AttnBwd b) {
    constexpr int LS = Tiles<T, DP>::LS, NC = DP / 16, ND = DP / 32, BE = 32;
    __shared__ __align__(16) T sq[BE * LS];
    __shared__ __align__(16) T sg[BE * LS];
    __shared__ __align__(16) float slse[BE], sdelta[BE], sslope[BE];
    __shared__ __align__(16) int slo[BE], shi[BE], spos[BE];
    const Attn& a = b.f;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, half = lane >> 5;
    const int kvh = blockIdx.x % a.Hkv, j0 = (blockIdx.x / a.Hkv) * BM;
    const int key = j0 + wave * 32 + (lane & 31);
    const bool valid = key < a.m.Tk;

    // the entries [e0, e1) whose rows may see keys of the block, and those
    // [f0, f1) whose rows all see all of them
    int e0 = 0, e1 = 0, f0 = 0, f1 = 0;
    {
        const int d0 = max(doc_of(a.m.k_off, a.m.docs, j0), 0);
        const int d1 = doc_of(a.m.k_off, a.m.docs, min(j0 + BM, a.m.Tk) - 1);
        if (d1 >= 0) {
            const Doc c = doc_at(a.m, d0), z = doc_at(a.m, d1);
            const int skip = c.lk - c.lq;  // position of the first row's key
            int first = c.q0;
            if (a.m.causal && j0 - c.k0 >= c.prefix) first = min(max(c.q0 + (j0 - c.k0) - skip, c.q0), c.q0 + c.lq);
            e0 = first * a.G;
            e1 = (z.q0 + z.lq) * a.G;
            if (d0 == d1 && j0 >= c.k0 && j0 + BM <= c.k0 + c.lk) {
                int all = c.q0;
                if (a.m.causal && j0 + BM - c.k0 > c.prefix)
                    all = min(max(c.q0 + (j0 + BM - 1 - c.k0) - skip, c.q0), c.q0 + c.lq);
                f0 = all * a.G;
                f1 = (c.q0 + c.lq) * a.G;
            }
        }
        e0 = __builtin_amdgcn_readfirstlane(e0);
        e1 = __builtin_amdgcn_readfirstlane(e1);
        f0 = __builtin_amdgcn_readfirstlane(f0);
        f1 = __builtin_amdgcn_readfirstlane(f1);
    }

    Frag<T> k[NC], v[NC];
    const T* kp = static_cast<const T*>(a.K) + kvh * a.k_hs + static_cast<long>(valid ? key : 0) * a.k_rs;
    const T* vp = static_cast<const T*>(a.V) + kvh * a.v_hs + static_cast<long>(valid ? key : 0) * a.v_rs;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int d = 16 * c + 8 * half, n = valid ? min(8, a.D - d) : 0;
        k[c] = load8(kp + d, n, a.vec);
        v[c] = load8(vp + d, n, a.vec);
    }
    const T* qb = static_cast<const T*>(a.Q) + static_cast<long>(kvh) * a.G * a.q_hs;
    const T* gb = static_cast<const T*>(b.dO) + static_cast<long>(kvh) * a.G * b.do_hs;
    Stage<T, DP, BE, AT> qs, gs;
    float2 r_stat;
    Row r_row;
    float r_slope = 0.0f;
    const auto load = [&](int base) {
#pragma unroll
        for (int i = 0; i < qs.N; ++i) {
            const int c = tid + i * AT, e = base + c / (DP / 8), d = 8 * (c % (DP / 8));
            const int n = e < e1 ? min(8, a.D - d) : 0;
            const int row = e < e1 ? e / a.G : 0, h = e < e1 ? e - row * a.G : 0;
            qs.f[i] = load8(qb + row * a.q_rs + h * a.q_hs + d, n, a.vec);
            gs.f[i] = load8(gb + row * b.do_rs + h * b.do_hs + d, n, a.vec);
        }
        if (tid < BE) {
            const int e = base + tid;
            r_stat = make_float2(__builtin_inff(), 0.0f);
            r_row = Row{INT_MAX, INT_MIN, 0};
            if (e < e1) {
                const int row = e / a.G, h = kvh * a.G + e - row * a.G;
                r_stat = b.stat[static_cast<long>(h) * a.m.Tq + row];
                r_row = b.rows[row];
                if (MODS && a.slopes) r_slope = a.slopes[h];
            }
        }
    };
    f32x16 dk[ND], dv[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) dk[d] = dv[d] = f32x16{};
    ScoreRule rule = score_rule<MODS>(a, kvh * a.G);
    if (e0 < e1) load(e0);
    for (int base = e0; base < e1; base += BE) {
        const bool masked = !(base >= f0 && base + BE <= f1);
        if (masked) {
            clean(qs, nullptr, tid);
            clean(gs, nullptr, tid);
        }
        store_tile(qs, sq, tid);
        store_tile(gs, sg, tid);
        if (tid < BE) {
            slse[tid] = r_stat.x;
            sdelta[tid] = r_stat.y;
            slo[tid] = r_row.lo;
            shi[tid] = r_row.hi;
            spos[tid] = r_row.pos;
            sslope[tid] = r_slope;
        }
        __syncthreads();
        if (base + BE < e1) load(base + BE);
        f32x16 s = f32x16{}, dp = f32x16{}, p;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            s = mma32(lds_rows(sq, LS, 0, c), k[c], s);
            dp = mma32(lds_rows(sg, LS, 0, c), v[c], dp);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const int i = acc_row(r, half);
            bool seen = true;
            if (masked) seen = key >= slo[i] && key < shi[i];
            if (MODS) rule.slope = sslope[i];
            float pr;
            s[r] = dscore<MODS>(rule, s[r], dp[r], slse[i], sdelta[i], MODS ? abs(spos[i] - key) : 0, seen, pr);
            p[r] = pr;
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const Frag<T> pf = acc_frag<T>(p, c), ds = acc_frag<T>(s, c);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                dv[d] = mma32(lds_cols(sg, LS, 0, 32 * d, c), pf, dv[d]);
                dk[d] = mma32(lds_cols(sq, LS, 0, 32 * d, c), ds, dk[d]);
            }
        }
        __syncthreads();
    }
    if (!valid) return;
    T* ok = static_cast<T*>(b.dK) + kvh * b.dk_hs + key * b.dk_rs;
    T* ov = static_cast<T*>(b.dV) + kvh * b.dv_hs + key * b.dv_rs;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * dt + 8 * g + 4 * half;
            store4(ok + d, a.D - d, b.vec_dk, dk[dt][4 * g] * a.scale, dk[dt][4 * g + 1] * a.scale,
                   dk[dt][4 * g + 2] * a.scale, dk[dt][4 * g + 3] * a.scale);
            store4(ov + d, a.D - d, b.vec_dv, dv[dt][4 * g], dv[dt][4 * g + 1], dv[dt][4 * g + 2], dv[dt][4 * g + 3]);
        }
}

// ─── host ───

// Whether a tensor's rows and heads start on multiples of `to` bytes.
bool aligned(const void* p, long rs, long hs, size_t size, size_t to = 16) {
    return reinterpret_cast<size_t>(p) % to == 0 && (rs * size) % to == 0 && (hs * size) % to == 0;
}

template <class F>
int dispatch(int dtype, int D, bool mods, F f) {
    if (dtype == KDEC_F32) {
        if (D <= 64) return mods ? f(float{}, std::integral_constant<int, 64>{}, std::true_type{})
                                 : f(float{}, std::integral_constant<int, 64>{}, std::false_type{});
        return mods ? f(float{}, std::integral_constant<int, 128>{}, std::true_type{})
                    : f(float{}, std::integral_constant<int, 128>{}, std::false_type{});
    }
    if (D <= 64) return mods ? f(bf16{}, std::integral_constant<int, 64>{}, std::true_type{})
                             : f(bf16{}, std::integral_constant<int, 64>{}, std::false_type{});
    return mods ? f(bf16{}, std::integral_constant<int, 128>{}, std::true_type{})
                : f(bf16{}, std::integral_constant<int, 128>{}, std::false_type{});
}

int check(kdec_ctx* ctx, const char* who, int dtype, const void* q_off, const void* k_off, int docs, float scale,
          float cap, int Tq, int Tk, int Hq, int Hkv, int D) {
    const auto bad = [&](const char* why) { return fail(ctx, KDEC_EINVAL, std::string(who) + ": " + why); };
    if (dtype != KDEC_F32 && dtype != KDEC_BF16) return bad("unknown type");
    if (Tq < 0 || Tk < 0 || docs < 0) return bad("negative size");
    if (Hq <= 0 || Hkv <= 0 || Hq % Hkv) return bad("query heads are not a multiple of the key heads");
    if (D <= 0 || D > 128) return bad("head width outside 1..128");
    if (static_cast<long>(Tq) * Hq >= INT_MAX - BM || static_cast<long>(Tk) >= INT_MAX - BM) return bad("too many rows");
    if (!(scale > 0.0f) || !(scale < HUGE_VALF)) return bad("scale must be positive");
    if (!(cap >= 0.0f) || !(cap < HUGE_VALF)) return bad("cap must be at least 0");
    if (docs > 0 && (!q_off || !k_off)) return bad("null offsets");
    return KDEC_OK;
}

}  // namespace
}  // namespace kdec

using namespace kdec;

extern "C" {

int kdec_attn_fwd(kdec_ctx* ctx, int dtype, const void* Q, long q_rs, long q_hs, const void* K, long k_rs, long k_hs,
                  const void* V, long v_rs, long v_hs, const int* q_off, const int* k_off, const int* k_len,
                  const int* prefix, int docs, int causal, const float* slopes, float scale, float cap, int Tq, int Tk,
                  int Hq, int Hkv, int D, void* O, long o_rs, long o_hs, float* lse) {
    if (!ctx) return KDEC_EINVAL;
    if (int rc = check(ctx, "kdec_attn_fwd", dtype, q_off, k_off, docs, scale, cap, Tq, Tk, Hq, Hkv, D)) return rc;
    if (Tq == 0) return KDEC_OK;
    KDEC_CHECK(ctx, Q && O && lse && (Tk == 0 || (K && V)), "kdec_attn_fwd: null tensor");
    const size_t size = dtype == KDEC_F32 ? 4 : 2;
    const int G = Hq / Hkv;
    Attn a{Q, K, V, q_rs, q_hs, k_rs, k_hs, v_rs, v_hs, {q_off, k_off, k_len, prefix, docs, causal != 0, Tq, Tk},
           slopes, scale, cap, Hq, Hkv, G, D, Tq * G,
           D % 8 == 0 && aligned(Q, q_rs, q_hs, size) && aligned(K, k_rs, k_hs, size) && aligned(V, v_rs, v_hs, size),
           O, o_rs, o_hs, D % 4 == 0 && aligned(O, o_rs, o_hs, size, 4 * size), lse, 1, nullptr, nullptr};
    // Few rows per document over many keys: a block per row. Rows of
    // different documents in one block would walk each other's keys.
    const bool rows = static_cast<long>(Tq) <= 8L * docs && static_cast<long>(Tk) >= 8L * Tq;
    const int chunks = static_cast<int>(cdiv(G, 32));
    const long tiles = rows ? static_cast<long>(Tq) * chunks : cdiv(a.E, BM);
    const long blocks = tiles * Hkv;
    KDEC_CHECK(ctx, blocks < INT_MAX, "kdec_attn_fwd: too many rows");
    // Split the keys where the rows alone do not fill the device, to no fewer
    // than 256 keys a part.
    const long each = docs > 0 ? Tk / docs : 0;
    long splits = cdiv(2L * ctx->num_cus, blocks);
    if (splits > each / 256) splits = each / 256;
    if (splits < 1) splits = 1;
    a.splits = static_cast<int>(splits);
    ProfScope ps(ctx, "attn", 0.0, 0.0);
    const size_t n = static_cast<size_t>(splits) * Hkv * a.E;
    std::unique_ptr<Workspace> ws;
    if (splits > 1) {
        ws = std::make_unique<Workspace>(ctx, n * (D + 2) * sizeof(float));
        if (!ws->p) return KDEC_ENOMEM;
        a.part_o = ws->as<float>();
        a.part_ml = a.part_o + n * D;
    }
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(splits));
    return dispatch(dtype, D, cap > 0.0f || slopes, [&](auto t, auto dp, auto mods) {
        typedef decltype(t) T;
        if (rows)
            hipLaunchKernelGGL((attn_rows_k<T, dp.value, mods.value>), grid, dim3(AT), 0, ctx->stream, a, chunks);
        else
            hipLaunchKernelGGL((attn_fwd_k<T, dp.value, mods.value>), grid, dim3(AT), 0, ctx->stream, a);
        if (a.splits > 1)
            hipLaunchKernelGGL(attn_join_k<T>, dim3(static_cast<unsigned>(cdiv(static_cast<long>(Hkv) * a.E, AT / 64))),
                               dim3(AT), 0, ctx->stream, a);
        return launch_check(ctx, "kdec_attn_fwd");
    });
}

int kdec_attn_bwd(kdec_ctx* ctx, int dtype, const void* Q, long q_rs, long q_hs, const void* K, long k_rs, long k_hs,
                  const void* V, long v_rs, long v_hs, const void* O, long o_rs, long o_hs, const float* lse,
                  const void* dO, long do_rs, long do_hs, const int* q_off, const int* k_off, const int* k_len,
                  const int* prefix, int docs, int causal, const float* slopes, float scale, float cap, int Tq, int Tk,
                  int Hq, int Hkv, int D, void* dQ, long dq_rs, long dq_hs, void* dK, long dk_rs, long dk_hs, void* dV,
                  long dv_rs, long dv_hs) {
    if (!ctx) return KDEC_EINVAL;
    if (int rc = check(ctx, "kdec_attn_bwd", dtype, q_off, k_off, docs, scale, cap, Tq, Tk, Hq, Hkv, D)) return rc;
    KDEC_CHECK(ctx, (Tq == 0 || (Q && O && lse && dO && dQ)) && (Tk == 0 || (K && V && dK && dV)),
               "kdec_attn_bwd: null tensor");
    if (Tq == 0 && Tk == 0) return KDEC_OK;
    const size_t size = dtype == KDEC_F32 ? 4 : 2;
    const int G = Hq / Hkv;
    AttnBwd b{};
    b.f = Attn{Q, K, V, q_rs, q_hs, k_rs, k_hs, v_rs, v_hs, {q_off, k_off, k_len, prefix, docs, causal != 0, Tq, Tk},
               slopes, scale, cap, Hq, Hkv, G, D, Tq * G,
               D % 8 == 0 && aligned(Q, q_rs, q_hs, size) && aligned(K, k_rs, k_hs, size) &&
                   aligned(V, v_rs, v_hs, size) && aligned(O, o_rs, o_hs, size) && aligned(dO, do_rs, do_hs, size),
               const_cast<void*>(O), o_rs, o_hs, false, const_cast<float*>(lse), 1, nullptr, nullptr};
    b.dO = dO;
    b.do_rs = do_rs;
    b.do_hs = do_hs;
    b.dQ = dQ;
    b.dK = dK;
    b.dV = dV;
    b.dq_rs = dq_rs;
    b.dq_hs = dq_hs;
    b.dk_rs = dk_rs;
    b.dk_hs = dk_hs;
    b.dv_rs = dv_rs;
    b.dv_hs = dv_hs;
    b.vec_dq = D % 4 == 0 && aligned(dQ, dq_rs, dq_hs, size, 4 * size);
    b.vec_dk = D % 4 == 0 && aligned(dK, dk_rs, dk_hs, size, 4 * size);
    b.vec_dv = D % 4 == 0 && aligned(dV, dv_rs, dv_hs, size, 4 * size);
    ProfScope ps(ctx, "attn", 0.0, 0.0);
    const size_t stat_bytes = static_cast<size_t>(Tq) * Hq * sizeof(float2);
    Workspace ws(ctx, stat_bytes + static_cast<size_t>(Tq) * sizeof(Row));
    if (!ws.p) return KDEC_ENOMEM;
    b.stat = ws.as<float2>();
    b.rows = reinterpret_cast<Row*>(ws.as<char>() + stat_bytes);
    const long q_blocks = cdiv(b.f.E, BM) * Hkv, k_blocks = cdiv(Tk, BM) * Hkv;
    KDEC_CHECK(ctx, k_blocks < INT_MAX, "kdec_attn_bwd: too many keys");
    return dispatch(dtype, D, cap > 0.0f || slopes, [&](auto t, auto dp, auto mods) {
        typedef decltype(t) T;
        if (Tq > 0) {
            hipLaunchKernelGGL(attn_stat_k<T>, dim3(static_cast<unsigned>(cdiv(static_cast<long>(Tq) * Hq, AT / 16))),
                               dim3(AT), 0, ctx->stream, b);
            hipLaunchKernelGGL((attn_dq_k<T, dp.value, mods.value>), dim3(static_cast<unsigned>(q_blocks)), dim3(AT), 0,
                               ctx->stream, b);
        }
        if (Tk > 0)
            hipLaunchKernelGGL((attn_dkv_k<T, dp.value, mods.value>), dim3(static_cast<unsigned>(k_blocks)), dim3(AT),
                               0, ctx->stream, b);
        return launch_check(ctx, "kdec_attn_bwd");
    });
}

}  // extern "C"
