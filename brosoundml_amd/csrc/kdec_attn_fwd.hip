// Attention of packed documents on gfx950, forward.
//
// Every row sees one contiguous run of keys [lo, hi): its document's, cut at
// its own position or at the document's prefix where the mask is causal. So
// a mask is two comparisons per score, a tile of keys that all rows of a
// block see takes none, and a block walks the keys from its rows' least lo to
// their greatest hi.
//
// One pass over the keys with the running maximum m and sum l of the
// softmax, in log2 units: p = 2^(t - m), with l and the output scaled by
// 2^(m_old - m) when the maximum moves by more than 8 (until then p is at
// most 2^8, which neither type minds). The scores are formed transposed,
// S^T = K Q^T, so that a lane holds one row's scores (row statistics need one
// exchange between the two lane halves) and the registers of S^T are, as they
// stand, the operand of O^T = V^T P (kdec_frag.hpp); V^T is read from the
// row-major tile with the transposing LDS read. Probabilities are rounded to
// the tensors' type for that product; their sum l takes them unrounded.
//
// Entries: the rows of the heads that share a key head, entry e = row * G +
// head within the group, so keys and values are staged once for the group.
//
// Long walks are bound by the matrix units and the exponentials between their
// products: 8192 causal rows, 16 heads on 4 of width 128, bf16, take 304 us
// (905 TFLOP/s of what the mask leaves; a large library product reaches 1320),
// 4 causal texts of 1900 to 4099 rows with a prefix and capped scores 318 (485
// TFLOP/s: the cap's exponential and reciprocal come on top). Packed texts of
// 20 to 510 tokens, 12 heads of width 64, take 31 us: their walks are a few
// tiles long, so that the way to the first tile and the longest documents count.
#include "kdec_attn.hpp"

namespace kdec {
namespace attn {
namespace {

constexpr int RN = 32;  // keys of a wave's tile in the few-rows kernel

struct Fwd {
    Args a;
    void* O;
    long o_rs, o_hs;
    bool vec_o;
    float* lse;
    int D_out;  // O's width (a.D may be padded)
    int splits;
    float *part_o, *part_ml;  // (splits, Hkv, E, D) and (splits, Hkv, E, 2)
};

// Running softmax state of one lane's column, in the units of m: raw products
// (times `unit` they are log2) without cap and bias, log2 with either.
struct Soft {
    float m = -INF, l = 0.0f;
};

// One step of the running softmax of a lane's column over N score blocks of
// 32 keys from j0 (whole: all of the wave's rows see all of them). Scores
// become probabilities; acc is rescaled when the column's maximum moves far enough.
template <bool MASKED, class T, int CAP, bool BIAS, int N, int ND>
__device__ inline void soft_step(const Score<T, CAP, BIAS>& rule, const Row& row, bool whole, int j0, int half,
                                 f32x16 (&s)[N], f32x16 (&acc)[ND], Soft& st) {
    constexpr bool RAW = !CAP && !BIAS;
    const float unit = RAW ? rule.unit : 1.0f;
    const float dist = static_cast<float>(row.pos - j0 - 4 * half);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float t = s[n][r], dt;
            if (!RAW) t = rule.of(t, dist - static_cast<float>(32 * n + acc_row(r, 0)), dt);
            s[n][r] = t;
        }
    if (MASKED && !whole) {
        const unsigned at = static_cast<unsigned>(j0 + 4 * half - row.lo);  // seen: at + key's place < len
        const unsigned len = row.hi > row.lo ? static_cast<unsigned>(row.hi - row.lo) : 0u;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                s[n][r] = at + static_cast<unsigned>(32 * n + acc_row(r, 0)) < len ? s[n][r] : -INF;
        asm volatile("");  // a branch
    }
    float mx = -INF;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[n][r]);
    mx = max32(mx);
    // each row by its own maximum: its sums do not depend on its neighbours'
    const bool moves = (mx - st.m) * unit > 8.0f || (st.m == -INF && mx > -INF);
    if (__builtin_amdgcn_ballot_w64(moves)) {
        const float m = moves ? mx : st.m;
        const float f = __builtin_amdgcn_exp2f((st.m - (m == -INF ? 0.0f : m)) * unit);
        st.l *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] *= f;
        st.m = m;
        asm volatile("");  // a branch, not sixty-four selects
    }
    const float m0 = (st.m == -INF ? 0.0f : st.m) * unit;
    float sum = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            const float p = __builtin_amdgcn_exp2f(RAW ? __builtin_fmaf(s[n][r], unit, -m0) : s[n][r] - m0);
            s[n][r] = p;
            sum += p;
        }
    st.l += sum;
}

// A column's output and lse, or its unfinished state where the keys are
// split. m in log2 units.
template <class T, int DP>
__device__ inline void finish(const Fwd& p, int kvh, int e, int row, int head, int split, int half,
                              const f32x16 (&acc)[DP / 32], float m, float l) {
    const Args& a = p.a;
    if (p.splits > 1) {
        const long at = (static_cast<long>(split) * a.Hkv + kvh) * a.E + e;
        float* o = p.part_o + at * a.D;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int d = 32 * dt + 8 * g + 4 * half;
                store4(o + d, a.D - d, true, acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]);
            }
        if (!half) {
            p.part_ml[2 * at] = m;
            p.part_ml[2 * at + 1] = l;
        }
        return;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* o = static_cast<T*>(p.O) + row * p.o_rs + head * p.o_hs;
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = 32 * dt + 8 * g + 4 * half;
            store4(o + d, p.D_out - d, p.vec_o, acc[dt][4 * g] * inv, acc[dt][4 * g + 1] * inv, acc[dt][4 * g + 2] * inv,
                   acc[dt][4 * g + 3] * inv);
        }
    if (!half) p.lse[static_cast<long>(head) * a.m.Tq + row] = l == 0.0f ? -INF : m * LN2 + logf(l);
}

// A block holds 128 / KS entries of one key head (32 per KS waves) and walks
// the keys that its rows see in tiles of 64, staged in shared memory two
// buffers deep with the next tile on its way. Two waves that share entries
// (KS) take 32 keys of each tile and are joined at the end.
// FOUR: the two halves of a tile one after the other, which leaves registers
// for a fourth wave per SIMD.
template <class T, int DP, int CAP, bool BIAS, int KS, bool FOUR = false>
__global__ __launch_bounds__(AT, sizeof(T) == 2 ? (FOUR ? 4 : DP == 64 ? 3 : 2) : 1) void attn_fwd_k(Fwd p) {
    constexpr int NC = DP / 16, ND = DP / 32;
    __shared__ __align__(16) T sk0[BN * DP], sk1[BN * DP], sv0[BN * DP], sv1[BN * DP];
    __shared__ unsigned bad[3][2];  // rows of the tile that hold values that are not finite
    __shared__ int red[4][4];
    __shared__ float sml[2][2][KS == 2 ? 64 : 1];
    const Args& a = p.a;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5;
    const int group = wave / KS, part = wave % KS;  // of the block's entries, of a tile's keys
    const int kvh = blockIdx.x % a.Hkv;
    int tile = blockIdx.x / a.Hkv;
    if (a.m.causal) tile = gridDim.x / a.Hkv - 1 - tile;  // the longest walks first
    Span sp;
    if (!span_at(a, BM / KS, tile, group, sp)) return;
    const Entry en = entry_of(a, kvh, sp.e0, sp.end, false);
    const bool valid = en.valid;
    const int row = en.row, head = en.head;
    const Row me = row_of(a, sp, en);
    if (tid < 6) bad[tid >> 1][tid & 1] = 0;
    const Walk w = walk_of(me, valid, red);
    const int tiles = w.hi > w.lo ? (w.hi - w.lo + BN - 1) / BN : 0;
    const int split = blockIdx.y;
    const int t0 = static_cast<int>(static_cast<long>(tiles) * split / p.splits);
    const int t1 = static_cast<int>(static_cast<long>(tiles) * (split + 1) / p.splits);

    const Score<T, CAP, BIAS> rule(a, head);
    Frag<T> q[NC];
    const T* qp = static_cast<const T*>(a.Q.p) + row * a.Q.rs + head * a.Q.hs;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int d = 16 * c + 8 * half;
        q[c] = load8(qp + d, valid ? min(8, a.D - d) : 0, true);
    }
    const T* kb = static_cast<const T*>(a.K.p) + kvh * a.K.hs;
    const T* vb = static_cast<const T*>(a.V.p) + kvh * a.V.hs;
    Copy<T, DP, BN, AT> ks, vs;
    ks.init(a.K.rs, a.D, tid);
    vs.init(a.V.rs, a.D, tid);
    const auto load = [&](int t, T* tk, T* tv) __attribute__((always_inline)) {
        const int j = w.lo + t * BN;
        ks.load(tk, kb + j * a.K.rs, a.K.rs, w.hi - j, a.D, wave);
        vs.load(tv, vb + j * a.V.rs, a.V.rs, w.hi - j, a.D, wave);
    };
    int f0, f1;
    split_walk(w, t0, t1, f0, f1);
    const auto is_masked = [&](int t) { return t < f0 || t >= f1; };
    // Waits for the thread's own loads of tile t. Values that are not finite
    // become zeros where rows are masked: their product with a probability
    // that the mask made zero would be NaN. A row that does see one of them is
    // marked after the step.
    const auto landed = [&](int t, T* tv) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0);
        if (is_masked(t)) {
            unsigned* m = bad[(t - t0) % 3];
            vs.clean(tv, tid, [&](int r) { atomicOr(&m[r >> 5], 1u << (r & 31)); });
        }
    };
    f32x16 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
    Soft st;
    bool poison = false;
    const auto step = [&](auto masked, int j0, const T* tk, const T* tv) __attribute__((always_inline)) {
        constexpr int N = FOUR || KS == 2 ? 1 : 2;  // 32 keys each, of a step of the softmax
        const bool whole = j0 >= w.wfull_lo && j0 + BN <= w.wfull_hi;
        if (KS == 2) j0 += 32 * part, tk += 32 * part * DP, tv += 32 * part * DP;
#pragma unroll
        for (int n0 = 0; n0 < 2 / KS; n0 += N) {
            f32x16 s[N];
#pragma unroll
            for (int n = 0; n < N; ++n) {
                s[n] = f32x16{};
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    s[n] = mma32(lds_rows<T, DP>(tk, 32 * (n0 + n), c), q[c], s[n]);
                    hold<T>();
                }
            }
            soft_step<decltype(masked)::value>(rule, me, whole, j0 + 32 * n0, half, s, acc, st);
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const Frag<T> v = acc_frag<T>(s[n], c);
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        acc[d] = mma32(lds_cols<DP, true>(tv, 32 * (n0 + n) + 16 * c, 32 * d), v, acc[d]);
                        hold<T>();
                    }
                }
        }
    };
    const auto walk = [&](auto masked, int t, const T* tk, const T* tv, T* nk, T* nv) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked)::value;
        const int j0 = w.lo + t * BN;
        if (t + 1 < t1) load(t + 1, nk, nv);
        if (tid < 2) bad[(t - t0 + 2) % 3][tid] = 0;
        if (w.wlo < j0 + BN && w.whi > j0) {
            step(masked, j0, tk, tv);
            if (MASKED) {
                const unsigned* m = bad[(t - t0) % 3];
                poison |= sees_bad(me.lo, me.hi, j0, m[0] | static_cast<unsigned long long>(m[1]) << 32);
            }
        }
        if (t + 1 < t1) landed(t + 1, nv);
        __syncthreads();
    };
    const auto walks = [&](auto masked, int from, int to) __attribute__((always_inline)) {
        for (int t = from; t < to; t += 2) {
            walk(masked, t, sk0, sv0, sk1, sv1);
            if (t + 1 < to) walk(masked, t + 1, sk1, sv1, sk0, sv0);
        }
    };
    if (t0 < t1) {
        load(t0, sk0, sv0);
        landed(t0, sv0);
        __syncthreads();
    }
    walks(std::true_type{}, t0, f0);
    walks(std::false_type{}, f0, f1);
    walks(std::true_type{}, f1, t1);
    float l = st.l + __shfl_xor(st.l, 32);
    // A row that sees a value that is not finite becomes NaN whole, whichever
    // tile brings the value.
    if (poison || sums_not_finite(acc)) l = __builtin_nanf("");
    if constexpr (KS == 2) {  // the walk's last barrier is behind the tiles' last reads
        float* other = reinterpret_cast<float*>(group ? sk1 : sk0);
        static_assert(sizeof(sk0) >= DP * 32 * sizeof(float), "a wave's sums take a tile's place");
        if (part) {
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) other[(16 * d + r) * 64 + lane] = acc[d][r];
            sml[group][0][lane] = st.m;
            sml[group][1][lane] = l;
        }
        __syncthreads();
        if (part) return;
        const float unit = CAP || BIAS ? 1.0f : rule.unit, om = sml[group][0][lane], m = fmaxf(st.m, om), m0 = m == -INF ? 0.0f : m;
        const float f = __builtin_amdgcn_exp2f((st.m - m0) * unit), of = __builtin_amdgcn_exp2f((om - m0) * unit);
        l = l * f + sml[group][1][lane] * of;
        st.m = m;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] = acc[d][r] * f + other[(16 * d + r) * 64 + lane] * of;
    }
    const Entry to = entry_of(a, kvh, sp.e0, sp.end, true);
    if (to.valid) finish<T, DP>(p, kvh, to.e, to.row, to.head, split, to.half, acc, st.m * (CAP || BIAS ? 1.0f : rule.unit), l);
}

// Few rows over long keys: a block holds the heads of one row that share a
// key head (up to 32) and its waves take the keys in turn, 32 at a time, each
// with a softmax state of its own; the four are joined at the end. Keys go
// from memory into the product's registers, values through the wave's own
// shared memory for their transpose, so no wave waits for another. Bound by
// memory: 48 requests over caches of up to 4096 tokens, 16 heads on 4 of width
// 128, bf16, take 48 us for 206 MB (4.3 TB/s; a large copy 4.7); one request
// over 6000 tokens of 12 heads of width 64 in float takes 21 us for 37 MB, most
// of it the offsets', the first keys' and the join's latency.
template <class T, int DP, int CAP, bool BIAS>
__global__ __launch_bounds__(AT, sizeof(T) == 2 ? 2 : 1) void attn_rows_k(Fwd p, int chunks) {
    constexpr int NC = DP / 16, ND = DP / 32;
    constexpr int JE = 8;  // columns joined at a time
    __shared__ __align__(16) T sv0[4][RN * DP], sv1[4][RN * DP];
    __shared__ float sml[4][2][32];
    typedef float Join[JE][DP + 1];
    static_assert(4 * sizeof(Join) <= sizeof(sv0), "the waves are joined in the values' place");
    Join* so = reinterpret_cast<Join*>(&sv0[0][0]);
    const Args& a = p.a;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5;
    int b = blockIdx.x;
    const int kvh = b % a.Hkv;
    b /= a.Hkv;
    const int chunk = b % chunks, row = b / chunks;
    const int nh = min(32, a.G - 32 * chunk);  // heads of this block
    const bool valid = (lane & 31) < nh;
    const int g = 32 * chunk + (valid ? (lane & 31) : 0), head = kvh * a.G + g, e = row * a.G + g;
    Row me = row_at(a.m, row, row);
    me.lo = __builtin_amdgcn_readfirstlane(me.lo);
    me.hi = __builtin_amdgcn_readfirstlane(me.hi);
    const int keys = me.hi > me.lo ? me.hi - me.lo : 0;
    const int tiles = (keys + RN - 1) / RN, split = blockIdx.y;
    const int t0 = static_cast<int>(static_cast<long>(tiles) * split / p.splits);
    const int t1 = static_cast<int>(static_cast<long>(tiles) * (split + 1) / p.splits);

    const Score<T, CAP, BIAS> rule(a, head);
    Frag<T> q[NC], k[NC];
    int k_at[NC];
    const T* qp = static_cast<const T*>(a.Q.p) + row * a.Q.rs + head * a.Q.hs;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int d = 16 * c + 8 * half;
        q[c] = load8(qp + d, valid ? min(8, a.D - d) : 0, true);
        k_at[c] = d < a.D ? static_cast<int>(((lane & 31) * a.K.rs + d) * static_cast<long>(sizeof(T))) : kFar;
    }
    const T* kb = static_cast<const T*>(a.K.p) + kvh * a.K.hs;
    const T* vb = static_cast<const T*>(a.V.p) + kvh * a.V.hs;
    Copy<T, DP, RN, 64> vs;
    vs.init(a.V.rs, a.D, lane);
    const auto load_k = [&](int t) __attribute__((always_inline)) {
        const int j = me.lo + t * RN;
        const __amdgpu_buffer_rsrc_t r = rows_rsrc(kb + j * a.K.rs, a.K.rs, min(me.hi - j, RN), a.D);
#pragma unroll
        for (int c = 0; c < NC; ++c) k[c] = buffer_load8(r, k_at[c], T{});
    };
    const auto load_v = [&](int t, T* tv) __attribute__((always_inline)) {
        const int j = me.lo + t * RN;
        vs.load(tv, vb + j * a.V.rs, a.V.rs, me.hi - j, a.D, 0);
    };
    f32x16 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
    Soft st;
    const auto walk = [&](int t, const T* tv, T* nv) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0);  // the tile's keys and values have landed
        if (t + 4 < t1) load_v(t + 4, nv);
        const int j0 = me.lo + t * RN;
        f32x16 s[1];
        s[0] = f32x16{};
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            s[0] = mma32(k[c], q[c], s[0]);
            hold<T>();
        }
        if (t + 4 < t1) load_k(t + 4);
        soft_step<true>(rule, me, j0 + RN <= me.hi, j0, half, s, acc, st);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const Frag<T> w = acc_frag<T>(s[0], c);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                acc[d] = mma32(lds_cols<DP, true>(tv, 16 * c, 32 * d), w, acc[d]);
                hold<T>();
            }
        }
    };
    if (t0 + wave < t1) {
        load_v(t0 + wave, sv0[wave]);
        load_k(t0 + wave);
    }
    for (int t = t0 + wave; t < t1; t += 8) {
        walk(t, sv0[wave], sv1[wave]);
        if (t + 4 < t1) walk(t + 4, sv1[wave], sv0[wave]);
    }
    // join the waves: their states' common maximum, then the sums in order
    const float unit = CAP || BIAS ? 1.0f : rule.unit;
    float l = st.l + __shfl_xor(st.l, 32);
    if (sums_not_finite(acc)) l = __builtin_nanf("");
    if (!half) {
        sml[wave][0][lane] = st.m * unit;
        sml[wave][1][lane] = l;
    }
    __syncthreads();
    const int col = lane & 31;
    const float m = fmaxf(fmaxf(sml[0][0][col], sml[1][0][col]), fmaxf(sml[2][0][col], sml[3][0][col]));
    const float m0 = m == -INF ? 0.0f : m;
    const float f = __builtin_amdgcn_exp2f(st.m * unit - m0);
    l = 0.0f;
    for (int w = 0; w < 4; ++w) l += sml[w][1][col] * __builtin_amdgcn_exp2f(sml[w][0][col] - m0);
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
    if (valid && wave == ((col / JE) & 3)) finish<T, DP>(p, kvh, e, row, head, split, half, acc, m, l);
}

// Joins the splits of an entry (at most 64): one wave per entry, a lane for
// every split's state, then lanes over the output, the splits in order.
template <class T>
__global__ __launch_bounds__(64) void attn_join_k(Fwd p) {
    const Args& a = p.a;
    const int lane = threadIdx.x;
    const long w = blockIdx.x, n = static_cast<long>(a.Hkv) * a.E;
    const int kvh = static_cast<int>(w / a.E), e = static_cast<int>(w - static_cast<long>(kvh) * a.E);
    const int row = e / a.G, head = kvh * a.G + e - row * a.G;
    float m = -INF, l = 0.0f;
    if (lane < p.splits) {
        const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + 2 * (lane * n + w));
        m = ml.x;
        l = ml.y;
    }
    float top = m;
    for (int o = 32; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
    const float f = __builtin_amdgcn_exp2f(m - (top == -INF ? 0.0f : top));  // zero past the splits
    l *= f;
    for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o);
    float o[2] = {0.0f, 0.0f};
    for (int s = 0; s < p.splits; s += 8) {  // eight loads in flight
        float v[8][2];
#pragma unroll
        for (int x = 0; x < 8; ++x)
#pragma unroll
            for (int i = 0; i < 2; ++i)
                v[x][i] = s + x < p.splits && lane + 64 * i < p.D_out ? p.part_o[((s + x) * n + w) * a.D + lane + 64 * i] : 0.0f;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            const float g = __shfl(f, s + x);
#pragma unroll
            for (int i = 0; i < 2; ++i) o[i] = __builtin_fmaf(g, v[x][i], o[i]);
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = static_cast<T*>(p.O) + row * p.o_rs + head * p.o_hs;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int d = lane + 64 * i;
        if (d < p.D_out) out[d] = static_cast<T>(o[i] * inv);
    }
    if (lane == 0) p.lse[static_cast<long>(head) * a.m.Tq + row] = l == 0.0f ? -INF : top * LN2 + logf(l);
}

// Whether a fourth wave per SIMD fits (a cap or a bias takes its registers).
template <class T, int DP>
constexpr bool four_fit(bool shaped) { return sizeof(T) == 2 && DP == 64 && !shaped; }

struct Launch {
    template <class T, int DP, int CAP, bool BIAS>
    static int run(kdec_ctx* ctx, const Fwd& p, dim3 grid, bool rows, int chunks, int shared, bool four) {
        if (rows) hipLaunchKernelGGL((attn_rows_k<T, DP, CAP, BIAS>), grid, dim3(AT), 0, ctx->stream, p, chunks);
        else if (shared == 2) hipLaunchKernelGGL((attn_fwd_k<T, DP, CAP, BIAS, 2>), grid, dim3(AT), 0, ctx->stream, p);
        else if (four_fit<T, DP>(CAP || BIAS) && four)
            hipLaunchKernelGGL((attn_fwd_k<T, DP, CAP, BIAS, 1, four_fit<T, DP>(CAP || BIAS)>), grid, dim3(AT), 0, ctx->stream, p);
        else hipLaunchKernelGGL((attn_fwd_k<T, DP, CAP, BIAS, 1>), grid, dim3(AT), 0, ctx->stream, p);
        if (p.splits > 1)
            hipLaunchKernelGGL(attn_join_k<T>, dim3(static_cast<unsigned>(static_cast<long>(p.a.Hkv) * p.a.E)), dim3(64), 0,
                               ctx->stream, p);
        return launch_check(ctx, "kdec_attn_fwd");
    }
};

}  // namespace
}  // namespace attn
}  // namespace kdec

using namespace kdec;
using namespace kdec::attn;

extern "C" int kdec_attn_fwd(kdec_ctx* ctx, int dtype, const void* Q, long q_rs, long q_hs, const void* K, long k_rs,
                             long k_hs, const void* V, long v_rs, long v_hs, const int* q_off, const int* k_off,
                             const int* k_len, const int* prefix, int docs, int causal, const float* slopes, float scale,
                             float cap, int Tq, int Tk, int Hq, int Hkv, int D, void* O, long o_rs, long o_hs, float* lse) {
    if (!ctx) return KDEC_EINVAL;
    if (int rc = check(ctx, "kdec_attn_fwd", dtype, q_off, k_off, docs, scale, cap, Tq, Tk, Hq, Hkv, D)) return rc;
    if (Tq == 0) return KDEC_OK;
    KDEC_CHECK(ctx, Q && O && lse && (Tk == 0 || (K && V)), "kdec_attn_fwd: null tensor");
    KDEC_CHECK(ctx, apart(o_rs, o_hs, Tq, Hq, D), "kdec_attn_fwd: rows of O overlap");
    const size_t size = dtype == KDEC_F32 ? 4 : 2;
    const int G = Hq / Hkv;
    ProfScope ps(ctx, "attn", 0.0, 0.0);
    Fwd p{};
    p.a = Args{{Q, q_rs, q_hs}, {K, k_rs, k_hs}, {V, v_rs, v_hs}, {q_off, k_off, k_len, prefix, docs, causal != 0, Tq, Tk},
               slopes, scale, cap, Hq, Hkv, G, D, Tq * G, false};
    std::unique_ptr<Workspace> packed[3], ws;
    if (!plain(p.a.Q, D, size) || !plain(p.a.K, D, size) || !plain(p.a.V, D, size)) {
        if (int rc = pack(ctx, dtype, p.a.Q, Tq, Hq, D, packed[0])) return rc;
        if (int rc = pack(ctx, dtype, p.a.K, Tk, Hkv, D, packed[1])) return rc;
        if (int rc = pack(ctx, dtype, p.a.V, Tk, Hkv, D, packed[2])) return rc;
        p.a.D = (D + 7) & ~7;
    }
    p.O = O;
    p.o_rs = o_rs;
    p.o_hs = o_hs;
    p.vec_o = D % 4 == 0 && aligned(Heads{O, o_rs, o_hs}, size, 4 * size);
    p.lse = lse;
    p.D_out = D;
    const int chunks = static_cast<int>(cdiv(G, 32));
    const int shared = waves_shared(ctx, cdiv(p.a.E, BM) * Hkv), held = BM / shared;
    p.a.by_doc = rows_by_document(ctx, docs, Tk, p.a.E, Hkv, held);
    // One row per document over many keys: a block per row. From two on, blocks
    // that end with their document read the keys once for all rows (bf16, 16
    // heads on 4 of width 128, 48 documents of 2000 keys: 2 rows 68 us for 48, 3
    // 74 for 48, 4 77 for 49), and where these would hold several documents, each
    // other's keys as well (1 row 43 for 135). A few rows of padding leave it at
    // that: their blocks end at once (1000 documents of 200 keys, 12 heads of
    // width 64, 24 rows more: 128 us, in blocks of several 259).
    const bool rows = static_cast<long>(Tk) >= 8L * Tq && Tq <= (p.a.by_doc ? docs : docs + docs / 4);
    const long tiles = rows ? static_cast<long>(Tq) * chunks : doc_blocks(p.a.by_doc, docs, p.a.E, held);
    const long blocks = tiles * Hkv;
    KDEC_CHECK(ctx, blocks < INT_MAX, "kdec_attn_fwd: too many rows");
    // Split the keys where the rows alone do not fill the device, to no fewer
    // than 256 keys a part (of 128, one float token over 6000 keys of 12 heads
    // takes 29 us with the join, of 256 it takes 26). Few rows take twice as
    // many parts: their documents differ in length, and the longest ends last.
    const long each = docs > 0 ? Tk / docs : 0;
    long splits = cdiv((rows ? 4L : 2L) * ctx->num_cus, blocks);
    if (splits > each / 256) splits = each / 256;
    if (splits > 64) splits = 64;  // what the join holds
    if (splits < 1) splits = 1;
    p.splits = static_cast<int>(splits);
    if (splits > 1) {
        const size_t n = static_cast<size_t>(splits) * Hkv * p.a.E;
        ws = std::make_unique<Workspace>(ctx, n * (p.a.D + 2) * sizeof(float));
        if (!ws->p) return KDEC_ENOMEM;
        p.part_o = ws->as<float>();
        p.part_ml = p.part_o + n * p.a.D;
    }
    // Four waves per SIMD where three do not hold all blocks at once and walks
    // are short, so that more of them side by side even out; long ones lose more
    // to the shorter steps (bf16, 12 heads of width 64, three and four waves: 32
    // texts of 20 to 510 rows 28.8 and 26.1 us, 64 of 256 37.2 and 33.7, 120 of
    // 128 27.7 and 25.2, 40 of 280 33.9 and 33.7, of 200 to 360 33.7 and 35.3, 100
    // of 500 151 and 143, 60 of 520 101 and 98, but 24 of 700 62.7 and 64.1, 8 of
    // 1024 42.8 and 45.2, 1 of 8192 246 and 262). The host knows the lengths' mean.
    // A document's last block counts half.
    const long real = (cdiv(p.a.E, BM) + docs / 2) * Hkv;
    const bool four = shared == 1 && real > 3L * ctx->num_cus && each <= 512;
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(splits));
    return dispatch<Launch>(dtype, D, cap, slopes != nullptr, ctx, p, grid, rows, chunks, shared, four);
}
