// Attention of packed documents on gfx950, backward.
//
// With P = exp(s - lse) formed again from the products and the forward's lse,
// delta = dO . O and dS = P (dO V^T - delta) (times the cap's derivative):
//   dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO.
// Two walks rather than one: dQ sums over a row's keys and is a walk over the
// keys as the forward is, dK and dV sum over a key's rows and heads and are a
// walk over those. Each then has one owner per result, which no other block
// adds to: five products would do for seven, but the sums would be made by
// atomics in an order that changes from call to call.
//
// 8192 causal rows, 16 heads on 4 of width 128, bf16: dQ 434 us (950 TFLOP/s of
// its three products), dK and dV 565 (970 of four), bound by the matrix units
// and the exponentials between the products. Packed texts of 20 to 510 tokens,
// 12 heads of width 64: 49 and 46 us.
//
// P and dS are rounded to the tensors' type for the products they enter (dS of
// masked tiles to twice its bits in dQ).
#include "kdec_attn.hpp"

namespace kdec {
namespace attn {
namespace {

struct Bwd {
    Args a;
    Heads O, dO;
    bool vec_o;  // O takes 16-byte loads
    const float* lse;
    int D_out;  // the gradients' width (a.D may be padded)
    void *dQ, *dK, *dV;
    long dq_rs, dq_hs, dk_rs, dk_hs, dv_rs, dv_hs;
    bool vec_dq, vec_dk, vec_dv;
    Row* rows;    // (Tq)
    float2* stat; // (Hq, Tq): lse in log2 units, delta = dO . O
    bool by_doc_k;  // blocks of keys end with their document
    int parts;    // blocks that share a key tile's rows
    float* part;  // (parts, Hkv, Tk, 2, D): their dK / scale and dV
};

// dQ: the forward's walk over the keys, with dQ^T = K^T dS^T in place of the
// output. Before it a block forms delta = dO . O of its rows and heads and
// writes what the walk over the rows takes: delta, lse in log2 units, and the
// rows' keys. O is rounded, and so is delta; but as sum_j P (dP - delta') is
// delta - delta', the walk's sums of dS give what is missing, and dK gets
// delta to float. Of dQ the missing part is about 2^-9 / sqrt(keys), so that
// rows of few keys show it: they only meet masked tiles, where dS enters the
// product as two terms, which leaves such rows the one error and the others
// that of dS's rounding. A row without keys gets lse = +inf, so that its probabilities
// are zeros; one whose query or delta is not finite gets NaN, which then marks
// every gradient that the row reaches. So does one that sees a key that is not
// finite: masked tiles clean such keys and note which they were, and in whole
// tiles they make a sum of dQ that is not finite.
template <class T, int DP, int CAP, bool BIAS, int KS>
__global__ __launch_bounds__(AT, (sizeof(T) == 2 ? 2 : 1) + (DP == 64 && !(sizeof(T) == 2 && CAP == FINE_CAP && BIAS))) void attn_dq_k(Bwd b) {
    constexpr int NC = DP / 16, ND = DP / 32;
    __shared__ __align__(16) T sk0[BN * DP], sk1[BN * DP], sv0[BN * DP], sv1[BN * DP];
    __shared__ unsigned bad[3][2];  // keys of the tile that are not finite
    __shared__ int red[4][4];
    __shared__ float srest[2][KS == 2 ? 64 : 1];
    const Args& a = b.a;
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
    const int t1 = w.hi > w.lo ? (w.hi - w.lo + BN - 1) / BN : 0;

    const Score<T, CAP, BIAS> rule(a, head);
    Frag<T> q[NC], g[NC];
    const T* qp = static_cast<const T*>(a.Q.p) + row * a.Q.rs + head * a.Q.hs;
    const T* gp = static_cast<const T*>(b.dO.p) + row * b.dO.rs + head * b.dO.hs;
    const T* op = static_cast<const T*>(b.O.p) + row * b.O.rs + head * b.O.hs;
    float lse2 = INF, delta = 0.0f;
    bool wild = false;  // (capped scores of such a query are finite)
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int d = 16 * c + 8 * half, n = valid ? min(8, a.D - d) : 0;
        q[c] = load8(qp + d, n, true);
        g[c] = load8(gp + d, n, true);
        wild |= not_finite(q[c]);
        const Frag<T> o = load8(op + d, valid ? min(8, b.D_out - d) : 0, b.vec_o);
#pragma unroll
        for (int i = 0; i < 8; ++i) delta = __builtin_fmaf(static_cast<float>(o[i]), static_cast<float>(g[c][i]), delta);
        if (sizeof(T) == 4) __builtin_amdgcn_sched_barrier(0);
    }
    delta += __shfl_xor(delta, 32);
    wild |= __shfl_xor(wild, 32) != 0;
    if (valid) {
        const float lse = b.lse[static_cast<long>(head) * a.m.Tq + row];
        lse2 = lse == -INF ? INF : lse * LOG2E;
        if (me.hi <= me.lo) delta = 0.0f;
        else if (wild || !(__builtin_fabsf(delta) < INF)) lse2 = __builtin_nanf("");
        if (!half && head == 0) b.rows[row] = me;
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
    split_walk(w, 0, t1, f0, f1);
    const auto landed = [&](int t, T* tk) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0);
        if (t < f0 || t >= f1) {  // a zero of dS times such a key
            unsigned* m = bad[t % 3];
            ks.clean(tk, tid, [&](int r) { atomicOr(&m[r >> 5], 1u << (r & 31)); });
        }
    };
    f32x16 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
    float rest = 0.0f;
    const auto step = [&](auto masked, int j0, const T* tk, const T* tv) __attribute__((always_inline)) {
        constexpr bool MASKED = decltype(masked)::value;
        const bool whole = j0 >= w.wfull_lo && j0 + BN <= w.wfull_hi;
        if (KS == 2) j0 += 32 * part, tk += 32 * part * DP, tv += 32 * part * DP;
        const unsigned at = static_cast<unsigned>(j0 + 4 * half - me.lo);
        const unsigned len = me.hi > me.lo ? static_cast<unsigned>(me.hi - me.lo) : 0u;
        const float dist = static_cast<float>(me.pos - j0 - 4 * half);
#pragma unroll
        for (int n = 0; n < 2 / KS; ++n) {
            f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                s = mma32(lds_rows<T, DP>(tk, 32 * n, c), q[c], s);
                hold<T>();
                dp = mma32(lds_rows<T, DP>(tv, 32 * n, c), g[c], dp);
                hold<T>();
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int k = 32 * n + acc_row(r, 0);
                float dt;
                const float ds = grad_p(rule, s[r], dist - static_cast<float>(k), lse2, dt) * (dp[r] - delta);
                s[r] = ds * dt;
                if (CAP) rest += !MASKED || at + static_cast<unsigned>(k) < len ? ds : 0.0f;
            }
            if (MASKED && !whole) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = at + static_cast<unsigned>(32 * n + acc_row(r, 0)) < len ? s[r] : 0.0f;
                asm volatile("");  // a branch
            }
            if (!CAP) {
#pragma unroll
                for (int r = 0; r < 16; ++r) rest += s[r];
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Terms<T, MASKED ? 2 : 1> ds(acc_floats(s, c));
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const Frag<T> kt = lds_cols<DP, true>(tk, 32 * n + 16 * c, 32 * d);
#pragma unroll
                    for (int x = ds.n - 1; x >= 0; --x) acc[d] = mma32(kt, ds.t[x], acc[d]);
                    hold<T>();
                }
            }
        }
    };
    const auto walk = [&](auto masked, int t, const T* tk, const T* tv, T* nk, T* nv) __attribute__((always_inline)) {
        const int j0 = w.lo + t * BN;
        if (t + 1 < t1) load(t + 1, nk, nv);
        if (tid < 2) bad[(t + 2) % 3][tid] = 0;
        if (w.wlo < j0 + BN && w.whi > j0) {
            step(masked, j0, tk, tv);
            if (decltype(masked)::value) {
                const unsigned* m = bad[t % 3];
                if (sees_bad(me.lo, me.hi, j0, m[0] | static_cast<unsigned long long>(m[1]) << 32)) rest = __builtin_nanf("");
            }
        }
        if (t + 1 < t1) landed(t + 1, nk);
        __syncthreads();
    };
    const auto walks = [&](auto masked, int from, int to) __attribute__((always_inline)) {
        for (int t = from; t < to; t += 2) {
            walk(masked, t, sk0, sv0, sk1, sv1);
            if (t + 1 < to) walk(masked, t + 1, sk1, sv1, sk0, sv0);
        }
    };
    if (t1 > 0) {
        load(0, sk0, sv0);
        landed(0, sk0);
        __syncthreads();
    }
    walks(std::true_type{}, 0, f0);
    walks(std::false_type{}, f0, f1);
    walks(std::true_type{}, f1, t1);
    if constexpr (KS == 2) {  // the walk's last barrier is behind the tiles' last reads
        float* other = reinterpret_cast<float*>(group ? sk1 : sk0);
        static_assert(sizeof(sk0) >= DP * 32 * sizeof(float), "a wave's sums take a tile's place");
        if (part) {
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int r = 0; r < 16; ++r) other[(16 * d + r) * 64 + lane] = acc[d][r];
            srest[group][lane] = rest;
        }
        __syncthreads();
        if (part) return;
        rest += srest[group][lane];
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] += other[(16 * d + r) * 64 + lane];
    }
    const Entry to = entry_of(a, kvh, sp.e0, sp.end, true);
    if (!to.valid) return;
    rest += __shfl_xor(rest, 32);
    float scale = a.scale;
    if (sums_not_finite(acc) || !(__builtin_fabsf(rest) < INF)) scale = lse2 = __builtin_nanf("");
    if (!to.half) b.stat[static_cast<long>(to.head) * a.m.Tq + to.row] = make_float2(lse2, delta + rest);
    T* o = static_cast<T*>(b.dQ) + to.row * b.dq_rs + to.head * b.dq_hs;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int d = 32 * dt + 8 * x + 4 * to.half;
            store4(o + d, b.D_out - d, b.vec_dq, acc[dt][4 * x] * scale, acc[dt][4 * x + 1] * scale, acc[dt][4 * x + 2] * scale,
                   acc[dt][4 * x + 3] * scale);
        }
}

// dK and dV: a block holds 32 keys for each of its KG pairs of waves (keys and
// values in registers) and walks the rows that see them, head by head of the
// group, in tiles of 64 whose queries and output gradients are staged in
// shared memory, two buffers deep and two tiles a turn. Scores are S = Q K^T
// here, a lane holding one key's column. The waves of a pair form P and dS of
// one half of a tile each, hand each other what it takes to keep one sum per
// wave -- the first gets the other's P and sums dV over the whole tile, the
// second the other's dS and sums dK -- and so hold half the accumulators
// each, which leaves room for two waves per SIMD whose arithmetic and
// products overlap (one wave with both sums: 900 us where two take 630, 8192
// causal rows of 16 heads on 4, width 128). All heads of the group belong to the
// same walk, so the sums over shared heads need no joining; where the key
// tiles alone do not fill the device, `parts` blocks share a walk and
// attn_dkv_join_k adds their sums.
// Wide heads in float, or with a bias, take the registers of a whole SIMD per
// wave: two pairs.
template <class T, int DP, bool BIAS> constexpr int key_groups() { return DP == 64 ? 2 : sizeof(T) == 4 || BIAS ? 2 : 4; }

template <class T, int DP, int CAP, bool BIAS>
__global__ __launch_bounds__((128 * key_groups<T, DP, BIAS>()), (sizeof(T) == 2 && DP == 64 ? 3 : key_groups<T, DP, BIAS>() == 4 ? 2 : 1)) void attn_dkv_k(Bwd b) {
    constexpr int NC = DP / 16, ND = DP / 32, BE = 64, PAIR = 2 * BE, KG = key_groups<T, DP, BIAS>(), NT = 128 * KG, KEYS = 32 * KG;
    // (aligned to come first: within the reach of the reads' own offsets)
    __shared__ __align__(256) T sq0[BE * DP], sq1[BE * DP], sg0[BE * DP], sg1[BE * DP];
    __shared__ Frag<T> pass[KG][2][2][64];  // by pair, half of the tile, step: the other wave's operand
    __shared__ int some[KG][2];             // whether the half's rows see any of the pair's keys
    __shared__ __align__(16) float slse[2][BE], sdelta[2][BE];
    __shared__ __align__(16) int slo[2][BE], shi[2][BE], spos[2][BE];
    const Args& a = b.a;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5;
    const int pair = wave % KG, role = wave / KG;
    const int kvh = blockIdx.x % a.Hkv, part = blockIdx.y;
    int j0 = (blockIdx.x / a.Hkv) * KEYS, end = a.m.Tk;  // the block's keys
    Piece piece{};
    if (b.by_doc_k) {
        if (!piece_at(a.m.k_off, a.m.docs, a.m.Tk, 1, KEYS, blockIdx.x / a.Hkv, piece)) return;
        j0 = piece.lo + piece.place * KEYS;
        end = piece.hi;
    }
    const int wkey = j0 + pair * 32, key = wkey + (lane & 31);
    const bool valid = key < end;

    // The rows [e0, e1) that may see keys of the block, and those [f0, f1)
    // that all see all of its keys below `stop`. Where a block ends with its
    // document, stop is the end of the document's keys: what a lane forms for
    // keys past it is dropped at the end.
    int e0 = 0, e1 = 0, f0 = 0, f1 = 0, stop = j0 + KEYS;
    {
        int d0, d1;
        if (b.by_doc_k) {
            d0 = piece.doc;
            d1 = piece.doc < a.m.docs ? piece.doc : -1;
        } else {
            d0 = max(doc_of(a.m.k_off, a.m.docs, j0), 0);
            d1 = doc_of(a.m.k_off, a.m.docs, min(j0 + KEYS, a.m.Tk) - 1);
        }
        if (d1 >= 0) {
            const Doc c = doc_at(a.m, d0), z = doc_at(a.m, d1);
            const int skip = c.lk - c.lq;  // position of the first row's key
            if (b.by_doc_k) stop = min(stop, c.k0 + c.lk);
            e0 = c.q0;
            if (a.m.causal && j0 - c.k0 >= c.prefix) e0 = min(max(c.q0 + (j0 - c.k0) - skip, c.q0), c.q0 + c.lq);
            e1 = z.q0 + z.lq;
            if (b.by_doc_k && j0 >= stop) e1 = e0;
            if (d0 == d1 && j0 >= c.k0 && j0 < stop && stop <= c.k0 + c.lk) {
                f0 = c.q0;
                if (a.m.causal && stop - c.k0 > c.prefix) f0 = min(max(c.q0 + (stop - 1 - c.k0) - skip, c.q0), c.q0 + c.lq);
                f1 = c.q0 + c.lq;
            }
        }
        e0 = __builtin_amdgcn_readfirstlane(e0);
        e1 = __builtin_amdgcn_readfirstlane(e1);
        f0 = __builtin_amdgcn_readfirstlane(f0);
        f1 = __builtin_amdgcn_readfirstlane(f1);
        stop = __builtin_amdgcn_readfirstlane(stop);
    }
    const int wstop = min(wkey + 32, stop);
    // Turns of two tiles, the group's heads one after another; of a head's
    // `per` turns, [p0, p1) are seen whole (rows past e1 are zeros and have
    // probabilities of zero, so the last turn may end anywhere).
    const int per = e1 > e0 ? (e1 - e0 + PAIR - 1) / PAIR : 0;
    int p0 = 0, p1 = 0;
    if (f1 > f0) {
        p0 = max((f0 - e0 + PAIR - 1) / PAIR, 0);
        p1 = f1 >= e1 ? per : (f1 - e0) / PAIR;
        if (p0 >= p1) p0 = p1 = 0;
    }
    const long turns = static_cast<long>(per) * a.G;
    const int u0 = static_cast<int>(turns * part / b.parts), u1 = static_cast<int>(turns * (part + 1) / b.parts);

    Frag<T> k[NC], v[NC];
    const T* kp = static_cast<const T*>(a.K.p) + kvh * a.K.hs + static_cast<long>(valid ? key : 0) * a.K.rs;
    const T* vp = static_cast<const T*>(a.V.p) + kvh * a.V.hs + static_cast<long>(valid ? key : 0) * a.V.rs;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
        const int d = 16 * c + 8 * half, n = valid ? min(8, a.D - d) : 0;
        k[c] = load8(kp + d, n, true);
        v[c] = load8(vp + d, n, true);
    }
    Copy<T, DP, BE, NT> qs, gs;
    qs.init(a.Q.rs, a.D, tid);
    gs.init(b.dO.rs, a.D, tid);
    int left = 2 * (u1 - u0), lg = 0, li = 0;  // tiles to load; the next one's head and place
    if (left) {
        lg = u0 / per;
        li = 2 * (u0 - lg * per);
    }
    float2 r_stat = make_float2(0.0f, 0.0f);
    Row r_row{0, 0, 0};
    bool l_masked = true;  // of the tile last asked for
    const auto load = [&](T* tq, T* tg) __attribute__((always_inline)) {
        const int head = kvh * a.G + lg, r = e0 + li * BE;
        qs.load(tq, static_cast<const T*>(a.Q.p) + head * a.Q.hs + r * a.Q.rs, a.Q.rs, e1 - r, a.D, wave);
        gs.load(tg, static_cast<const T*>(b.dO.p) + head * b.dO.hs + r * b.dO.rs, b.dO.rs, e1 - r, a.D, wave);
        if (tid < BE) {
            r_stat = make_float2(INF, 0.0f);
            r_row = Row{INT_MAX, INT_MIN, 0};
            if (r + tid < e1) {
                r_stat = b.stat[static_cast<long>(head) * a.m.Tq + r + tid];
                r_row = b.rows[r + tid];
            }
        }
        l_masked = (li >> 1) < p0 || (li >> 1) >= p1;
        --left;
        if (++li == 2 * per) {
            li = 0;
            ++lg;
        }
    };
    const auto landed = [&](T* tq, T* tg, int buf) __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0);
        if (tid < BE) {
            slse[buf][tid] = r_stat.x;
            sdelta[buf][tid] = r_stat.y;
            slo[buf][tid] = r_row.lo;
            shi[buf][tid] = r_row.hi;
            spos[buf][tid] = r_row.pos;
        }
        if (l_masked) {  // zeros of P and dS times such values
            qs.clean(tq, tid, [](int) {});
            gs.clean(tg, tid, [](int) {});
        }
    };
    // The two waves of a pair run code of their own, with the same barriers.
    const auto run = [&](auto which) __attribute__((always_inline)) {
        constexpr int ROLE = decltype(which)::value;
        f32x16 acc[ND];  // dV (the pair's first wave) or dK / scale (its second)
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
        const auto step = [&](auto masked, const Score<T, CAP, BIAS>& rule, const T* tq, const T* tg, int buf)
                              __attribute__((always_inline)) {
            constexpr bool MASKED = decltype(masked)::value;
            constexpr int n0 = 32 * ROLE;  // the wave's half
            const T *hq = tq + n0 * DP, *hg = tg + n0 * DP;
            bool any = wkey < wstop, whole = true;  // some, all of the half's rows and the wave's keys meet
            if (MASKED) {
                const int i = n0 + (lane & 31), lo = slo[buf][i], hi = shi[buf][i];
                any = __builtin_amdgcn_ballot_w64(lo < wstop && hi > wkey) != 0;
                whole = __builtin_amdgcn_ballot_w64(!(lo <= wkey && hi >= wstop)) == 0;
                if (lane == 0) some[pair][ROLE] = any;
            }
            Frag<T> own[2];
            if (any) {
                f32x16 s = f32x16{}, p = f32x16{};  // products, then dS and P
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    s = mma32(lds_rows<T, DP>(hq, 0, c), k[c], s);
                    hold<T>();
                    p = mma32(lds_rows<T, DP>(hg, 0, c), v[c], p);
                    hold<T>();
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int i0 = n0 + 8 * q + 4 * half;
                    const f32x4 lse = *reinterpret_cast<const f32x4*>(&slse[buf][i0]);
                    const f32x4 delta = *reinterpret_cast<const f32x4*>(&sdelta[buf][i0]);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int r = 4 * q + x, i = i0 + x;
                        float dt;
                        float pr = grad_p(rule, s[r], BIAS ? static_cast<float>(spos[buf][i] - key) : 0.0f, lse[x], dt);
                        s[r] = pr * (p[r] - delta[x]) * dt;
                        p[r] = pr;
                    }
                    if (MASKED || CAP || BIAS) __builtin_amdgcn_sched_barrier(0);
                    hold<T>();
                }
                if (MASKED && !whole) {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        typedef int i32x4 __attribute__((ext_vector_type(4)));
                        const i32x4 lo = *reinterpret_cast<const i32x4*>(&slo[buf][n0 + 8 * q + 4 * half]);
                        const i32x4 hi = *reinterpret_cast<const i32x4*>(&shi[buf][n0 + 8 * q + 4 * half]);
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const bool seen = key >= lo[x] && key < hi[x];
                            p[4 * q + x] = seen ? p[4 * q + x] : 0.0f;
                            s[4 * q + x] = seen ? s[4 * q + x] : 0.0f;
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    asm volatile("");  // a branch
                }
                if constexpr (ROLE) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        own[c] = acc_frag<T>(s, c);
                        pass[pair][1][c][lane] = acc_frag<T>(p, c);
                    }
                } else {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        own[c] = acc_frag<T>(p, c);
                        pass[pair][0][c][lane] = acc_frag<T>(s, c);
                    }
                }
            }
            __syncthreads();
            const T *mine = ROLE ? hq : hg, *other = (ROLE ? tq : tg) + (32 - n0) * DP;
            if (any) {
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        acc[d] = mma32(lds_cols<DP, true>(mine, 16 * c, 32 * d), own[c], acc[d]);
                        hold<T>();
                    }
            }
            if (MASKED ? some[pair][1 - ROLE] : any) {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const Frag<T> f = pass[pair][1 - ROLE][c][lane];
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        acc[d] = mma32(lds_cols<DP, true>(other, 16 * c, 32 * d), f, acc[d]);
                        hold<T>();
                    }
                }
            }
        };
        const auto walks = [&](auto masked, const Score<T, CAP, BIAS>& rule, int from, int to) __attribute__((always_inline)) {
            for (int i = from; i < to; ++i) {
                load(sq1, sg1);
                step(masked, rule, sq0, sg0, 0);
                landed(sq1, sg1, 1);
                __syncthreads();
                const bool more = left > 0;
                if (more) load(sq0, sg0);
                step(masked, rule, sq1, sg1, 1);
                if (more) landed(sq0, sg0, 0);
                __syncthreads();
            }
        };
        if (left) {
            load(sq0, sg0);
            landed(sq0, sg0, 0);
            __syncthreads();
            for (int u = u0; u < u1;) {
                const int g = u / per, i0 = u - g * per, i1 = min(per, i0 + u1 - u);
                const Score<T, CAP, BIAS> rule(a, kvh * a.G + g);
                walks(std::true_type{}, rule, i0, min(p0, i1));
                walks(std::false_type{}, rule, max(i0, p0), min(p1, i1));
                walks(std::true_type{}, rule, max(i0, p1), i1);
                u += i1 - i0;
            }
        }
        if (!valid) return;
        if (key >= stop) {
#pragma unroll
            for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
        }
        T* out = ROLE ? static_cast<T*>(b.dK) + kvh * b.dk_hs + key * b.dk_rs : static_cast<T*>(b.dV) + kvh * b.dv_hs + key * b.dv_rs;
        const float f = ROLE ? a.scale : 1.0f;
        float* o = b.part + (((static_cast<long>(part) * a.Hkv + kvh) * a.m.Tk + key) * 2 + 1 - ROLE) * a.D;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int d = 32 * dt + 8 * q + 4 * half;
                if (b.parts > 1)
                    store4(o + d, a.D - d, true, acc[dt][4 * q], acc[dt][4 * q + 1], acc[dt][4 * q + 2], acc[dt][4 * q + 3]);
                else
                    store4(out + d, b.D_out - d, ROLE ? b.vec_dk : b.vec_dv, acc[dt][4 * q] * f, acc[dt][4 * q + 1] * f,
                           acc[dt][4 * q + 2] * f, acc[dt][4 * q + 3] * f);
            }
    };
    if (role) run(std::integral_constant<int, 1>{});
    else run(std::integral_constant<int, 0>{});
}

// The parts' dK and dV added in their order, four columns a thread.
template <class T>
__global__ __launch_bounds__(AT) void attn_dkv_join_k(Bwd b) {
    const Args& a = b.a;
    const long n = static_cast<long>(a.Hkv) * a.m.Tk * 2 * a.D;
    const long e = 4 * (static_cast<long>(blockIdx.x) * AT + threadIdx.x);
    if (e >= n) return;
    f32x4 s = f32x4{};
    for (int i = 0; i < b.parts; ++i) s += *reinterpret_cast<const f32x4*>(b.part + i * n + e);
    const long r = e / (2 * a.D);
    int d = static_cast<int>(e - r * 2 * a.D);
    const long kvh = r / a.m.Tk, key = r - kvh * a.m.Tk;
    if (d < a.D) {
        store4(static_cast<T*>(b.dK) + kvh * b.dk_hs + key * b.dk_rs + d, b.D_out - d, b.vec_dk, s[0] * a.scale, s[1] * a.scale,
               s[2] * a.scale, s[3] * a.scale);
    } else {
        d -= a.D;
        store4(static_cast<T*>(b.dV) + kvh * b.dv_hs + key * b.dv_rs + d, b.D_out - d, b.vec_dv, s[0], s[1], s[2], s[3]);
    }
}

struct Launch {
    template <class T, int DP, int CAP, bool BIAS>
    static int run(kdec_ctx* ctx, const Bwd& b, int shared, long q_blocks, long k_blocks, size_t part_n) {
        const auto blocks = [](long n) { return dim3(static_cast<unsigned>(n)); };
        if (b.a.m.Tq > 0) {
            if (shared == 2) hipLaunchKernelGGL((attn_dq_k<T, DP, CAP, BIAS, 2>), blocks(q_blocks), dim3(AT), 0, ctx->stream, b);
            else hipLaunchKernelGGL((attn_dq_k<T, DP, CAP, BIAS, 1>), blocks(q_blocks), dim3(AT), 0, ctx->stream, b);
        }
        if (b.a.m.Tk > 0) {
            constexpr int KG = key_groups<T, DP, BIAS>();
            hipLaunchKernelGGL((attn_dkv_k<T, DP, CAP, BIAS>), dim3(static_cast<unsigned>(k_blocks), static_cast<unsigned>(b.parts)),
                               dim3(128 * KG), 0, ctx->stream, b);
            if (b.parts > 1)
                hipLaunchKernelGGL(attn_dkv_join_k<T>, blocks(cdiv(part_n / 4, AT)), dim3(AT), 0, ctx->stream, b);
        }
        return launch_check(ctx, "kdec_attn_bwd");
    }
};

}  // namespace
}  // namespace attn
}  // namespace kdec

using namespace kdec;
using namespace kdec::attn;

extern "C" int kdec_attn_bwd(kdec_ctx* ctx, int dtype, const void* Q, long q_rs, long q_hs, const void* K, long k_rs,
                             long k_hs, const void* V, long v_rs, long v_hs, const void* O, long o_rs, long o_hs,
                             const float* lse, const void* dO, long do_rs, long do_hs, const int* q_off, const int* k_off,
                             const int* k_len, const int* prefix, int docs, int causal, const float* slopes, float scale,
                             float cap, int Tq, int Tk, int Hq, int Hkv, int D, void* dQ, long dq_rs, long dq_hs, void* dK,
                             long dk_rs, long dk_hs, void* dV, long dv_rs, long dv_hs) {
    if (!ctx) return KDEC_EINVAL;
    if (int rc = check(ctx, "kdec_attn_bwd", dtype, q_off, k_off, docs, scale, cap, Tq, Tk, Hq, Hkv, D)) return rc;
    KDEC_CHECK(ctx, (Tq == 0 || (Q && O && lse && dO && dQ)) && (Tk == 0 || (K && V && dK && dV)),
               "kdec_attn_bwd: null tensor");
    KDEC_CHECK(ctx, apart(dq_rs, dq_hs, Tq, Hq, D) && apart(dk_rs, dk_hs, Tk, Hkv, D) && apart(dv_rs, dv_hs, Tk, Hkv, D),
               "kdec_attn_bwd: rows of a gradient overlap");
    if (Tq == 0 && Tk == 0) return KDEC_OK;
    const size_t size = dtype == KDEC_F32 ? 4 : 2;
    const int G = Hq / Hkv;
    ProfScope ps(ctx, "attn", 0.0, 0.0);
    Bwd b{};
    b.a = Args{{Q, q_rs, q_hs}, {K, k_rs, k_hs}, {V, v_rs, v_hs}, {q_off, k_off, k_len, prefix, docs, causal != 0, Tq, Tk},
               slopes, scale, cap, Hq, Hkv, G, D, Tq * G, false};
    b.O = Heads{O, o_rs, o_hs};
    b.dO = Heads{dO, do_rs, do_hs};
    b.vec_o = plain(b.O, D, size);
    std::unique_ptr<Workspace> packed[4];
    if (!plain(b.a.Q, D, size) || !plain(b.a.K, D, size) || !plain(b.a.V, D, size) || !plain(b.dO, D, size)) {
        if (int rc = pack(ctx, dtype, b.a.Q, Tq, Hq, D, packed[0])) return rc;
        if (int rc = pack(ctx, dtype, b.a.K, Tk, Hkv, D, packed[1])) return rc;
        if (int rc = pack(ctx, dtype, b.a.V, Tk, Hkv, D, packed[2])) return rc;
        if (int rc = pack(ctx, dtype, b.dO, Tq, Hq, D, packed[3])) return rc;
        b.a.D = (D + 7) & ~7;
    }
    b.lse = lse;
    b.D_out = D;
    b.dQ = dQ;
    b.dK = dK;
    b.dV = dV;
    b.dq_rs = dq_rs;
    b.dq_hs = dq_hs;
    b.dk_rs = dk_rs;
    b.dk_hs = dk_hs;
    b.dv_rs = dv_rs;
    b.dv_hs = dv_hs;
    b.vec_dq = D % 4 == 0 && aligned(Heads{dQ, dq_rs, dq_hs}, size, 4 * size);
    b.vec_dk = D % 4 == 0 && aligned(Heads{dK, dk_rs, dk_hs}, size, 4 * size);
    b.vec_dv = D % 4 == 0 && aligned(Heads{dV, dv_rs, dv_hs}, size, 4 * size);
    const size_t stat_bytes = (static_cast<size_t>(Tq) * Hq * sizeof(float2) + 255) & ~size_t(255);
    const int keys = D <= 64 || dtype == KDEC_F32 || slopes ? 64 : 128;  // of a block
    b.by_doc_k = by_document(ctx, docs, Tk, Hkv, keys);
    const int shared = waves_shared(ctx, cdiv(b.a.E, BM) * Hkv), held = BM / shared;
    b.a.by_doc = rows_by_document(ctx, docs, Tk, b.a.E, Hkv, held);
    const long q_blocks = doc_blocks(b.a.by_doc, docs, b.a.E, held) * Hkv, k_blocks = doc_blocks(b.by_doc_k, docs, Tk, keys) * Hkv;
    KDEC_CHECK(ctx, k_blocks < INT_MAX, "kdec_attn_bwd: too many keys");
    // Key tiles too few to fill the device (causal walks differ in length, so
    // two blocks per CU) share their rows among parts of no fewer than four
    // turns of 128 rows.
    const long turns = docs > 0 ? cdiv(Tq / docs, 128) * G : 1;
    long parts = k_blocks > 0 ? cdiv(2L * ctx->num_cus, k_blocks) : 1;
    if (parts > turns / 4) parts = turns / 4;
    if (parts < 1) parts = 1;
    b.parts = static_cast<int>(parts);
    const size_t row_bytes = (static_cast<size_t>(Tq) * sizeof(Row) + 255) & ~size_t(255);
    const size_t part_n = parts > 1 ? static_cast<size_t>(Hkv) * Tk * 2 * b.a.D : 0;
    Workspace ws(ctx, stat_bytes + row_bytes + parts * part_n * sizeof(float));
    if (!ws.p) return KDEC_ENOMEM;
    b.stat = ws.as<float2>();
    b.rows = reinterpret_cast<Row*>(ws.as<char>() + stat_bytes);
    b.part = reinterpret_cast<float*>(ws.as<char>() + stat_bytes + row_bytes);
    return dispatch<Launch>(dtype, D, cap, slopes != nullptr, ctx, b, shared, q_blocks, k_blocks, part_n);
}
