// Attention over a cache of 8-bit codes on gfx950.
//
// A key's score is its scale times q . codes, a value enters the output with
// its scale in its probability: o = sum_j (p_j vs_j) codes_j / sum_j p_j. The
// codes themselves are exact in bf16, so the products are bf16 ones. Float tensors
// enter them as three bf16 terms, which hold their 24 bits, and p vs as three as
// well. For bf16 tensors p vs enters as two, which leave 2^-16 of it at most: o is
// off by its own rounding alone (relative error 0.0017, as the formula's in float
// sums rounded once; one term made it 0.0023), whatever else a call holds. Where
// memory bounds a call the second term costs nothing (one token for 48 requests 26.8
// us, with one 26.6), where the vector unit does a seventh (5 documents of 200 rows
// 70 us for 62).
//
// A block holds 16 or 32 entries (rows of one document times the heads that share
// a key head) and its four waves take tiles of 32 keys in turn, each with a
// softmax state of its own, joined at the end; long caches are split over blocks
// as well and joined by a second launch. Codes go from memory into the products'
// registers, the next tile's on their way. Depth slots and output rows stand for
// whatever bytes a lane has: of a key 16 bytes in each 64, the query's fragments
// following, and of a value ND neighbouring columns, so that row m of the
// output's block dt is column ND m + dt and no byte moves between lanes.
//
// Steps are bound by memory: one token for 48 requests over up to 4096 keys, 16
// heads on 4 of width 128, 28 us for 106 MB (3.9 TB/s) and 4 for the join. Pieces of
// 90 to 301 rows with a cap (80 to 95 us by their lengths; the products, the values'
// twice, would take 28) are bound by the vector unit: codes to floats, exponentials
// of cap and softmax, the probabilities' terms.
#include "kdec_attn.hpp"

namespace kdec {
namespace attn {
namespace {

constexpr int CN = 32;  // keys of a wave's tile
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

struct Cached {
    Args a;  // K, V: bytes
    const float *ks, *vs;
    void* O;
    long o_rs, o_hs;
    bool vec_o, vec_q;
    float* lse;
    int rows, pieces;  // rows of a block; blocks that the heads of a row take (where a block holds fewer)
    int splits;
    float *part_o, *part_ml;  // (splits, Hkv, E, DP) and (splits, Hkv, E, 2)
};

// Bytes i and j of two registers, signed numbers, as two bf16: a float of at most
// eight bits is its upper half.
__device__ inline unsigned codes2(unsigned x, int i, unsigned y, int j) {
    const auto one = [](unsigned v, int b) { return __float_as_uint(static_cast<float>(static_cast<int>(v << (24 - 8 * b)) >> 24)); };
    return __builtin_amdgcn_perm(one(y, j), one(x, i), 0x07060302);
}

__device__ inline f32x4 mma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// The larger of the values of the four lanes that share a column.
__device__ inline float max_column(float x) {
    const unsigned u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    const unsigned lo = r[0], hi = r[1];
    return max32(fmaxf(__uint_as_float(lo), __uint_as_float(hi)));
}

// The document that holds a row, the same in all lanes, or -1.
__device__ inline int doc_holding(const Docs& m, int row) {
    const int lane = threadIdx.x & 63;
    if (m.docs <= 0) return -1;
    const int d0 = m.docs > 64 ? max(doc_of(m.q_off, m.docs, row), 0) : 0;
    const int off = d0 + lane <= m.docs ? m.q_off[d0 + lane] : INT_MAX;
    const int d = d0 + __builtin_popcountll(__builtin_amdgcn_ballot_w64(off <= row)) - 1;
    return __builtin_amdgcn_readfirstlane(d >= 0 && d < m.docs && row < m.q_off[d + 1] ? d : -1);
}

// A stretch of a block's rows that one document holds (or none), from row0 on.
struct Segment {
    Doc doc;
    int causal, stop;  // the row behind it
    __device__ inline int position(int row) const { return row - doc.q0 + doc.lk - doc.lq; }
    // Keys that a row sees, from the slot's first: more of them from row to row.
    __device__ inline int sees(int row) const {
        return causal ? min(max(max(position(row) + 1, doc.prefix), 0), doc.lk) : doc.lk;
    }
};
// The rows of a block: `rows` from a multiple of it (doc: -2), or as many of one
// document (or of the rows before the first or past the last, -1 and docs), found
// by a scan over the documents' numbers of blocks.
__device__ inline bool block_rows(const Cached& p, int b, int& row0, int& end, int& doc) {
    const Docs& m = p.a.m;
    doc = -2;
    row0 = b * p.rows;
    end = min(row0 + p.rows, m.Tq);
    if (!p.a.by_doc) return true;
    Piece piece;
    if (!piece_at(m.q_off, m.docs, m.Tq, 1, p.rows, b, piece)) return false;
    doc = piece.doc;
    row0 = piece.lo + piece.place * p.rows;
    end = min(row0 + p.rows, piece.hi);
    return true;
}
// A part's tiles: of every document an equal share. (Parts of a fixed length, the
// same work for short and long documents, were slower: one token for 48 requests
// over 90 to 4096 keys 31 us for 26, since fewer of them run at once.)
__device__ inline void part_tiles(const Cached& p, int tiles, int& t0, int& t1) {
    t0 = static_cast<int>(static_cast<long>(tiles) * blockIdx.y / p.splits);
    t1 = static_cast<int>(static_cast<long>(tiles) * (blockIdx.y + 1) / p.splits);
}
__device__ inline Segment segment_at(const Docs& m, int row0, int end, int doc) {
    Segment s{Doc{0, 0, 0, 0, 0}, m.causal, end};
    const int d = doc == -2 ? doc_holding(m, row0) : doc;
    if (d >= 0 && d < m.docs) {
        s.doc = doc_at(m, d);
        if (doc == -2) s.stop = min(m.q_off[d + 1], end);
    } else if (doc == -2 && m.docs > 0 && row0 < m.q_off[0]) {
        s.stop = min(m.q_off[0], end);
    }
    s.stop = __builtin_amdgcn_readfirstlane(max(s.stop, row0 + 1));
    return s;
}

__device__ inline void empty_part(const Cached& p, int kvh, int e) {
    const long to = (static_cast<long>(blockIdx.y) * p.a.Hkv + kvh) * p.a.E + e;
    p.part_ml[2 * to] = -INF;
    p.part_ml[2 * to + 1] = 0.0f;
}

// One step of the running softmax of a lane's column over the scores of 32 keys
// from j0, `at` the lane's first: s become probabilities, acc is rescaled when
// the column's maximum moves far enough: m in the units of raw products without cap
// and bias, in log2 units with either.
struct Soft {
    float m = -INF, l = 0.0f;
};
template <bool MASKED, class T, int CAP, bool BIAS, int ND>
__device__ inline void cache_soft(const Score<T, CAP, BIAS>& rule, int pos, unsigned seen, int at, f32x4 (&s)[2], f32x4 (&acc)[ND], Soft& st) {
    constexpr bool RAW = !CAP && !BIAS;
    const float unit = RAW ? rule.unit : 1.0f, dist = static_cast<float>(pos - at);
    float mx = -INF;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float t = s[b][r], dt;
            if (!RAW) t = rule.of(t, dist - static_cast<float>(16 * b + r), dt);
            if (MASKED) t = static_cast<unsigned>(at + 16 * b + r) < seen ? t : -INF;
            s[b][r] = t;
            mx = fmaxf(mx, t);
        }
    mx = max_column(mx);
    // each column by its own maximum: its sums do not depend on its neighbours'
    const bool moves = (mx - st.m) * unit > 8.0f || (st.m == -INF && mx > -INF);
    if (__builtin_amdgcn_ballot_w64(moves)) {
        const float m = moves ? mx : st.m, f = __builtin_amdgcn_exp2f((st.m - (m == -INF ? 0.0f : m)) * unit);
        st.l *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] *= f;
        st.m = m;
        asm volatile("");  // a branch
    }
    const float m0 = (st.m == -INF ? 0.0f : st.m) * unit;
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float p = __builtin_amdgcn_exp2f(RAW ? __builtin_fmaf(s[b][r], unit, -m0) : s[b][r] - m0);
            s[b][r] = p;
            st.l += p;
        }
}

// CB: blocks of 16 entries that a wave holds.
template <class T, int DP, int CAP, bool BIAS, int CB>
__global__ __launch_bounds__(AT, sizeof(T) == 2 ? (CB == 1 ? 3 : 2) : 1) void attn_cache_k(Cached p) {
    constexpr int NC = DP / 32, NK = DP / 64, ND = DP / 16, TERMS = sizeof(T) == 2 ? 1 : 3, WTERMS = sizeof(T) == 2 ? 2 : 3, PITCH = DP + 4, COLS = 16 * CB;
    __shared__ __align__(16) float so[4][COLS][PITCH];
    __shared__ __align__(16) float scales[4][2][CN];
    __shared__ float sml[4][2][COLS];
    const Args& a = p.a;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, col = lane & 15, quarter = lane >> 4;
    int b = blockIdx.x;
    const int kvh = b % a.Hkv;
    b /= a.Hkv;
    const int piece = b % p.pieces, split = blockIdx.y, W = code_width(a.D);
    int row0, end, doc;
    if (!block_rows(p, b / p.pieces, row0, end, doc)) return;
    const signed char* kb = static_cast<const signed char*>(a.K.p) + kvh * a.K.hs;
    const signed char* vb = static_cast<const signed char*>(a.V.p) + kvh * a.V.hs;
    const float* ks = p.ks + static_cast<long>(kvh) * a.m.Tk;
    const float* vs = p.vs + static_cast<long>(kvh) * a.m.Tk;
    int k_at[NK], v_at[4];
#pragma unroll
    for (int i = 0; i < NK; ++i) k_at[i] = 64 * i + 16 * quarter < W ? static_cast<int>(col * a.K.rs) + 64 * i + 16 * quarter : kFar;
#pragma unroll
    for (int r = 0; r < 4; ++r) v_at[r] = ND * col < W ? static_cast<int>((4 * quarter + r) * a.V.rs) + ND * col : kFar;

    // the documents that the block's rows belong to, one after the other
    while (row0 < end) {
        const Segment sg = segment_at(a.m, row0, end, doc);
        const int e0 = row0 * a.G + COLS * piece, e1 = min(sg.stop * a.G, p.pieces > 1 ? min(e0 + COLS, (row0 + 1) * a.G) : INT_MAX);
        const int k0 = sg.doc.k0, all = sg.sees(row0), keys = sg.sees((e1 - 1) / a.G);
        const int tiles = (keys + CN - 1) / CN;
        int t0, t1;
        part_tiles(p, tiles, t0, t1);
        if (split > 0 && t0 == t1) {  // nothing of this document's
            if (tid < min(e1 - e0, COLS)) empty_part(p, kvh, e0 + tid);
            row0 = sg.stop;
            continue;
        }
        int pos[CB];
        unsigned seen[CB];
        float slope[CB];
#pragma unroll
        for (int x = 0; x < CB; ++x) {
            const int e = e0 + 16 * x + col, row = e < e1 ? e / a.G : row0;
            pos[x] = sg.position(row);
            seen[x] = e < e1 ? static_cast<unsigned>(sg.sees(row)) : 0u;
            slope[x] = BIAS && e < e1 ? a.slopes[kvh * a.G + e - row * a.G] : 0.0f;
        }
        Score<T, CAP, BIAS> rule(a);

        // Loads past the part's last tile find empty descriptors: without a branch
        // around them the products wait for their own operand's loads alone.
        u32x4 kr[2][NK];
        float kscale, vscale;
        const auto load_k = [&](int t) __attribute__((always_inline)) {
            const long j = k0 + static_cast<long>(t) * CN;
            const int n = t < t1 ? min(keys - t * CN, CN) : 0;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const __amdgpu_buffer_rsrc_t r = rows_rsrc(kb + (j + 16 * g) * a.K.rs, a.K.rs, n - 16 * g, W);
#pragma unroll
                for (int i = 0; i < NK; ++i)
                    kr[g][i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, k_at[i], 0, 0));
            }
            const __amdgpu_buffer_rsrc_t kr_ = rows_rsrc(ks + j, 1, n, 1), vr_ = rows_rsrc(vs + j, 1, n, 1);
            kscale = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(kr_, 4 * (lane & 31), 0, 0));
            vscale = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(vr_, 4 * (lane & 31), 0, 0));
        };
        unsigned vr[8][ND / 4];  // ND columns of key 16 g + 4 quarter + r at 4 g + r
        const auto load_v = [&](int t) __attribute__((always_inline)) {
            const long j = k0 + static_cast<long>(t) * CN;
            const int n = t < t1 ? min(keys - t * CN, CN) : 0;
#pragma unroll
            for (int g = 0; g < 2; ++g) {
                const __amdgpu_buffer_rsrc_t s = rows_rsrc(vb + (j + 16 * g) * a.V.rs, a.V.rs, n - 16 * g, W);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if constexpr (ND == 8) {
                        const u32x2 w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(s, v_at[r], 0, 0));
                        vr[4 * g + r][0] = w[0];
                        vr[4 * g + r][1] = w[1];
                    } else {
                        vr[4 * g + r][0] = __builtin_amdgcn_raw_buffer_load_b32(s, v_at[r], 0, 0);
                    }
                }
            }
        };
        f32x4 acc[CB][ND];
        Soft st[CB];
#pragma unroll
        for (int x = 0; x < CB; ++x)
#pragma unroll
            for (int i = 0; i < ND; ++i) acc[x][i] = f32x4{};
        bf16x8 q[CB][NC][TERMS];
        const auto step = [&](auto masked, int t) __attribute__((always_inline)) {
            constexpr bool MASKED = decltype(masked)::value;
            // an infinite scale as NaN: its scores could be minus infinity, or a cap's end
            const float scale = lane >> 5 ? vscale : kscale;
            scales[wave][lane >> 5][lane & 31] = __builtin_fmaf(scale, 0.0f, scale);
            f32x4 s[CB][2];
#pragma unroll
            for (int g = 0; g < 2; ++g) {
#pragma unroll
                for (int x = 0; x < CB; ++x) s[x][g] = f32x4{};
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    u32x4 w;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const unsigned u = kr[g][c >> 1][2 * (c & 1) + (i >> 1)];
                        w[i] = codes2(u, 2 * (i & 1), u, 2 * (i & 1) + 1);
                    }
                    const bf16x8 k = __builtin_bit_cast(bf16x8, w);
#pragma unroll
                    for (int x = 0; x < CB; ++x)
#pragma unroll
                        for (int m = 0; m < TERMS; ++m) s[x][g] = mma16(k, q[x][c][m], s[x][g]);
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            load_k(t + 4);
            f32x4 f[2];
#pragma unroll
            for (int g = 0; g < 2; ++g) f[g] = *reinterpret_cast<const f32x4*>(&scales[wave][0][16 * g + 4 * quarter]);
            const int at = t * CN + 4 * quarter;
#pragma unroll
            for (int x = 0; x < CB; ++x) {
#pragma unroll
                for (int g = 0; g < 2; ++g) s[x][g] *= f[g];
                rule.slope = slope[x] * LOG2E;
                cache_soft<MASKED>(rule, pos[x], seen[x], at, s[x], acc[x], st[x]);
            }
#pragma unroll
            for (int g = 0; g < 2; ++g) f[g] = *reinterpret_cast<const f32x4*>(&scales[wave][1][16 * g + 4 * quarter]);
#pragma unroll
            for (int x = 0; x < CB; ++x)
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    s[x][g] *= f[g];
                    if (MASKED)  // a value that the row does not see stays out whatever its scale
#pragma unroll
                        for (int r = 0; r < 4; ++r) s[x][g][r] = static_cast<unsigned>(at + 16 * g + r) < seen[x] ? s[x][g][r] : 0.0f;
                }
            __builtin_amdgcn_sched_barrier(0);  // the values' floats come after the scores'
            bf16x8 w[CB][WTERMS];
#pragma unroll
            for (int x = 0; x < CB; ++x) {
                const Terms<bf16, WTERMS> terms(__builtin_shufflevector(s[x][0], s[x][1], 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                for (int m = 0; m < WTERMS; ++m) w[x][m] = terms.t[m];
            }
#pragma unroll
            for (int i = 0; i < ND; ++i) {
                u32x4 u;
#pragma unroll
                for (int j = 0; j < 4; ++j) u[j] = codes2(vr[2 * j][i >> 2], i & 3, vr[2 * j + 1][i >> 2], i & 3);
                const bf16x8 v = __builtin_bit_cast(bf16x8, u);
#pragma unroll
                for (int x = 0; x < CB; ++x)
#pragma unroll
                    for (int m = 0; m < WTERMS; ++m) acc[x][i] = mma16(v, w[x][m], acc[x][i]);
            }
            load_v(t + 4);
        };
        load_k(t0 + wave);
        load_v(t0 + wave);
#pragma unroll
        for (int x = 0; x < CB; ++x) {
            const int e = e0 + 16 * x + col, row = e < e1 ? e / a.G : row0, head = e < e1 ? kvh * a.G + e - row * a.G : 0;
            const T* qp = static_cast<const T*>(a.Q.p) + row * a.Q.rs + head * a.Q.hs;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int at = 64 * (c >> 1) + 16 * quarter + 8 * (c & 1);
                const Frag<T> f = load8(qp + at, e < e1 ? max(min(8, a.D - at), 0) : 0, p.vec_q);
                if constexpr (TERMS == 1) {
                    q[x][c][0] = f;
                    asm volatile("" : "+v"(q[x][c][0]));  // here, not behind the loop's loads
                } else {
                    const Terms<bf16, TERMS> t(f);
#pragma unroll
                    for (int m = 0; m < TERMS; ++m) q[x][c][m] = t.t[m];
                }
            }
        }
        // tiles that every row sees whole, then the others
        const int whole = min(all / CN, t1);
        int t = t0 + wave;
        for (; t < whole; t += 4) step(std::false_type{}, t);
        for (; t < t1; t += 4) step(std::true_type{}, t);

        // join the waves: their states' common maximum, then the sums in order
        // (the thread's number anew, so that no address of this is held above)
        int thread = tid;
        asm volatile("" : "+v"(thread));
        const int c1 = thread & 15, q1 = thread >> 4 & 3;
        const float unit = CAP || BIAS ? 1.0f : rule.unit;
#pragma unroll
        for (int x = 0; x < CB; ++x) {
            float l = st[x].l, zero = 0.0f;
#pragma unroll
            for (int i = 0; i < ND; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) zero = __builtin_fmaf(acc[x][i][r], 0.0f, zero);
            l += zero == 0.0f ? 0.0f : __builtin_nanf("");  // a value that is not finite makes the whole row NaN
            l += __shfl_xor(l, 16);
            l += __shfl_xor(l, 32);
            if (q1 == 0) {
                sml[wave][0][16 * x + c1] = st[x].m * unit;
                sml[wave][1][16 * x + c1] = l;
            }
            if (e0 + 16 * x + c1 < e1)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int i = 0; i < ND; i += 4)
                        *reinterpret_cast<f32x4*>(&so[wave][16 * x + c1][ND * (4 * q1 + r) + i]) =
                            f32x4{acc[x][i][r], acc[x][i + 1][r], acc[x][i + 2][r], acc[x][i + 3][r]};
        }
        __syncthreads();
        const int n = max(min(e1 - e0, COLS), 0);
        for (int i = thread; i < n * (DP / 4); i += AT) {
            const int cc = i / (DP / 4), d4 = 4 * (i - cc * (DP / 4));
            float m = -INF, l = 0.0f;
#pragma unroll
            for (int w = 0; w < 4; ++w) m = fmaxf(m, sml[w][0][cc]);
            f32x4 v = f32x4{};
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                const float f = __builtin_amdgcn_exp2f(sml[w][0][cc] - (m == -INF ? 0.0f : m));
                l += sml[w][1][cc] * f;
                v += *reinterpret_cast<const f32x4*>(&so[w][cc][d4]) * f;
            }
            const int at = e0 + cc, r = at / a.G, h = kvh * a.G + at - r * a.G;
            if (p.splits > 1) {
                const long to = (static_cast<long>(split) * a.Hkv + kvh) * a.E + at;
                *reinterpret_cast<f32x4*>(p.part_o + to * DP + d4) = v;
                if (d4 == 0) {
                    p.part_ml[2 * to] = m;
                    p.part_ml[2 * to + 1] = l;
                }
            } else {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                store4(static_cast<T*>(p.O) + r * p.o_rs + h * p.o_hs + d4, a.D - d4, p.vec_o, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                if (d4 == 0) p.lse[static_cast<long>(h) * a.m.Tq + r] = l == 0.0f ? -INF : m * LN2 + logf(l);
            }
        }
        __syncthreads();
        row0 = sg.stop;
    }
}

// Joins the splits of an entry (at most 64): one wave per entry, a lane for
// every split's state, then lanes over the output, the splits in order.
template <class T, int DP>
__global__ __launch_bounds__(64) void attn_cache_join_k(Cached p) {
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
    float o[DP / 64];
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) o[i] = 0.0f;
    for (int s = 0; s < p.splits; s += 8) {  // eight loads in flight
        float v[8][DP / 64];
#pragma unroll
        for (int x = 0; x < 8; ++x)
#pragma unroll
            for (int i = 0; i < DP / 64; ++i)  // parts of no weight hold nothing
                v[x][i] = __builtin_amdgcn_readlane(__float_as_int(f), s + x) ? p.part_o[((s + x) * n + w) * DP + lane + 64 * i] : 0.0f;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            const float g = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(f), s + x));
#pragma unroll
            for (int i = 0; i < DP / 64; ++i) o[i] = __builtin_fmaf(g, v[x][i], o[i]);
        }
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T* out = static_cast<T*>(p.O) + row * p.o_rs + head * p.o_hs;
#pragma unroll
    for (int i = 0; i < DP / 64; ++i) {
        const int d = lane + 64 * i;
        if (d < a.D) out[d] = static_cast<T>(o[i] * inv);
    }
    if (lane == 0) p.lse[static_cast<long>(head) * a.m.Tq + row] = l == 0.0f ? -INF : top * LN2 + logf(l);
}

struct Launch {
    template <class T, int DP, int CAP, bool BIAS>
    static int run(kdec_ctx* ctx, const Cached& p, dim3 grid, int cols) {
        if (cols == 16) hipLaunchKernelGGL((attn_cache_k<T, DP, CAP, BIAS, 1>), grid, dim3(AT), 0, ctx->stream, p);
        else hipLaunchKernelGGL((attn_cache_k<T, DP, CAP, BIAS, 2>), grid, dim3(AT), 0, ctx->stream, p);
        if (p.splits > 1)
            hipLaunchKernelGGL((attn_cache_join_k<T, DP>), dim3(static_cast<unsigned>(static_cast<long>(p.a.Hkv) * p.a.E)), dim3(64), 0,
                               ctx->stream, p);
        return launch_check(ctx, "kdec_attn_cache_fwd");
    }
};

}  // namespace
}  // namespace attn
}  // namespace kdec

using namespace kdec;
using namespace kdec::attn;

extern "C" int kdec_attn_cache_fwd(kdec_ctx* ctx, int dtype, const void* Q, long q_rs, long q_hs, const void* Kc, long kc_rs, long kc_hs,
                                   const void* Vc, long vc_rs, long vc_hs, const float* k_scale, const float* v_scale, const int* q_off,
                                   const int* k_off, const int* k_len, const int* prefix, int docs, int causal, const float* slopes,
                                   float scale, float cap, int Tq, int Tk, int Hq, int Hkv, int D, void* O, long o_rs, long o_hs,
                                   float* lse) {
    if (!ctx) return KDEC_EINVAL;
    const DeviceScope device(ctx);
    const char* who = "kdec_attn_cache_fwd";
    if (int rc = check(ctx, who, dtype, q_off, k_off, docs, scale, cap, Tq, Tk, Hq, Hkv, D)) return rc;
    const Heads k{Kc, kc_rs, kc_hs}, v{Vc, vc_rs, vc_hs};
    if (int rc = check_codes(ctx, who, k, v, k_scale, v_scale, Tk, Hkv, D)) return rc;
    if (Tq == 0) return KDEC_OK;
    KDEC_CHECK(ctx, Q && O && lse, "kdec_attn_cache_fwd: null tensor");
    KDEC_CHECK(ctx, apart(o_rs, o_hs, Tq, Hq, D), "kdec_attn_cache_fwd: rows of O overlap");
    const size_t size = dtype == KDEC_F32 ? 4 : 2;
    const int G = Hq / Hkv, DP = D <= 64 ? 64 : 128;
    ProfScope ps(ctx, "attn", 0.0, 0.0);
    Cached p{};
    p.a = Args{{Q, q_rs, q_hs}, k, v, {q_off, k_off, k_len, prefix, docs, causal != 0, Tq, Tk}, slopes, scale, cap, Hq, Hkv, G, D, Tq * G, false};
    p.ks = k_scale;
    p.vs = v_scale;
    p.O = O;
    p.o_rs = o_rs;
    p.o_hs = o_hs;
    p.vec_o = D % 4 == 0 && aligned(Heads{O, o_rs, o_hs}, size, 4 * size);
    p.vec_q = D % 8 == 0 && aligned(p.a.Q, size, 16);
    p.lse = lse;
    // Entries of a block: 16 where a document's rows have no more, else 32 that
    // share a code's way to a float (bf16, 16 heads on 4 of width 128, blocks of 16
    // and 32: 48 documents of 90 to 4096 keys and 1 row 32 us and 45, 16 of 2000 to
    // 4096 and 4 rows 22.8 and 23.6, 8 rows 30 and 27, 5 of them and 200 rows 83 and
    // 70; rows that leave blocks of 32 part empty cost that again, 20 of 1000 to 2000
    // keys and 10 to 40 rows 36 and 43). Rows: what these hold, fewer where documents
    // have fewer.
    const long mean = docs > 0 ? cdiv(Tq, docs) : Tq;
    const int cols = mean * G <= 16 ? 16 : 32;
    p.pieces = static_cast<int>(cdiv(G, cols));
    p.rows = static_cast<int>(G >= cols ? 1 : mean < cols / G ? mean : cols / G);
    // Blocks that end with their document where rows may not be even, as far as
    // finding them is quick: one that holds rows of two walks twice (48 documents of
    // up to 4096 keys, 1 to 4 rows 51 us for 63, 2 to 9 rows 62 for 79, 5 of 100 to
    // 300 rows 91 for 102; even ones of 4 rows 24.6 for 22.5).
    p.a.by_doc = p.rows > 1 && docs > 0 && docs < 127 && (Tq % docs != 0 || mean % p.rows != 0);
    const long units = cdiv(Tq, p.rows) * p.pieces * Hkv, blocks = doc_blocks(p.a.by_doc, docs, Tq, p.rows) * p.pieces * Hkv;
    KDEC_CHECK(ctx, grid_holds(blocks, AT) && static_cast<long>(Hkv) * p.a.E < INT_MAX, "kdec_attn_cache_fwd: too many rows");
    // Split the keys where the rows alone do not fill the device, as far as all
    // parts' blocks are on it at once (48 documents of 90 to 4096 keys and 1 row: 4
    // parts, which fill it, 26 us, 3 and 6 parts 31 and 32), to no fewer than 256
    // keys a part (one float row over 6000 keys, 12 heads of width 64: 15.9 us with
    // the join, of 128 keys 16.8). The device is not filled evenly where the parts do
    // not divide it (32 heads on 8, 90 to 4096 keys, 1, 2 and 3 parts: 24 requests 41
    // us, 44 and 39 and by the rule, of 4, 35; 32 46, 51 and 51 by the rule; 48 73, 64
    // by the rule and 63), and past half of it one part is the rule's (50 requests 73,
    // 68, 64; 64 83, 78, 77; 96 116, 112, 112).
    const long each = docs > 0 ? Tk / docs : 0, held = (dtype == KDEC_F32 ? (cols == 16 ? 2L : 1L) : cols == 16 ? 3L : 2L) * ctx->num_cus;
    long splits = held / units;
    if (splits > each / 256) splits = each / 256;
    if (splits > 64) splits = 64;  // what the join holds
    if (splits < 1) splits = 1;
    p.splits = static_cast<int>(splits);
    const size_t n = splits > 1 ? static_cast<size_t>(splits) * Hkv * p.a.E : 0;
    Workspace ws(ctx, n * (DP + 2) * sizeof(float));
    if (!ws.p) return KDEC_ENOMEM;
    p.part_o = ws.as<float>();
    p.part_ml = p.part_o + n * DP;
    return dispatch<Launch>(dtype, D, cap, slopes != nullptr, ctx, p, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(splits)),
                            cols);
}
