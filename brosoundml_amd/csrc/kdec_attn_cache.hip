// Attention over a cache of 8-bit codes on gfx950.
//
// A key's score is its scale times q . codes, a value enters the output with
// its scale in its probability: o = sum_j (p_j vs_j) codes_j / sum_j p_j. The
// codes themselves are exact in bf16, so the products are bf16 ones whose only
// roundings are those of p vs (bf16 tensors); float tensors enter as three bf16
// terms, which hold their 24 bits.
//
// A block holds 32 entries (rows of one document times the heads that share a
// key head) and its four waves take tiles of 32 keys in turn, each with a
// softmax state of its own, joined at the end; long caches are split over
// blocks as well and joined by a second launch. Codes go from memory into the
// products' registers, the next tile's on their way: a lane holds a key's half
// row (depth slots stand for the lane's own bytes, the query's fragments
// follow), and of the values ND neighbouring columns at a time, so that row m of
// the output's block dt is column ND m + dt and no byte moves between lanes.
#include "kdec_attn.hpp"

namespace kdec {
namespace attn {
namespace {

constexpr int CN = 32;  // keys of a wave's tile, entries of a block

struct Cached {
    Args a;  // K, V: bytes
    const float *ks, *vs;
    void* O;
    long o_rs, o_hs;
    bool vec_o, vec_q;
    float* lse;
    int rows, pieces;  // rows of a block; blocks that the heads of a row take (more than 32 of them)
    int splits;
    float *part_o, *part_ml;  // (splits, Hkv, E, DP) and (splits, Hkv, E, 2)
};

// Four signed bytes of each of two registers as bf16, exact.
__device__ inline bf16 code(unsigned x, int i) {
    return static_cast<bf16>(static_cast<float>(static_cast<signed char>(x >> (8 * i))));
}

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
template <int DP>
struct Keys {
    static constexpr int N = DP / 32;
    u32x4 k[N];   // the lane's key: bytes DP / 2 * half ..
    float scale;  // lanes below 32: the key's, above: the value's
};
struct Values {
    unsigned v[16];  // columns ND * (lane % 32) .. of the keys 8 (i / 4) + 4 half + i % 4
};

template <class T, int DP, int CAP, bool BIAS>
__global__ __launch_bounds__(AT, sizeof(T) == 2 ? 2 : 1) void attn_cache_k(Cached p) {
    constexpr int NC = DP / 16, ND = DP / 32, TERMS = sizeof(T) == 2 ? 1 : 3, PITCH = DP + 4;
    __shared__ __align__(16) float so[4][CN][PITCH];
    __shared__ __align__(16) float scales[4][2][CN];
    __shared__ float sml[4][2][CN];
    const Args& a = p.a;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, half = lane >> 5, col = lane & 31;
    int b = blockIdx.x;
    const int kvh = b % a.Hkv;
    b /= a.Hkv;
    const int piece = b % p.pieces, split = blockIdx.y, W = code_width(a.D);
    int row0 = b / p.pieces * p.rows;
    const int end = min(row0 + p.rows, a.m.Tq);
    const signed char* kb = static_cast<const signed char*>(a.K.p) + kvh * a.K.hs;
    const signed char* vb = static_cast<const signed char*>(a.V.p) + kvh * a.V.hs;
    const float* ks = p.ks + static_cast<long>(kvh) * a.m.Tk;
    const float* vs = p.vs + static_cast<long>(kvh) * a.m.Tk;
    int k_at[Keys<DP>::N], v_at[4];
#pragma unroll
    for (int i = 0; i < Keys<DP>::N; ++i) {
        const int byte = DP / 2 * half + 16 * i;
        k_at[i] = byte < W ? static_cast<int>(col * a.K.rs) + byte : kFar;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v_at[j] = ND * col < W ? static_cast<int>((4 * half + j) * a.V.rs) + ND * col : kFar;

    // the documents that the block's rows belong to, one after the other
    while (row0 < end) {
        const int doc = __builtin_amdgcn_readfirstlane(doc_of_row(a.m.q_off, a.m.docs, row0, row0));
        int stop = end;  // of this document's rows, or of rows that belong to none
        if (doc >= 0) {
            stop = min(a.m.q_off[doc + 1], end);
        } else if (a.m.docs > 0 && row0 < a.m.q_off[0]) {
            stop = min(a.m.q_off[0], end);
        }
        stop = __builtin_amdgcn_readfirstlane(max(stop, row0 + 1));
        const int e0 = row0 * a.G + CN * piece, e1 = min(stop * a.G, p.pieces > 1 ? min(e0 + CN, (row0 + 1) * a.G) : INT_MAX);
        const int e = e0 + col;
        const bool valid = e < e1;
        const int row = valid ? e / a.G : row0, head = kvh * a.G + (valid ? e - row * a.G : 0);
        Row me{INT_MAX, INT_MIN, 0};
        if (doc >= 0) me = row_in(a.m, doc, row);
        if (!valid) me = Row{INT_MAX, INT_MIN, 0};
        // keys that any of the rows sees, and that all of them see
        int lo = me.lo, hi = me.hi, all_lo = valid ? me.lo : INT_MIN, all_hi = valid ? me.hi : INT_MAX;
        for (int o = 16; o; o >>= 1) {
            lo = min(lo, __shfl_xor(lo, o));
            hi = max(hi, __shfl_xor(hi, o));
            all_lo = max(all_lo, __shfl_xor(all_lo, o));
            all_hi = min(all_hi, __shfl_xor(all_hi, o));
        }
        lo = __builtin_amdgcn_readfirstlane(lo);
        hi = __builtin_amdgcn_readfirstlane(hi);
        all_lo = __builtin_amdgcn_readfirstlane(all_lo);
        all_hi = __builtin_amdgcn_readfirstlane(all_hi);
        const int tiles = hi > lo ? (hi - lo + CN - 1) / CN : 0;
        const int t0 = static_cast<int>(static_cast<long>(tiles) * split / p.splits);
        const int t1 = static_cast<int>(static_cast<long>(tiles) * (split + 1) / p.splits);

        const Score<T, CAP, BIAS> rule(a, head);
        bf16x8 q[NC][TERMS];
        const T* qp = static_cast<const T*>(a.Q.p) + row * a.Q.rs + head * a.Q.hs;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = DP / 2 * half + 8 * c;
            const Frag<T> f = load8(qp + d, valid ? max(min(8, a.D - d), 0) : 0, p.vec_q);
            if constexpr (TERMS == 1) {
                q[c][0] = f;
            } else {
                const Terms<bf16, TERMS> t(f);
#pragma unroll
                for (int k = 0; k < TERMS; ++k) q[c][k] = t.t[k];
            }
        }
        Keys<DP> x;
        const auto load_k = [&](int t) __attribute__((always_inline)) {
            const int j = lo + t * CN, n = min(hi - j, CN);
            const __amdgpu_buffer_rsrc_t kr = rows_rsrc(kb + j * a.K.rs, a.K.rs, n, W);
#pragma unroll
            for (int i = 0; i < Keys<DP>::N; ++i)
                x.k[i] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(kr, k_at[i], 0, 0));
            x.scale = col < n ? (half ? vs : ks)[j + col] : 0.0f;
        };
        Values y;
        const auto load_v = [&](int t) __attribute__((always_inline)) {
            const int j = lo + t * CN, n = min(hi - j, CN);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const __amdgpu_buffer_rsrc_t vr = rows_rsrc(vb + (j + 8 * g) * a.V.rs, a.V.rs, n - 8 * g, W);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (DP == 128) y.v[4 * g + i] = __builtin_amdgcn_raw_buffer_load_b32(vr, v_at[i], 0, 0);
                    else y.v[4 * g + i] = __builtin_amdgcn_raw_buffer_load_b16(vr, v_at[i], 0, 0);
                }
            }
        };
        f32x16 acc[ND];
#pragma unroll
        for (int d = 0; d < ND; ++d) acc[d] = f32x16{};
        Soft st;
        const auto step = [&](int t) __attribute__((always_inline)) {
            const int j0 = lo + t * CN;
            const bool whole = j0 >= all_lo && j0 + CN <= all_hi;
            scales[wave][half][col] = x.scale;
            f32x16 s[1];
            s[0] = f32x16{};
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                bf16x8 k;
#pragma unroll
                for (int i = 0; i < 8; ++i) k[i] = code(x.k[c >> 1][2 * (c & 1) + (i >> 2)], i & 3);
#pragma unroll
                for (int m = 0; m < TERMS; ++m) s[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k, q[c][m], s[0], 0, 0, 0);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (t + 4 < t1) load_k(t + 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const f32x4 f = *reinterpret_cast<const f32x4*>(&scales[wave][0][8 * i + 4 * half]);
#pragma unroll
                for (int r = 0; r < 4; ++r) s[0][4 * i + r] *= f[r];
            }
            soft_step<true>(rule, me, whole, j0, half, s, acc, st);
            f32x4 f[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = *reinterpret_cast<const f32x4*>(&scales[wave][1][8 * i + 4 * half]);
            if (whole) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[0][r] *= f[r >> 2][r & 3];
            } else {  // a value that the row does not see stays out whatever its scale
                const unsigned at = static_cast<unsigned>(j0 + 4 * half - me.lo), len = me.hi > me.lo ? static_cast<unsigned>(me.hi - me.lo) : 0u;
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[0][r] = at + static_cast<unsigned>(acc_row(r, 0)) < len ? s[0][r] * f[r >> 2][r & 3] : 0.0f;
            }
            __builtin_amdgcn_sched_barrier(0);  // the values' floats come after the scores'
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const Terms<bf16, TERMS> w(acc_floats(s[0], c));
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    bf16x8 v;
#pragma unroll
                    for (int i = 0; i < 8; ++i) v[i] = code(y.v[8 * c + i], d);
#pragma unroll
                    for (int m = 0; m < TERMS; ++m) acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(v, w.t[m], acc[d], 0, 0, 0);
                }
            }
            if (t + 4 < t1) load_v(t + 4);
        };
        if (t0 + wave < t1) {
            load_k(t0 + wave);
            load_v(t0 + wave);
        }
        for (int t = t0 + wave; t < t1; t += 4) step(t);
        // join the waves: their states' common maximum, then the sums in order
        // (the thread's number anew, so that no address of this is held above)
        int thread = tid;
        asm volatile("" : "+v"(thread));
        const int c1 = thread & 31, h1 = thread >> 5 & 1;
        const float unit = CAP || BIAS ? 1.0f : rule.unit;
        float l = st.l + __shfl_xor(st.l, 32);
        if (sums_not_finite(acc)) l = __builtin_nanf("");
        if (!h1) {
            sml[wave][0][c1] = st.m * unit;
            sml[wave][1][c1] = l;
        }
        __syncthreads();
        const float m = fmaxf(fmaxf(sml[0][0][c1], sml[1][0][c1]), fmaxf(sml[2][0][c1], sml[3][0][c1]));
        const float m0 = m == -INF ? 0.0f : m, f = __builtin_amdgcn_exp2f(st.m * unit - m0);
        if (e0 + c1 < e1)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float* to = &so[wave][c1][ND * acc_row(r, h1)];
#pragma unroll
                for (int d = 0; d < ND; ++d) to[d] = acc[d][r] * f;
            }
        __syncthreads();
        const int n = max(min(e1 - e0, CN), 0);
        for (int i = thread; i < n * (DP / 4); i += AT) {
            const int cc = i / (DP / 4), d = 4 * (i - cc * (DP / 4));
            float mm = -INF, ll = 0.0f;
            for (int w = 0; w < 4; ++w) mm = fmaxf(mm, sml[w][0][cc]);
            for (int w = 0; w < 4; ++w) ll += sml[w][1][cc] * __builtin_amdgcn_exp2f(sml[w][0][cc] - (mm == -INF ? 0.0f : mm));
            f32x4 v = f32x4{};
            for (int w = 0; w < 4; ++w) v += *reinterpret_cast<const f32x4*>(&so[w][cc][d]);
            const int at = e0 + cc, r = at / a.G, h = kvh * a.G + at - r * a.G;
            if (p.splits > 1) {
                const long to = (static_cast<long>(split) * a.Hkv + kvh) * a.E + at;
                *reinterpret_cast<f32x4*>(p.part_o + to * DP + d) = v;
                if (d == 0) {
                    p.part_ml[2 * to] = mm;
                    p.part_ml[2 * to + 1] = ll;
                }
            } else {
                const float inv = ll == 0.0f ? 0.0f : 1.0f / ll;
                store4(static_cast<T*>(p.O) + r * p.o_rs + h * p.o_hs + d, a.D - d, p.vec_o, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                if (d == 0) p.lse[static_cast<long>(h) * a.m.Tq + r] = ll == 0.0f ? -INF : mm * LN2 + logf(ll);
            }
        }
        __syncthreads();
        row0 = stop;
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
            for (int i = 0; i < DP / 64; ++i) v[x][i] = s + x < p.splits ? p.part_o[((s + x) * n + w) * DP + lane + 64 * i] : 0.0f;
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            const float g = __shfl(f, s + x);
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
    static int run(kdec_ctx* ctx, const Cached& p, dim3 grid) {
        hipLaunchKernelGGL((attn_cache_k<T, DP, CAP, BIAS>), grid, dim3(AT), 0, ctx->stream, p);
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
    p.pieces = static_cast<int>(cdiv(G, CN));
    // Rows of a block: what 32 entries hold, fewer where documents have fewer.
    const long mean = docs > 0 ? cdiv(Tq, docs) : Tq;
    p.rows = static_cast<int>(G >= CN ? 1 : mean < CN / G ? mean : CN / G);
    const long blocks = cdiv(Tq, p.rows) * p.pieces * Hkv;
    KDEC_CHECK(ctx, blocks < INT_MAX && static_cast<long>(Hkv) * p.a.E < INT_MAX, "kdec_attn_cache_fwd: too many rows");
    // Split the keys where the rows alone do not fill the device.
    const long each = docs > 0 ? Tk / docs : 0;
    long splits = cdiv(4L * ctx->num_cus, blocks);
    if (splits > each / 256) splits = each / 256;
    if (splits > 64) splits = 64;  // what the join holds
    if (splits < 1) splits = 1;
    p.splits = static_cast<int>(splits);
    const size_t n = splits > 1 ? static_cast<size_t>(splits) * Hkv * p.a.E : 0;
    Workspace ws(ctx, n * (DP + 2) * sizeof(float));
    if (!ws.p) return KDEC_ENOMEM;
    p.part_o = ws.as<float>();
    p.part_ml = p.part_o + n * DP;
    return dispatch<Launch>(dtype, D, cap, slopes != nullptr, ctx, p, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(splits)));
}
