// What the attention kernels of both directions share: the documents, the
// score's formula, and the checks and layouts of their arguments.
#pragma once

#include <climits>
#include <cmath>
#include <cstdlib>
#include <memory>
#include <type_traits>

#include "kdec_frag.hpp"
#include "kdec_internal.hpp"

namespace kdec {
namespace attn {

constexpr int AT = 256;  // threads of a block
constexpr int BM = 128;  // entries or keys that a block holds, 32 per wave
constexpr int BN = 64;   // keys or rows of a tile that it walks
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr float INF = __builtin_inff();

// Keeps the operand reads of later products behind this one: a float product
// takes eight matrix instructions, which cover the next read, and its operands
// twice the registers, which more reads ahead would not leave.
template <class T>
__device__ inline void hold() {
    if (sizeof(T) == 4) __builtin_amdgcn_sched_barrier(0);
}

struct Docs {
    const int *q_off, *k_off, *k_len, *prefix;
    int docs, causal, Tq, Tk;
};

struct Heads {  // a (rows, heads, D) tensor
    const void* p;
    long rs, hs;
};

struct Args {
    Heads Q, K, V;
    Docs m;
    const float* slopes;
    float scale, cap;
    int Hq, Hkv, G, D, E;  // G = Hq / Hkv, E = Tq * G entries per key head
    bool by_doc;           // blocks of entries end with their document
};

// Bytes that a token takes in one head of a cache of 8-bit codes.
__host__ __device__ constexpr int code_width(int D) { return (D + 15) & ~15; }

struct Row {
    int lo, hi, pos;  // keys [lo, hi), the key row at the row's own position
};

// The last document whose offset is not past i, or -1.
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

__device__ inline Row row_in(const Docs& m, int d, int i) {
    const Doc c = doc_at(m, d);
    const int p = i - c.q0 + c.lk - c.lq;  // position of its last key
    const int n = m.causal ? min(max(max(p + 1, c.prefix), 0), c.lk) : c.lk;
    if (n <= 0) return Row{INT_MAX, INT_MIN, 0};
    return Row{c.k0, c.k0 + n, c.k0 + p};
}

// The document of every lane's row i, or -1; `first` is the least of the wave's
// rows (all lanes take part). The wave reads 64 offsets at once, from the
// document of its first row, and each lane finds its own among them; only rows
// past 64 documents (most of them empty, then) search memory.
__device__ inline int doc_of_row(const int* q_off, int docs, int i, int first) {
    const int lane = threadIdx.x & 63;
    if (docs <= 0) return -1;
    int d0 = 0;
    if (docs > 64) d0 = max(doc_of(q_off, docs, __builtin_amdgcn_readfirstlane(first)), 0);
    const int off = d0 + lane <= docs ? q_off[d0 + lane] : INT_MAX;
    int n = 0;  // how many of the 64 are not past i
#pragma unroll
    for (int s = 32; s; s >>= 1) n += __shfl(off, n + s - 1) <= i ? s : 0;
    n += __shfl(off, min(n, 63)) <= i;
    int d = d0 + n - 1;
    if (n == 64) d = doc_of(q_off, docs, i);
    return d < 0 || d >= docs || i >= q_off[d + 1] ? -1 : d;
}

// The keys of every lane's row i, `first` the least of the wave's rows.
__device__ inline Row row_at(const Docs& m, int i, int first) {
    const int d = doc_of_row(m.q_off, m.docs, i, first);
    return d < 0 ? Row{INT_MAX, INT_MIN, 0} : row_in(m, d, i);
}

// Blocks that end with their document. Documents, and the rows before the
// first and past the last as two more, are cut into blocks of `size`; a row
// counts `each` times. Every lane takes one document's number of blocks, a
// scan over the wave finds block b's: rows [lo, hi) of document doc (-1 and
// docs are the two others), whose block `place` it is. False past the last.
struct Piece {
    int doc, lo, hi, place;
};
__device__ inline bool piece_at(const int* off, int docs, int rows, int each, int size, int b, Piece& p) {
    const int lane = threadIdx.x & 63;
    const auto at = [&](int d) { return d < 0 ? 0 : docs > 0 && d <= docs ? min(max(off[d], 0), rows) : rows; };
    int before = 0;
    for (int base = -1; base <= docs; base += 64) {
        const int lo = at(base + lane), hi = at(base + lane + 1);
        const int n = hi > lo ? ((hi - lo) * each + size - 1) / size : 0;
        const int sum = wave_scan(n);
        const int all = __builtin_amdgcn_readlane(sum, 63);
        if (b - before < all) {
            const int l = __builtin_popcountll(__builtin_amdgcn_ballot_w64(before + sum <= b));
            if (l > 63) return false;
            p.doc = base + l;
            p.lo = __builtin_amdgcn_readlane(lo, l);
            p.hi = __builtin_amdgcn_readlane(hi, l);
            p.place = b - before - __builtin_amdgcn_readlane(sum - n, l);
            return p.place >= 0 && p.place < __builtin_amdgcn_readlane(n, l);
        }
        before += all;
    }
    return false;
}

// A lane's entry: row * G + head of the group. `again` hides that the second
// call gives what the first gave, so that a kernel's end forms it anew and its
// loops need not hold it.
struct Entry {
    int e, row, head, half;
    bool valid;
};
__device__ inline Entry entry_of(const Args& a, int kvh, int first, int end, bool again) {
    Entry r;
    int lane = threadIdx.x & 63, G = a.G;
    if (again) {
        unsigned ones = ~0u;
        asm volatile("" : "+s"(ones), "+s"(G));
        lane = __builtin_amdgcn_mbcnt_hi(ones, __builtin_amdgcn_mbcnt_lo(ones, 0));
    }
    r.half = lane >> 5;
    r.e = first + (lane & 31);
    r.valid = r.e < end;
    r.row = r.valid ? r.e / G : 0;
    r.head = kvh * G + (r.valid ? r.e - r.row * G : 0);
    return r;
}

// Block `tile`'s entries of a key head, `size` of them at most: its group's
// 32 from e0, the end of those there are, and the document that holds them all
// (by_doc).
struct Span {
    int e0, end, doc;
};
__device__ inline bool span_at(const Args& a, int size, int tile, int group, Span& s) {
    if (!a.by_doc) {
        s = Span{tile * size + group * 32, a.E, 0};
        return true;
    }
    Piece p;
    if (!piece_at(a.m.q_off, a.m.docs, a.m.Tq, a.G, size, tile, p)) return false;
    s = Span{p.lo * a.G + p.place * size + group * 32, p.hi * a.G, p.doc};
    return true;
}
__device__ inline Row row_of(const Args& a, const Span& s, const Entry& e) {
    Row r{INT_MAX, INT_MIN, 0};
    if (!a.by_doc) r = row_at(a.m, e.row, min(s.e0, a.E - 1) / a.G);
    else if (s.doc >= 0 && s.doc < a.m.docs) r = row_in(a.m, s.doc, e.row);
    return e.valid ? r : Row{INT_MAX, INT_MIN, 0};
}

// The larger of a value and that of the lane 32 away.
__device__ inline float max32(float x) {
    const unsigned u = __float_as_uint(x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const unsigned lo = r[0], hi = r[1];
    return fmaxf(__uint_as_float(lo), __uint_as_float(hi));
}

// Whether one of a column's sums is not finite, in either lane half: they are
// times zero added to one register, which costs one instruction a sum and no
// registers at the kernels' ends.
template <int ND>
__device__ inline bool sums_not_finite(const f32x16 (&acc)[ND]) {
    float zero = 0.0f;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) zero = __builtin_fmaf(acc[d][r], 0.0f, zero);
    return !(zero + __shfl_xor(zero, 32) == 0.0f);
}

// What a block of 128 entries (32 per wave) walks: keys [lo, hi) in tiles of
// 64, of which those in [full_lo, full_hi) are seen by every row; a wave's
// rows see keys of [wlo, whi), and all of them those of [wfull_lo, wfull_hi).
struct Walk {
    int lo, hi, full_lo, full_hi, wlo, whi, wfull_lo, wfull_hi;
};
__device__ inline Walk walk_of(const Row& me, bool valid, int (&red)[4][4]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
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
    __syncthreads();
    const auto u = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    return Walk{u(min(min(red[0][0], red[1][0]), min(red[2][0], red[3][0]))),
                u(max(max(red[0][1], red[1][1]), max(red[2][1], red[3][1]))),
                u(max(max(red[0][2], red[1][2]), max(red[2][2], red[3][2]))),
                u(min(min(red[0][3], red[1][3]), min(red[2][3], red[3][3]))),
                u(lo), u(hi), u(full_lo), u(full_hi)};
}
// Whether [lo, hi) holds a marked key of the 64 at j0.
__device__ inline bool sees_bad(int lo, int hi, int j0, unsigned long long bad) {
    const int a = min(max(lo - j0, 0), 64), b = min(max(hi - j0, 0), 64);
    if (b <= a) return false;
    const unsigned long long upto = b == 64 ? ~0ull : (1ull << b) - 1;
    return (upto & ~((1ull << a) - 1) & bad) != 0;
}

// Tiles [t0, f0) and [f1, t1) of a walk are masked, those between are seen
// whole by every row; the first two numbers of tiles are even, so that each
// loop starts at the first buffer.
__device__ inline void split_walk(const Walk& w, int t0, int t1, int& f0, int& f1) {
    f0 = f1 = t0;
    if (w.full_hi > w.full_lo && w.full_lo <= w.hi) {
        f0 = min(max((w.full_lo - w.lo + BN - 1) / BN, t0), t1);
        f0 = min(f0 + ((f0 - t0) & 1), t1);
        f1 = min(max((w.full_hi - w.lo) / BN, f0), t1);
        f1 -= (f1 - f0) & 1;
    }
    if (f0 >= f1) f0 = f1 = t0;
}

// Scores in log2 units from raw products. CAP is how the cap's tanh is formed:
// 1 - 2 / (1 + e^2x) is off by 2^-23 absolutely, and the score by cap times
// that; up to caps of NEAR_CAP that is 2^-17, which a bf16 probability cannot
// show. Beyond, and for float, the odd series takes over near zero (its next
// term, 62/2835 x^9, is below 2^-25 of x up to 0.15), which takes a fifth
// longer (4 causal texts of 3000 rows, 16 heads on 4 of width 128, bf16, cap
// 100: forward 230 -> 278 us, backward 854 -> 1005).
enum Cap { NO_CAP, QUICK_CAP, FINE_CAP };
constexpr float NEAR_CAP = 64.0f;
template <class T, int CAP, bool BIAS>
struct Score {
    float unit;   // product to log2 units
    float k, c2;  // cap: tanh's argument is s k / (2 log2 e), the score c2 tanh
    float slope;  // bias per step of distance, log2 units
    __device__ inline explicit Score(const Args& a) {  // without a head's slope
        unit = a.scale * LOG2E;
        k = CAP ? 2.0f * LOG2E * a.scale / a.cap : 0.0f;
        c2 = a.cap * LOG2E;
        slope = 0.0f;
    }
    __device__ inline Score(const Args& a, int head) : Score(a) { slope = BIAS ? a.slopes[head] * LOG2E : 0.0f; }
    __device__ inline float tanh_(float s) const {
        const float x2 = s * k;
        float th = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x2)), 1.0f);
        if (CAP == FINE_CAP) {
            const float x = x2 * (0.5f / LOG2E), q = x * x;
            const float near = x * (1.0f + q * (-1.0f / 3 + q * (2.0f / 15 + q * (-17.0f / 315))));
            th = __builtin_fabsf(x) < 0.15f ? near : th;
        }
        return th;
    }
    // dist = position - key, dt: the score's derivative by scale * product
    __device__ inline float of(float s, float dist, float& dt) const {
        float t;
        dt = 1.0f;
        if (CAP) {
            const float th = tanh_(s);
            dt = __builtin_fmaf(-th, th, 1.0f);
            t = c2 * th;
            if (BIAS) t = __builtin_fmaf(-slope, __builtin_fabsf(dist), t);
        } else {
            t = s * unit;
            if (BIAS) t = __builtin_fmaf(s, unit, -slope * __builtin_fabsf(dist));
        }
        return t;
    }
};

// A probability formed again from a raw product and the row's lse in log2
// units; dt is the score's derivative by scale * product.
template <class T, int CAP, bool BIAS>
__device__ inline float grad_p(const Score<T, CAP, BIAS>& rule, float s, float dist, float lse2, float& dt) {
    if (!CAP && !BIAS) {
        dt = 1.0f;
        return __builtin_amdgcn_exp2f(__builtin_fmaf(s, rule.unit, -lse2));
    }
    return __builtin_amdgcn_exp2f(rule.of(s, dist, dt) - lse2);
}

// ─── host ───

// Whether blocks of `size` entries (or keys) end with their document. Else
// blocks of several documents leave fewer waves without rows, though a block
// then walks the keys of all of them, the most of which a wave does not see.
// Documents of half a block or more gain from it (8192 rows, 12 heads of width
// 64, bf16, forward and backward together: documents of about 1024 rows 311 ->
// 197 us, 256 132 -> 98, 64 91 -> 89, but 32 89 -> 119), as long as two turns
// of the scan find them (900 documents of 100 rows: 817 -> 1154). So do
// shorter ones where blocks of several would not fill the device, since a
// block walks one document's keys then (54 documents of 3 rows over 120 keys, 12
// heads of width 128: forward 83 -> 22 us, backward 136 -> 71; 48 of 4 rows over
// 2000, 16 heads on 4: backward 566 -> 379).
inline bool by_document(kdec_ctx* ctx, int docs, long entries, int heads, int size) {
    return docs < 127 && (docs * static_cast<long>(size / 2) <= entries || cdiv(entries, size) * heads < ctx->num_cus);
}
// The same for blocks of rows, which walk keys: past two turns of the scan they
// end with their document as well where a document's walk is long against the
// scan. A turn takes about as long as half a tile of 64 keys, and blocks of
// several documents walk as many tiles in all, but on B of the 2 num_cus places
// that the others fill: (keys / 64 + docs / 128) B < keys / 64 * 2 num_cus.
// (Causal forward, bf16, 16 heads on 4 of width 128, of several documents and of
// one: 128 requests of 2 rows over 1000 keys 87 and 48 us, 200 of 4 126 and 89,
// 256 of 2 over 200 52 and 35, 512 of 8 over 300 75 and 98, 512 of 2 over 60 25
// and 48; 12 heads of width 64: 200 of 2 over 1000 220 and 117, 1000 of 2 over
// 200 162 and 216.)
inline bool rows_by_document(kdec_ctx* ctx, int docs, long keys, long entries, int heads, int size) {
    if (docs < 127) return by_document(ctx, docs, entries, heads, size);
    const long each = keys / docs, all = 2L * ctx->num_cus, blocks = cdiv(entries, size) * heads;
    return (2 * each + docs) * (blocks < all ? blocks : all) < 2 * each * all;
}
inline long doc_blocks(bool by_doc, int docs, long entries, int size) { return cdiv(entries, size) + (by_doc ? docs + 2 : 0); }

// Waves of a block that share 32 entries: one where blocks of 128 entries fill
// the device, else two, each with half of every tile's keys. Then twice as
// many blocks walk half as long (7 documents of up to 333 rows, 8 heads of
// width 64, float with a bias: forward 33 -> 23 us, dQ 43 -> 29; 2 of 1000
// rows, 16 heads on 4 of width 128, bf16: forward 51 -> 32). Filled, two lose
// the join's time and half of a tile's use (2 of 2000 rows: 78 -> 99).
inline int waves_shared(kdec_ctx* ctx, long blocks) { return blocks < ctx->num_cus ? 2 : 1; }

// Kernels of a call by its type, width and score: L::run<T, DP, CAP, BIAS>.
template <class L, class T, int DP, int CAP, class... P>
int by_bias(bool bias, P&&... p) {
    return bias ? L::template run<T, DP, CAP, true>(p...) : L::template run<T, DP, CAP, false>(p...);
}
template <class L, class T, int DP, class... P>
int by_score(float cap, bool bias, P&&... p) {
    if (cap > 0.0f && sizeof(T) == 2 && cap <= NEAR_CAP) return by_bias<L, T, DP, sizeof(T) == 2 ? QUICK_CAP : FINE_CAP>(bias, p...);
    return cap > 0.0f ? by_bias<L, T, DP, FINE_CAP>(bias, p...) : by_bias<L, T, DP, NO_CAP>(bias, p...);
}
template <class L, class... P>
int dispatch(int dtype, int D, float cap, bool bias, P&&... p) {
    if (dtype == KDEC_F32) return D <= 64 ? by_score<L, float, 64>(cap, bias, p...) : by_score<L, float, 128>(cap, bias, p...);
    return D <= 64 ? by_score<L, bf16, 64>(cap, bias, p...) : by_score<L, bf16, 128>(cap, bias, p...);
}

inline int check(kdec_ctx* ctx, const char* who, int dtype, const void* q_off, const void* k_off, int docs, float scale,
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

// Whether an output's rows and heads can lie apart (none repeated, no steps
// shorter than a row).
inline bool apart(long rs, long hs, long rows, int heads, int D) {
    return (rows <= 1 || std::labs(rs) >= D) && (heads == 1 || std::labs(hs) >= D);
}

// Whether a tensor's rows and heads start on multiples of `to` bytes.
inline bool aligned(const Heads& h, size_t size, size_t to) {
    return reinterpret_cast<size_t>(h.p) % to == 0 && (h.rs * size) % to == 0 && (h.hs * size) % to == 0;
}
// A cache of 8-bit codes: its tensors have to be what the kernels' loads take
// (16 bytes of a row at once, a tile's offsets below 2^30).
inline int check_codes(kdec_ctx* ctx, const char* who, const Heads& k, const Heads& v, const float* ks, const float* vs, int Tk, int H,
                       int D) {
    const auto bad = [&](const char* why) { return fail(ctx, KDEC_EINVAL, std::string(who) + ": " + why); };
    if (Tk > 0 && !(k.p && v.p && ks && vs)) return bad("null cache");
    for (const Heads* h : {&k, &v}) {
        if (!aligned(*h, 1, 16)) return bad("the cache's rows and heads must start on multiples of 16 bytes");
        if (h->rs < 0 || h->rs >= (1L << 24) || h->hs < 0) return bad("the cache's strides are outside what the kernels take");
    }
    return KDEC_OK;
}
// Whether the kernels' loads take a tensor as it stands: 16 bytes at a time,
// a tile's offsets below 2^30 bytes.
inline bool plain(const Heads& h, int D, size_t size) {
    return D % 8 == 0 && aligned(h, size, 16) && (BM * h.rs + D) * static_cast<long>(size) < (1L << 30) && h.rs >= 0;
}

// Copies a tensor that they do not take into aligned rows, padded to a
// multiple of 8 columns. The kernels then run on the copy with D8 columns.
template <class T>
__global__ __launch_bounds__(AT) void pack_k(Heads h, T* out, long n, int heads, int D, int D8) {
    for (long e = static_cast<long>(blockIdx.x) * AT + threadIdx.x; e < n; e += static_cast<long>(gridDim.x) * AT) {
        const long r = e / D8;
        const int d = static_cast<int>(e - r * D8);
        const long row = r / heads;
        out[e] = d < D ? static_cast<const T*>(h.p)[row * h.rs + (r - row * heads) * h.hs + d] : static_cast<T>(0.0f);
    }
}
inline int pack(kdec_ctx* ctx, int dtype, Heads& h, int rows, int heads, int D, std::unique_ptr<Workspace>& ws) {
    const int D8 = (D + 7) & ~7;
    const long n = static_cast<long>(rows) * heads * D8;
    if (n == 0) return KDEC_OK;
    ws = std::make_unique<Workspace>(ctx, n * (dtype == KDEC_F32 ? 4 : 2));
    if (!ws->p) return KDEC_ENOMEM;
    const long blocks = cdiv(n, AT) < 16L * ctx->num_cus ? cdiv(n, AT) : 16L * ctx->num_cus;
    if (dtype == KDEC_F32)
        hipLaunchKernelGGL(pack_k<float>, dim3(static_cast<unsigned>(blocks)), dim3(AT), 0, ctx->stream, h, ws->as<float>(), n, heads,
                           D, D8);
    else
        hipLaunchKernelGGL(pack_k<bf16>, dim3(static_cast<unsigned>(blocks)), dim3(AT), 0, ctx->stream, h, ws->as<bf16>(), n, heads, D,
                           D8);
    h = Heads{ws->p, static_cast<long>(heads) * D8, D8};
    return KDEC_OK;
}

}  // namespace attn
}  // namespace kdec
