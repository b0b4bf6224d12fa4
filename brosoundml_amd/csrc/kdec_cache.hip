// A key and value cache in 8 bits on gfx950: written as its tokens come, read
// back as floats. The attention over it is kdec_attn_cache.hip.
//
// A token's values in one head share a scale, s = max(max |x| / 127, 2^-126) in
// float, and are held as the integers nearest to x / s, ties to the even one,
// decided exactly: the codes are those of the definition on every machine. A
// token with a value that is not finite gets the scale NaN and codes of zero.
//
// 8 or 16 lanes take the values of a token in a head, eight each; bound by
// memory, or for single tokens by the launch and three dependent loads. 32 texts
// of 77 to 1000 tokens, 12 heads of width 64, bf16: written in 23 us for 87 MB (3.7
// TB/s), read back in 17 (5.1), float 39 and 27 for 144 MB; 48 single tokens of 4
// heads of width 128, bf16, in 5.1 and 3.9.
#include "kdec_attn.hpp"

namespace kdec {
namespace {

using attn::Docs;
using attn::Heads;

constexpr int CT = 256;
typedef signed char i8x8 __attribute__((ext_vector_type(8)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

struct Codes {
    signed char *k, *v;
    long k_rs, k_hs, v_rs, v_hs;  // bytes
    float *ks, *vs;               // (heads, rows)
};

// The cache row of query row i, or -1: the document's last row is its last
// filled key.
__device__ inline long cache_row(const Docs& m, int i, int first) {
    const int d = attn::doc_of_row(m.q_off, m.docs, min(i, m.Tq - 1), first);
    if (d < 0 || i >= m.Tq) return -1;
    const attn::Doc c = attn::doc_at(m, d);
    const int p = i - c.q0 + c.lk - c.lq;
    return p < 0 ? -1 : static_cast<long>(c.k0) + p;
}

// The largest magnitude of eight values as the bits of a float; more than
// infinity's where one of them is NaN.
__device__ inline unsigned top8(bf16x8 f) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    const u32x4 b = __builtin_bit_cast(u32x4, f) & 0x7FFF7FFFu;
    u16x2 m = __builtin_bit_cast(u16x2, static_cast<unsigned>(b[0]));
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, static_cast<unsigned>(b[i])));
    return static_cast<unsigned>(max(m[0], m[1])) << 16;
}
__device__ inline unsigned top8(f32x8 f) {
    unsigned m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(f[i]) & 0x7FFFFFFFu);
    return m;
}
// The largest over L neighbouring lanes, in all of them.
template <int L>
__device__ inline unsigned top_lanes(unsigned x) {
    const auto with = [&](auto ctrl) __attribute__((always_inline)) {
        x = max(x, static_cast<unsigned>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), decltype(ctrl)::value, 15, 15, true)));
    };
    with(std::integral_constant<int, 0xB1>{});   // the lane beside
    with(std::integral_constant<int, 0x4E>{});   // the pair beside
    with(std::integral_constant<int, 0x141>{});  // the four of eight opposite
    if (L == 16) with(std::integral_constant<int, 0x140>{});  // the eight of sixteen opposite
    return x;
}

// max |x| / 127 to the nearest float: the product with 1 / 127 and one correction
// by its exact remainder (127 and the rounded 1 / 127 meet the conditions under
// which that is the quotient). Quotients below 2^-126, of a top below 2^-119, make
// the scale 2^-126 whatever their last bit; just above, the remainder is subnormal (a
// top near 2^-119 leaves about 2^-143), which these kernels' floats keep.
__device__ inline float scale_of(float top) {
    const float c = 1.0f / 127.0f, q = top * c;
    return fmaxf(__builtin_fmaf(__builtin_fmaf(-q, 127.0f, top), c, q), 0x1p-126f);
}

// Eight values' codes under scale s, as bytes. x / s by the reciprocal is off by
// 2^-22 of it, so that its nearest integer q (the low bits of 1.5 2^23 + q) is
// the quotient's own, but next to a half: the remainder x - q s is exact, and
// tells by being half of s or more.
__device__ inline u32x2 nearest8(const f32x8& x, float s) {
    const float inv = __builtin_amdgcn_rcpf(s), magic = 0x1.8p23f;
    float t[8], most = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        t[i] = __builtin_fmaf(x[i], inv, magic);
        most = fmaxf(most, __builtin_fabsf(__builtin_fmaf(magic - t[i], s, x[i])));
    }
    if (__builtin_amdgcn_ballot_w64(2.0f * most >= s)) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float r = __builtin_fmaf(magic - t[i], s, x[i]), r2 = 2.0f * __builtin_fabsf(r);
            if (r2 > s || (r2 == s && (__float_as_uint(t[i]) & 1))) t[i] += r > 0.0f ? 1.0f : -1.0f;
        }
    }
    u32x2 c;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        c[i] = __builtin_amdgcn_perm(__float_as_uint(t[4 * i + 1]), __float_as_uint(t[4 * i]), 0x0c0c0400) |
               __builtin_amdgcn_perm(__float_as_uint(t[4 * i + 3]), __float_as_uint(t[4 * i + 2]), 0x04000c0c);
    return c;
}

// L lanes take UNITS heads' keys or values of a row (unit u: head u / 2, keys or
// values), their loads together, on their way during the search for the row's
// place. More units a thread leave fewer waves, fewer a search for each (17000
// rows of 12 heads of width 64, bf16, written and read back: 2 units 25.8 and 20.7
// us, 4 24.2 and 16.9, 8 23.5 and 17.7; 48 rows of 4 heads of width 128: 4.4 and
// 3.6, 5.0 and 3.9, 6.6 and 4.6).
constexpr int UNITS = 4;
template <class T, int L>
__global__ __launch_bounds__(CT) void cache_write_k(Docs m, Heads K, Heads V, Codes o, int H, int D, int W, bool vec) {
    const int per = CT / L, lane = threadIdx.x % L, row = blockIdx.x * per + threadIdx.x / L;
    const int c = 8 * lane, n = max(min(8, D - c), 0), u0 = blockIdx.y * UNITS;
    Frag<T> f[UNITS];
#pragma unroll
    for (int j = 0; j < UNITS; ++j) {
        const Heads& h = (u0 + j) & 1 ? V : K;
        const T* p = static_cast<const T*>(h.p) + min(row, m.Tq - 1) * h.rs + min((u0 + j) >> 1, H - 1) * h.hs + c;
        f[j] = load8(p, n, vec);
    }
    const long at = cache_row(m, row, __builtin_amdgcn_readfirstlane(row));
    signed char* to[2] = {o.k + at * o.k_rs + c, o.v + at * o.v_rs + c};
    float* scales[2] = {o.ks + at, o.vs + at};
#pragma unroll
    for (int j = 0; j < UNITS; ++j) {
        const bool keys = !((u0 + j) & 1);
        const int head = (u0 + j) >> 1;
        const unsigned top = top_lanes<L>(top8(f[j]));
        if (at < 0 || head >= H) continue;
        const bool bad = top >= 0x7F800000u;
        const float s = bad ? __builtin_nanf("") : scale_of(__uint_as_float(top));
        f32x8 x;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(f[j][i]);
        u32x2 q = nearest8(x, s);
        if (bad) q = u32x2{};
        if (c < W) *reinterpret_cast<u32x2*>((keys ? to[0] : to[1]) + head * (keys ? o.k_hs : o.v_hs)) = q;
        if (lane == 0) (keys ? scales[0] : scales[1])[static_cast<long>(head) * m.Tk] = s;
    }
}

template <class T, int L>
__global__ __launch_bounds__(CT) void cache_read_k(Docs m, Codes o, int H, int D, int W, T* K, long k_rs, long k_hs, T* V, long v_rs,
                                                   long v_hs, bool vec) {
    const int per = CT / L, lane = threadIdx.x % L, row = blockIdx.x * per + threadIdx.x / L;
    const int c = 8 * lane, n = max(min(8, D - c), 0), u0 = blockIdx.y * UNITS;
    const long at = cache_row(m, row, __builtin_amdgcn_readfirstlane(row));
    if (row >= m.Tq) return;
    i8x8 q[UNITS];
    float s[UNITS];
#pragma unroll
    for (int j = 0; j < UNITS; ++j) {
        const bool keys = !((u0 + j) & 1);
        const int head = min((u0 + j) >> 1, H - 1);
        const signed char* from = (keys ? o.k + at * o.k_rs + head * o.k_hs : o.v + at * o.v_rs + head * o.v_hs) + c;
        q[j] = i8x8{};
        s[j] = 0.0f;
        if (at >= 0 && c < W) q[j] = *reinterpret_cast<const i8x8*>(from);
        if (at >= 0) s[j] = (keys ? o.ks : o.vs)[static_cast<long>(head) * m.Tk + at];
    }
#pragma unroll
    for (int j = 0; j < UNITS; ++j) {
        const bool keys = !((u0 + j) & 1);
        const int head = (u0 + j) >> 1;
        if (head >= H) break;
        T* to = (keys ? K + row * k_rs + head * k_hs : V + row * v_rs + head * v_hs) + c;
        Frag<T> f;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = static_cast<T>(s[j] * static_cast<float>(q[j][i]));
        if (vec) {
            if (n > 0) *reinterpret_cast<Frag<T>*>(to) = f;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) to[i] = f[i];
        }
    }
}

// Whether eight elements of a tensor's rows can be moved at once.
bool wide(const Heads& h, int D, int es) { return D % 8 == 0 && attn::aligned(h, es, 16); }

int check(kdec_ctx* ctx, const char* who, int dtype, const void* q_off, const void* k_off, int docs, int Tq, int Tk, int H, int D,
          const Codes& o) {
    if (int rc = attn::check(ctx, who, dtype, q_off, k_off, docs, 1.0f, 0.0f, Tq, Tk, H, H, D)) return rc;
    return attn::check_codes(ctx, who, {o.k, o.k_rs, o.k_hs}, {o.v, o.v_rs, o.v_hs}, o.ks, o.vs, Tk, H, D);
}

}  // namespace
}  // namespace kdec

using namespace kdec;

extern "C" {

int kdec_cache_write(kdec_ctx* ctx, int dtype, const void* K, long k_rs, long k_hs, const void* V, long v_rs, long v_hs,
                     const int* q_off, const int* k_off, const int* k_len, int docs, int Tq, int Tk, int H, int D, void* Kc, long kc_rs,
                     long kc_hs, void* Vc, long vc_rs, long vc_hs, float* k_scale, float* v_scale) {
    if (!ctx) return KDEC_EINVAL;
    const DeviceScope device(ctx);
    const Codes o{static_cast<signed char*>(Kc), static_cast<signed char*>(Vc), kc_rs, kc_hs, vc_rs, vc_hs, k_scale, v_scale};
    if (int rc = check(ctx, "kdec_cache_write", dtype, q_off, k_off, docs, Tq, Tk, H, D, o)) return rc;
    const int W = attn::code_width(D);
    KDEC_CHECK(ctx, attn::apart(kc_rs, kc_hs, Tk, H, W) && attn::apart(vc_rs, vc_hs, Tk, H, W), "kdec_cache_write: rows of the cache overlap");
    if (Tq == 0 || Tk == 0 || docs == 0) return KDEC_OK;
    KDEC_CHECK(ctx, K && V, "kdec_cache_write: null tensor");
    const int es = dtype == KDEC_F32 ? 4 : 2;
    const Docs m{q_off, k_off, k_len, nullptr, docs, 0, Tq, Tk};
    const Heads k{K, k_rs, k_hs}, v{V, v_rs, v_hs};
    const bool vec = wide(k, D, es) && wide(v, D, es);
    ProfScope ps(ctx, "cache", 0.0, 2.0 * Tq * H * (static_cast<double>(es) * D + W + 4));
    const int L = W <= 64 ? 8 : 16;
    const dim3 grid(static_cast<unsigned>(cdiv(Tq, CT / L)), static_cast<unsigned>(cdiv(2L * H, UNITS)));
    KDEC_CHECK(ctx, cdiv(2L * H, UNITS) <= 65535, "kdec_cache_write: too many heads");
    KDEC_CHECK(ctx, grid_holds(cdiv(Tq, CT / L), CT), "kdec_cache_write: too many rows");
    const auto run = [&](auto k_) { hipLaunchKernelGGL(k_, grid, dim3(CT), 0, ctx->stream, m, k, v, o, H, D, W, vec); };
    if (dtype == KDEC_F32) run(L == 8 ? cache_write_k<float, 8> : cache_write_k<float, 16>);
    else run(L == 8 ? cache_write_k<bf16, 8> : cache_write_k<bf16, 16>);
    return launch_check(ctx, "kdec_cache_write");
}

int kdec_cache_read(kdec_ctx* ctx, int dtype, const void* Kc, long kc_rs, long kc_hs, const void* Vc, long vc_rs, long vc_hs,
                    const float* k_scale, const float* v_scale, const int* q_off, const int* k_off, const int* k_len, int docs, int Tq,
                    int Tk, int H, int D, void* K, long k_rs, long k_hs, void* V, long v_rs, long v_hs) {
    if (!ctx) return KDEC_EINVAL;
    const DeviceScope device(ctx);
    const auto bytes = [](const void* p) { return static_cast<signed char*>(const_cast<void*>(p)); };
    const Codes o{bytes(Kc), bytes(Vc), kc_rs, kc_hs, vc_rs, vc_hs, const_cast<float*>(k_scale), const_cast<float*>(v_scale)};
    if (int rc = check(ctx, "kdec_cache_read", dtype, q_off, k_off, docs, Tq, Tk, H, D, o)) return rc;
    if (Tq == 0) return KDEC_OK;
    KDEC_CHECK(ctx, K && V, "kdec_cache_read: null tensor");
    KDEC_CHECK(ctx, attn::apart(k_rs, k_hs, Tq, H, D) && attn::apart(v_rs, v_hs, Tq, H, D), "kdec_cache_read: rows of an output overlap");
    const int es = dtype == KDEC_F32 ? 4 : 2, W = attn::code_width(D);
    const Docs m{q_off, k_off, k_len, nullptr, docs, 0, Tq, Tk};
    const bool vec = wide({K, k_rs, k_hs}, D, es) && wide({V, v_rs, v_hs}, D, es);
    ProfScope ps(ctx, "cache", 0.0, 2.0 * Tq * H * (static_cast<double>(es) * D + W + 4));
    const int L = W <= 64 ? 8 : 16;
    const dim3 grid(static_cast<unsigned>(cdiv(Tq, CT / L)), static_cast<unsigned>(cdiv(2L * H, UNITS)));
    KDEC_CHECK(ctx, cdiv(2L * H, UNITS) <= 65535, "kdec_cache_read: too many heads");
    KDEC_CHECK(ctx, grid_holds(cdiv(Tq, CT / L), CT), "kdec_cache_read: too many rows");
    const auto run = [&](auto k_, auto ty) {
        typedef decltype(ty) E;
        hipLaunchKernelGGL(k_, grid, dim3(CT), 0, ctx->stream, m, o, H, D, W, static_cast<E*>(K), k_rs, k_hs, static_cast<E*>(V), v_rs, v_hs,
                           vec);
    };
    if (dtype == KDEC_F32) run(L == 8 ? cache_read_k<float, 8> : cache_read_k<float, 16>, 0.0f);
    else run(L == 8 ? cache_read_k<bf16, 8> : cache_read_k<bf16, 16>, bf16{});
    return launch_check(ctx, "kdec_cache_read");
}

}  // extern "C"
