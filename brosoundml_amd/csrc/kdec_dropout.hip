// Dropout with a residual on gfx950, its mask from the counter-based
// generator of kdec_philox.hpp and never stored.
//
// Y = R + keep * mask * X, the sum in float and rounded once. One lane forms
// the eight mask halves of eight columns and handles those columns.
#include "kdec_frag.hpp"
#include "kdec_internal.hpp"
#include "kdec_philox.hpp"

namespace kdec {
namespace {

constexpr int DT = 256;

template <class T, bool RES>
__global__ __launch_bounds__(DT) void dropout_k(const T* X, long x_rs, const T* R, long r_rs, T* Y, long y_rs,
                                                unsigned rows, int cols, unsigned groups, bool vec, Drop d) {
    const unsigned per = gridDim.x * DT;  // at most 2^31
    const unsigned long long total = static_cast<unsigned long long>(rows) * groups;
    for (unsigned long long e = blockIdx.x * DT + threadIdx.x; e < total; e += per) {
        unsigned row, g;
        if (total <= 0xFFFFFFFFull) {
            row = static_cast<unsigned>(e) / groups;
            g = static_cast<unsigned>(e) - row * groups;
        } else {
            row = static_cast<unsigned>(e / groups);
            g = static_cast<unsigned>(e - static_cast<unsigned long long>(row) * groups);
        }
        const int c = 8 * static_cast<int>(g), n = min(8, cols - c);
        Frag<T> x = load8(X + row * x_rs + c, n, vec), r;
        if (RES) r = load8(R + row * r_rs + c, n, vec);
        unsigned w[4];
        drop_words(d, row, g, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = kept(d, w, i) ? d.keep * static_cast<float>(x[i]) : 0.0f;
            x[i] = static_cast<T>(RES ? v + static_cast<float>(r[i]) : v);
        }
        T* y = Y + row * y_rs + c;
        if (vec) {
            *reinterpret_cast<Frag<T>*>(y) = x;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) y[i] = x[i];
        }
    }
}

template <class T>
void launch(kdec_ctx* ctx, const void* X, long x_rs, const void* R, long r_rs, void* Y, long y_rs, long rows,
            int cols, const Drop& d) {
    const int el = 16 / static_cast<int>(sizeof(T));  // elements per 16 bytes
    const auto ok = [&](const void* p, long rs) { return reinterpret_cast<size_t>(p) % 16 == 0 && rs % el == 0; };
    const bool vec = cols % 8 == 0 && ok(X, x_rs) && ok(Y, y_rs) && (!R || ok(R, r_rs));
    const unsigned groups = static_cast<unsigned>(cdiv(cols, 8));
    long blocks = cdiv(rows * groups, DT);
    if (blocks > 16L * ctx->num_cus) blocks = 16L * ctx->num_cus;
    const auto k = R ? dropout_k<T, true> : dropout_k<T, false>;
    hipLaunchKernelGGL(k, dim3(static_cast<unsigned>(blocks)), dim3(DT), 0, ctx->stream, static_cast<const T*>(X),
                       x_rs, static_cast<const T*>(R), r_rs, static_cast<T*>(Y), y_rs, static_cast<unsigned>(rows),
                       cols, groups, vec, d);
}

}  // namespace
}  // namespace kdec

using namespace kdec;

extern "C" {

int kdec_dropout(kdec_ctx* ctx, int dtype, const void* X, long x_rs, const void* R, long r_rs, void* Y, long y_rs,
                 long rows, int cols, float p, long seed, long offset) {
    if (!ctx) return KDEC_EINVAL;
    KDEC_CHECK(ctx, dtype == KDEC_F32 || dtype == KDEC_BF16, "kdec_dropout: unknown type");
    KDEC_CHECK(ctx, rows >= 0 && rows <= 0xFFFFFFFFL && cols >= 0 && cols <= 0x7FFFFFF0, "kdec_dropout: bad sizes");
    Drop d;
    KDEC_CHECK(ctx, make_drop(p, seed, offset, d), "kdec_dropout: p must be at least 0 and below 1");
    if (rows == 0 || cols == 0) return KDEC_OK;
    KDEC_CHECK(ctx, X && Y, "kdec_dropout: null tensor");
    KDEC_CHECK(ctx, rows == 1 || y_rs >= cols, "kdec_dropout: row stride of Y too small");
    ProfScope ps(ctx, "dropout", 0.0,
                 static_cast<double>(rows) * cols * (dtype == KDEC_F32 ? 4 : 2) * (R ? 3 : 2));
    if (dtype == KDEC_F32) launch<float>(ctx, X, x_rs, R, r_rs, Y, y_rs, rows, cols, d);
    else launch<bf16>(ctx, X, x_rs, R, r_rs, Y, y_rs, rows, cols, d);
    return launch_check(ctx, "kdec_dropout");
}

}  // extern "C"
