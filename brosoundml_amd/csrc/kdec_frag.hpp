// Matrix fragments of the token operators on gfx950, one set of names for
// bf16 and float operands.
//
// A fragment is 8 elements per lane: of a 32 x 16 operand (rows m or columns
// n of one matrix product step of depth 16), lane l holds row l % 32 and the
// depth slots 8 * (l / 32) .. + 7. bf16 takes it in one
// v_mfma_f32_32x32x16_bf16; float in eight v_mfma_f32_32x32x2_f32, product i
// over element i of both lane halves. Depth slots may stand for any depth
// indices as long as both operands use the same ones, which is what lets an
// accumulator become the next product's operand without moving between lanes:
// accumulator register r of lane l is row acc_row(r, l / 32), column l % 32,
// so registers 8c .. 8c + 7 are a fragment whose slots are the rows
// 16 c + 8 (i / 4) + 4 (l / 32) + i % 4.
#pragma once

#include <hip/hip_runtime.h>

namespace kdec {

typedef __bf16 bf16;
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

template <class T> struct FragOf;
template <> struct FragOf<bf16> { typedef bf16x8 type; };
template <> struct FragOf<float> { typedef f32x8 type; };
template <class T> using Frag = typename FragOf<T>::type;

__device__ inline f32x16 mma32(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ inline f32x16 mma32(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
}

__device__ inline int acc_row(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

// Registers 8c .. 8c + 7 of an accumulator as a fragment (see above): bf16
// rounds to nearest even, float takes them as they are.
template <class T>
__device__ inline Frag<T> acc_frag(const f32x16& s, int c) {
    Frag<T> f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = static_cast<T>(s[8 * c + i]);
    return f;
}

// 8 elements at p, of which the first n are the tensor's (zeros beyond).
// vec: p is aligned to 16 bytes and n is a multiple of 16 bytes' elements.
__device__ inline bf16x8 load8(const bf16* p, int n, bool vec) {
    bf16x8 f = bf16x8{};
    if (vec) {
        if (n > 0) f = *reinterpret_cast<const bf16x8*>(p);
        return f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? p[i] : static_cast<bf16>(0.0f);
    return f;
}
__device__ inline f32x8 load8(const float* p, int n, bool vec) {
    f32x8 f = f32x8{};
    if (vec) {
        f32x4 a = f32x4{}, b = f32x4{};
        if (n > 0) a = *reinterpret_cast<const f32x4*>(p);
        if (n > 4) b = *reinterpret_cast<const f32x4*>(p + 4);
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? p[i] : 0.0f;
    return f;
}

// The depth-16 step c of a tile held row-major in shared memory (stride `ls`
// elements) as an operand whose rows are the tile's rows row0 .. row0 + 31.
template <class T>
__device__ inline Frag<T> lds_rows(const T* tile, int ls, int row0, int c) {
    const int l = threadIdx.x & 63;
    return *reinterpret_cast<const Frag<T>*>(tile + (row0 + (l & 31)) * ls + 16 * c + 8 * (l >> 5));
}

// The same tile transposed: an operand whose rows are the tile's columns
// col0 .. col0 + 31 and whose depth slots are the rows of acc_frag(c) of the
// 32-row block at row0. bf16 reads it with the transposing LDS read, which
// hands lane i of 16 the column i of a 4 x 16 block whose row j the lanes
// 4j .. 4j + 3 address.
__device__ inline bf16x8 lds_cols(const bf16* tile, int ls, int row0, int col0, int c) {
    typedef __attribute__((address_space(3))) short4v lds4;
    const int l = threadIdx.x & 63;
    const bf16* p = tile + (row0 + 16 * c + 4 * (l >> 5) + ((l >> 2) & 3)) * ls + col0 + 16 * ((l >> 4) & 1) + 4 * (l & 3);
    union { short4v s[2]; bf16x8 v; } u;
    u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)p);
    u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(p + 8 * ls));
    return u.v;
}
__device__ inline f32x8 lds_cols(const float* tile, int ls, int row0, int col0, int c) {
    const int l = threadIdx.x & 63;
    const float* p = tile + (row0 + 16 * c + 4 * (l >> 5)) * ls + col0 + (l & 31);
    f32x8 f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = p[(8 * (i >> 2) + (i & 3)) * ls];
    return f;
}

// lds_rows with the depth slots of acc_frag, the other operand of lds_cols.
__device__ inline bf16x8 lds_rows_acc(const bf16* tile, int ls, int row0, int c) {
    const int l = threadIdx.x & 63;
    const bf16* p = tile + (row0 + (l & 31)) * ls + 16 * c + 4 * (l >> 5);
    const bf16x4 a = *reinterpret_cast<const bf16x4*>(p), b = *reinterpret_cast<const bf16x4*>(p + 8);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
__device__ inline f32x8 lds_rows_acc(const float* tile, int ls, int row0, int c) {
    const int l = threadIdx.x & 63;
    const float* p = tile + (row0 + (l & 31)) * ls + 16 * c + 4 * (l >> 5);
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 8);
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// A float fragment as bf16 terms whose sum holds it to 16 (two terms) or 24
// bits (three): products with a bf16 operand then lose nothing that float
// sums would keep. Float operands are one term.
template <class T, int N> struct Terms;
template <int N> struct Terms<bf16, N> {
    static constexpr int n = N;
    bf16x8 t[N];
    __device__ explicit Terms(f32x8 f) {
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                t[k][i] = static_cast<bf16>(f[i]);
                f[i] -= static_cast<float>(t[k][i]);
            }
    }
};
template <int N> struct Terms<float, N> {
    static constexpr int n = 1;
    f32x8 t[1];
    __device__ explicit Terms(f32x8 f) { t[0] = f; }
};

// Four values rounded to T at p, of which the first n are the tensor's.
// vec: p is aligned to the four and n is 0 or 4 (or less).
template <class T>
__device__ inline void store4(T* p, int n, bool vec, float a, float b, float c, float d) {
    const T v[4] = {static_cast<T>(a), static_cast<T>(b), static_cast<T>(c), static_cast<T>(d)};
    if (n <= 0) return;
    if (vec) {
        typedef T V4 __attribute__((ext_vector_type(4)));
        *reinterpret_cast<V4*>(p) = V4{v[0], v[1], v[2], v[3]};
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < n) p[i] = v[i];
}

// Whether any of the fragment's values is not finite.
template <class T>
__device__ inline bool any_nonfinite(const Frag<T>& f) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) bad |= !(__builtin_fabsf(static_cast<float>(f[i])) < __builtin_inff());
    return bad;
}
template <class T>
__device__ inline Frag<T> finite_or_zero(Frag<T> f) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (!(__builtin_fabsf(static_cast<float>(f[i])) < __builtin_inff())) f[i] = static_cast<T>(0.0f);
    return f;
}

}  // namespace kdec
