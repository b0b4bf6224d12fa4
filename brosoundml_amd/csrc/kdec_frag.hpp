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

#include <type_traits>

#include "kdec_buffer.hpp"

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

__device__ inline f32x8 acc_floats(const f32x16& s, int c) {
    f32x8 f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = s[8 * c + i];
    return f;
}

// Whether a fragment of this lane's holds a value that is not finite: its
// largest magnitude as an integer (bf16), zero times its values (float).
__device__ inline bool not_finite(bf16x8 f) {
    typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
    const u16x8 b = __builtin_bit_cast(u16x8, f) & static_cast<unsigned short>(0x7FFF);
    const auto m4 = __builtin_elementwise_max(b.lo, b.hi);
    const auto m2 = __builtin_elementwise_max(m4.lo, m4.hi);
    return m2[0] >= 0x7F80 || m2[1] >= 0x7F80;
}
__device__ inline bool not_finite(f32x8 f) {
    float zero = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) zero = __builtin_fmaf(f[i], 0.0f, zero);
    return !(zero == 0.0f);
}

// A fragment with zeros for its values that are not finite.
template <class F>
__device__ inline F finite_part(F f) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = __builtin_fabsf(static_cast<float>(f[i])) < __builtin_inff() ? f[i] : 0.0f;
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

// A tile in shared memory: rows of DP elements in units of 16 bytes. It is
// read two ways, a unit of each of 16 rows at once (lds_rows) and a stretch of
// columns of 2 or 4 rows at once (lds_cols); either takes one cycle of the 64
// banks only if the units fall on different banks. Rows are a multiple or an
// even part of the banks, so the units of a row are permuted by an exclusive
// or with bits of the row that set apart the rows of both reads. Float tiles
// settle for two cycles and simpler addresses: their products take sixteen
// times as long.
template <class T, int DP>
struct Tile {
    static constexpr int U = 16 / static_cast<int>(sizeof(T)), NU = DP / U;
    __device__ static inline int swz(int row) {
        if (sizeof(T) == 2 && NU >= 16) return (row & 3) << 2 | (row >> 2 & 3);
        if (sizeof(T) == 2 && NU == 8) return (row >> 1 & 1) << 2 | (row >> 2 & 3);
        if (sizeof(T) == 2 && NU == 4) return row >> 2 & 3;
        if (sizeof(T) == 4) return NU == 8 ? row >> 1 & 7 : row & 7;
        return 0;
    }
    __device__ static inline int at(int row, int unit) { return row * DP + U * (unit ^ swz(row)); }
    // 8 elements to column 8 * chunk
    __device__ static inline void put8(T* tile, int row, int chunk, const Frag<T>& f) {
        if constexpr (sizeof(T) == 2) {
            *reinterpret_cast<Frag<T>*>(tile + at(row, chunk)) = f;
        } else {
            *reinterpret_cast<f32x4*>(tile + at(row, 2 * chunk)) = __builtin_shufflevector(f, f, 0, 1, 2, 3);
            *reinterpret_cast<f32x4*>(tile + at(row, 2 * chunk + 1)) = __builtin_shufflevector(f, f, 4, 5, 6, 7);
        }
    }
};

// A lane's place in a tile, in a register of its own: which tile and which of
// its row blocks then is the read's own offset. (Left alone, the compiler
// merges the two and keeps a register per tile and block.)
__device__ inline int own_reg(int at) {
    asm("" : "+v"(at));
    return at;
}

// The depth-16 step c of a tile as an operand whose rows are the tile's rows
// row0 .. row0 + 31, depth along the tile's columns.
template <class T, int DP>
__device__ inline Frag<T> lds_rows(const T* tile, int row0, int c) {
    const int l = threadIdx.x & 63;
    typedef Tile<T, DP> Tl;
    if constexpr (sizeof(T) == 2) {
        return *reinterpret_cast<const Frag<T>*>(tile + row0 * DP + own_reg(Tl::at(l & 31, 2 * c + (l >> 5))));
    } else {
        const float* p = tile + row0 * DP;
        const f32x4 a = *reinterpret_cast<const f32x4*>(p + own_reg(Tl::at(l & 31, 4 * c + 2 * (l >> 5))));
        const f32x4 b = *reinterpret_cast<const f32x4*>(p + own_reg(Tl::at(l & 31, 4 * c + 2 * (l >> 5) + 1)));
        return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
}

// A tile's columns col0 .. col0 + 31 as an operand's rows, depth along the 16
// tile rows from row0, in the order of acc_frag's slots (ACC) or in their own.
// bf16 reads it with the transposing LDS read, which hands lane i of 16 the
// column i of a 4 x 16 block whose row j the lanes 4j .. 4j + 3 address.
template <int DP, bool ACC>
__device__ inline bf16x8 lds_cols(const bf16* tile, int row0, int col0) {
    typedef __attribute__((address_space(3))) short4v lds4;
    const int l = threadIdx.x & 63;
    // row0 is a multiple of 16, after which the permutation repeats
    const int row = (ACC ? 4 : 8) * (l >> 5) + (l >> 2 & 3), col = col0 + 16 * (l >> 4 & 1) + 4 * (l & 3);
    union { short4v s[2]; bf16x8 v; } u;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        u.s[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds4*)(tile + row0 * DP + own_reg(Tile<bf16, DP>::at(row + (ACC ? 8 : 4) * i, col >> 3) + (col & 7))));
    return u.v;
}
template <int DP, bool ACC>
__device__ inline f32x8 lds_cols(const float* tile, int row0, int col0) {
    static_assert(DP >= 64, "the permutation below is that of these widths: the low three bits of the row");
    const int l = threadIdx.x & 63, half = l >> 5;
    f32x8 f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = ACC ? 8 * (i >> 2) + (i & 3) : i;  // row0 is a multiple of 16, col0 of 32
        const int low = ACC ? 4 * half + (i & 3) : i;    // the row's low three bits
        const int at = own_reg((ACC ? 4 : 8) * half * DP + 4 * (((l & 31) >> 2) ^ low) + (l & 3));
        f[i] = tile[at + (row0 + r) * DP + col0];
    }
    return f;
}

// Bounds-checked loads of a tensor's rows: of `rows` rows (any number) from a
// wave-uniform base, each D columns; what lies past them is zeros. kFar is an
// offset past every descriptor's end (all are below 2^30 bytes).
constexpr int kFar = 0x60000000;
template <class T>
__device__ inline __amdgpu_buffer_rsrc_t rows_rsrc(const T* base, long rs, int rows, int D) {
    return uniform_rsrc(base, rows > 0 ? static_cast<int>(((rows - 1) * rs + D) * static_cast<long>(sizeof(T))) : 0);
}
__device__ inline bf16x8 buffer_load8(__amdgpu_buffer_rsrc_t r, int off, bf16) {
    return __builtin_bit_cast(bf16x8, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}
__device__ inline f32x8 buffer_load8(__amdgpu_buffer_rsrc_t r, int off, float) {
    const f32x4 a = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
    const f32x4 b = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off + 16, 0, 0));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}

// Waits until at most N of the wave's memory loads (copies among them) are
// outstanding.
template <int N>
__device__ inline void wait_loads() {
    __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4) << 14 | 7 << 4 | 15 << 8);
}

// A barrier for shared memory alone: the wave's own reads and writes of it are
// done, its copies from memory may still be on their way (__syncthreads would
// wait for them too).
__device__ inline void lds_barrier() {
    __builtin_amdgcn_s_waitcnt(15 | 3 << 14 | 7 << 4);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// 16 bytes per lane from the descriptor's offset `off` to shared memory at
// `to` (wave-uniform) + 16 * lane.
__device__ inline void copy16(__amdgpu_buffer_rsrc_t r, void* to, int off) {
    typedef __attribute__((address_space(3))) void Shared;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (Shared*)to, 16, off, 0, 0, 0);
}

// Copies a tile of ROWS rows from memory straight into shared memory, 16 bytes
// per thread at a time: unit u of the tile is written by thread u mod NT, so
// the permutation of a row's units is made on the side of the memory
// addresses. A thread's offset stays from tile to tile; those of its further
// units are whole steps of rows away where the permutation repeats after that
// many rows, and are kept one by one where it does not.
template <class T, int DP, int ROWS, int NT>
struct Copy {
    typedef Tile<T, DP> Tl;
    static constexpr int N = ROWS * Tl::NU / NT, STEP = NT / Tl::NU;
    static constexpr bool SAME = STEP % (sizeof(T) == 4 && Tl::NU > 8 ? 8 : 16) == 0;
    int off[SAME ? 1 : N], step;
    __device__ inline void init(long rs, int D, int tid) {
        step = static_cast<int>(STEP * rs * static_cast<long>(sizeof(T)));
#pragma unroll
        for (int i = 0; i < (SAME ? 1 : N); ++i) {
            const int u = tid + i * NT, row = u / Tl::NU, col = Tl::U * ((u % Tl::NU) ^ Tl::swz(row));
            off[i] = col < D ? static_cast<int>((row * rs + col) * static_cast<long>(sizeof(T))) : kFar;
        }
    }
    __device__ inline void load(T* tile, const T* base, long rs, int rows, int D, int wave) const {
        const __amdgpu_buffer_rsrc_t r = rows_rsrc(base, rs, min(rows, ROWS), D);
#pragma unroll
        for (int i = 0; i < N; ++i)
            copy16(r, tile + (64 * wave + i * NT) * Tl::U, SAME ? off[0] + i * step : off[SAME ? 0 : i]);
    }
    // The thread's own units of the tile (its loads have landed): values that
    // are not finite become zeros, f(row) is told of their rows. bf16 takes a
    // unit as it is; float units are half a fragment.
    template <class F>
    __device__ static inline void clean(T* tile, int tid, F f) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            typedef T V __attribute__((ext_vector_type(Tl::U)));
            V* p = reinterpret_cast<V*>(tile + (tid + i * NT) * Tl::U);
            V v = *p;
            bool bad = false;
#pragma unroll
            for (int x = 0; x < Tl::U; ++x)
                if (!(__builtin_fabsf(static_cast<float>(v[x])) < __builtin_inff())) {
                    v[x] = static_cast<T>(0.0f);
                    bad = true;
                }
            if (bad) {
                *p = v;
                f((tid + i * NT) / Tl::NU);
            }
        }
    }
};

// A float fragment as bf16 terms whose sum holds it to 16 (two terms) or 24
// bits (three): products with a bf16 operand then lose nothing that float
// sums would keep. Float operands are one term. WILD: a value that is not
// finite is the first term alone.
template <class T, int N, bool WILD = false> struct Terms;
template <int N, bool WILD> struct Terms<bf16, N, WILD> {
    static constexpr int n = N;
    bf16x8 t[N];
    __device__ explicit Terms(f32x8 f) {
#pragma unroll
        for (int k = 0; k < N; ++k)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                t[k][i] = static_cast<bf16>(f[i]);
                if (k + 1 == N) continue;
                f[i] -= static_cast<float>(t[k][i]);
                if (WILD && k == 0) f[i] = f[i] == f[i] ? f[i] : 0.0f;  // infinity less infinity, or NaN
            }
    }
};
template <int N, bool WILD> struct Terms<float, N, WILD> {
    static constexpr int n = 1;
    f32x8 t[1];
    __device__ explicit Terms(f32x8 f) { t[0] = f; }
};

// The sum over a wave's lanes up to each lane's own.
__device__ inline int wave_scan(int x) {
    const auto add = [&](auto ctrl, auto rows) __attribute__((always_inline)) {
        x += __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 15, false);
    };
    typedef std::integral_constant<int, 15> All;
    add(std::integral_constant<int, 0x111>{}, All{});  // lanes of 16 to the right by 1, 2, 4, 8
    add(std::integral_constant<int, 0x112>{}, All{});
    add(std::integral_constant<int, 0x114>{}, All{});
    add(std::integral_constant<int, 0x118>{}, All{});
    add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 10>{});  // the 16's last lane to the next 16
    add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 12>{});  // lane 31 to the upper half
    return x;
}

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

}  // namespace kdec
