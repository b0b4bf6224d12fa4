// The counter-based generator behind dropout: Philox4x32-10 (Salmon, Moraes,
// Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011).
//
// The mask of an element depends on the seed, the offset and the element's
// row and column alone, so a kernel forms it where it needs it and nothing
// is stored: key = the seed's two words, counter = (col >> 3, row, the
// offset's two words), and the eight 16-bit halves of the result belong to
// the eight columns 8 (col >> 3) .. + 7.
#pragma once

#include <hip/hip_runtime.h>

namespace kdec {

struct Drop {
    unsigned k0, k1, o0, o1;
    unsigned thr;  // dropped where the half is below it: p in 1/65536
    float keep;    // the kept values' factor, 65536 / (65536 - thr)
};

// p in [0, 1) to Drop; false where p (or what it rounds to) is not below 1.
inline bool make_drop(float p, long seed, long offset, Drop& d) {
    if (!(p >= 0.0f && p < 1.0f)) return false;
    const int thr = static_cast<int>(static_cast<double>(p) * 65536.0 + 0.5);
    if (thr >= 65536) return false;
    d.k0 = static_cast<unsigned>(seed);
    d.k1 = static_cast<unsigned>(static_cast<unsigned long>(seed) >> 32);
    d.o0 = static_cast<unsigned>(offset);
    d.o1 = static_cast<unsigned>(static_cast<unsigned long>(offset) >> 32);
    d.thr = static_cast<unsigned>(thr);
    d.keep = static_cast<float>(65536.0 / (65536 - thr));
    return true;
}

// The eight halves of columns 8 g .. 8 g + 7 of a row: w[i / 2], low half
// where i is even.
__device__ inline void drop_words(const Drop& d, unsigned row, unsigned g, unsigned (&w)[4]) {
    unsigned c0 = g, c1 = row, c2 = d.o0, c3 = d.o1, k0 = d.k0, k1 = d.k1;
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const unsigned long long a = static_cast<unsigned long long>(c0) * 0xD2511F53u;
        const unsigned long long b = static_cast<unsigned long long>(c2) * 0xCD9E8D57u;
        c0 = static_cast<unsigned>(b >> 32) ^ c1 ^ k0;
        c2 = static_cast<unsigned>(a >> 32) ^ c3 ^ k1;
        c1 = static_cast<unsigned>(b);
        c3 = static_cast<unsigned>(a);
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    w[0] = c0;
    w[1] = c1;
    w[2] = c2;
    w[3] = c3;
}

__device__ inline bool kept(const Drop& d, const unsigned (&w)[4], int i) {
    return ((i & 1) ? w[i >> 1] >> 16 : w[i >> 1] & 0xFFFFu) >= d.thr;
}

}  // namespace kdec
