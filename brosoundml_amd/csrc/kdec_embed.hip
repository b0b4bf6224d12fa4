// Embedding lookup on gfx950, and the gradient of its table by sorted tokens.
//
// Forward: Y[t] = scale * table[ids[t]], a row of zeros where the id is outside
// the table. Sixteen bytes a lane; bound by memory.
//
// Backward: dtable[v] = beta dtable[v] + scale * sum of dY[t] over the tokens t
// of id v, in ascending t. Tokens are sorted by id first, cut into pieces of a
// fixed number of sorted tokens, and a wave walks a piece for a stretch of
// columns: a run of one id that lies inside the piece goes to the table, what a
// run leaves at a piece's ends goes to a partial row, and the partial rows of a
// run are added in the pieces' order. So every piece is the same work however
// often an id occurs, and every sum has one order.
//
// The sort is one launch: block b owns a range of ids, looks at all tokens,
// counts those of lower ids and ranks its own (within 64 tokens by ballots over
// the id's bits, then by wave and id with one scan). It also begins its ids' rows of the table (cleared, or scaled by beta),
// before anything else: these stores go their way while the block sorts. More tokens than a block
// holds take a radix sort over several blocks.
#include "kdec_frag.hpp"
#include "kdec_internal.hpp"

#include <climits>
#include <type_traits>

namespace kdec {
namespace {

constexpr int ET = 256;         // threads of the copying and summing blocks
constexpr int ST = 1024;        // threads of a sorting block
constexpr int SI = 16;          // tokens a thread of it holds at most
constexpr int CHUNK = ST * SI;  // tokens a sorting block holds
constexpr int WAVES = ST / 64;
constexpr int DIGITS = 256;

// A lane's part of a row: 16 bytes, a value at a time where rows do not start on
// them (16381 rows of 1021 bf16: lookup 35 us and sums 42 where 1024 columns take 12
// and 14; 8190 rows of 765 floats 16 and 12 for 8 and 9).
template <class T> constexpr int PART = 16 / sizeof(T);
template <class T> struct PartOf;
template <> struct PartOf<float> { typedef f32x4 type; };
template <> struct PartOf<bf16> { typedef bf16x8 type; };
template <class T> using Part = typename PartOf<T>::type;

template <class T>
__device__ inline Part<T> load_part(const T* p, int n, bool vec) {
    Part<T> f = Part<T>{};
    if (vec) {
        if (n > 0) f = *reinterpret_cast<const Part<T>*>(p);
        return f;
    }
#pragma unroll
    for (int i = 0; i < PART<T>; ++i) f[i] = i < n ? p[i] : static_cast<T>(0.0f);
    return f;
}

// Four parts a thread, a block's width apart: their ids, then their rows are on
// their way together (16381 rows of 1024 bf16 from a table of 32000: 12.2 us, one
// part a thread 13.2; rows that one round of blocks holds take the same).
constexpr int J = 4;
template <class T>
__global__ __launch_bounds__(ET) void embed_k(const T* __restrict__ table, long t_rs, const int* __restrict__ ids, T* __restrict__ Y,
                                              long y_rs, int rows, int vocab, int cols, unsigned groups, bool vec, float scale) {
    constexpr int E = PART<T>;
    const unsigned long long total = static_cast<unsigned long long>(rows) * groups;
    for (unsigned long long e0 = static_cast<unsigned long long>(blockIdx.x) * (ET * J) + threadIdx.x; e0 < total;
         e0 += static_cast<unsigned long long>(gridDim.x) * (ET * J)) {
        long row[J];
        int c[J], id[J];
        Part<T> f[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const unsigned long long e = min(e0 + static_cast<unsigned long long>(j) * ET, total - 1);
            if (total <= 0xFFFFFFFFull) {
                const unsigned r = static_cast<unsigned>(e) / groups;
                row[j] = r;
                c[j] = E * static_cast<int>(static_cast<unsigned>(e) - r * groups);
            } else {
                row[j] = static_cast<long>(e / groups);
                c[j] = E * static_cast<int>(e - static_cast<unsigned long long>(row[j]) * groups);
            }
            id[j] = ids[row[j]];
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const bool in = static_cast<unsigned>(id[j]) < static_cast<unsigned>(vocab);
            f[j] = load_part(table + (in ? id[j] * t_rs + c[j] : 0), in ? min(E, cols - c[j]) : 0, vec);
        }
#pragma unroll
        for (int j = 0; j < J; ++j) {
            if (e0 + static_cast<unsigned long long>(j) * ET >= total) break;
            T* y = Y + row[j] * y_rs + c[j];
#pragma unroll
            for (int i = 0; i < E; ++i) f[j][i] = static_cast<T>(scale * static_cast<float>(f[j][i]));
            if (vec) {
                *reinterpret_cast<Part<T>*>(y) = f[j];
            } else {
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (i < cols - c[j]) y[i] = f[j][i];
            }
        }
    }
}

// ─── sort ───

struct Tokens {
    int *id, *at;  // ids in order, and the tokens that have them
};

struct Sort {
    const int* ids;
    int T, vocab, bits;  // bits of a digit
    float* table;        // cleared or scaled by the blocks beside the sort
    long n;
    float beta;
};

// Ids outside the table sort behind it.
__device__ inline int key_of(int id, int vocab) { return static_cast<unsigned>(id) < static_cast<unsigned>(vocab) ? id : vocab; }

// Clears n floats or scales them by beta, from place `first` on in steps of `step`
// threads.
__device__ inline void begin_rows(float* to, long n, float beta, long first, long step) {
    if (beta == 1.0f) return;
    const long quads = reinterpret_cast<size_t>(to) % 16 == 0 ? n / 4 : 0;
    f32x4* q = reinterpret_cast<f32x4*>(to);
    if (beta == 0.0f) {
#pragma unroll 4
        for (long i = first; i < quads; i += step) q[i] = f32x4{};
        for (long i = 4 * quads + first; i < n; i += step) to[i] = 0.0f;
    } else {
#pragma unroll 4
        for (long i = first; i < quads; i += step) q[i] *= beta;
        for (long i = 4 * quads + first; i < n; i += step) to[i] *= beta;
    }
}

// A block's tokens by one digit. Wave w holds the tokens 64 n w .. + 64 n - 1 of
// the block's, thread by thread (token 64 g + lane of them in place g).
struct Ranks {
    int n;            // places in use, the same in all waves
    int digit[SI];    // -1: no token
    int place[SI];    // rank among the same digit's of the 64 tokens, their number above it
};
__device__ inline void rank64(int digit, int bits, int& place) {
    const int lane = threadIdx.x & 63;
    unsigned long long same = __builtin_amdgcn_ballot_w64(digit >= 0);
    place = 0;
    if (!same) return;
    for (int b = 0; b < bits; ++b) {
        const unsigned long long one = __builtin_amdgcn_ballot_w64(digit >> b & 1);
        same &= (digit >> b & 1) ? one : ~one;
    }
    const int before = __builtin_popcountll(same & ((1ull << lane) - 1));
    place = before | __builtin_popcountll(same) << 8;
}

// The sum of the first n of the block's waves' values.
__device__ inline int first_waves(const int* sums, int n) {
    const int lane = threadIdx.x & 63;
    return __builtin_amdgcn_readlane(wave_scan(lane < n ? sums[min(lane, WAVES - 1)] : 0), 63);
}

// Counts cnt[wave][digit], then their exclusive sums, digits first: where each
// wave's tokens of a digit begin in the block's order.
__device__ inline void block_offsets(Ranks& r, int bits, int (*cnt)[DIGITS], int* sums) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    for (int i = tid; i < WAVES * DIGITS; i += ST) (&cnt[0][0])[i] = 0;
    __syncthreads();
#pragma unroll
    for (int g = 0; g < SI; ++g)
        if (g < r.n) {
            rank64(r.digit[g], bits, r.place[g]);
            if (r.digit[g] >= 0 && (r.place[g] & 255) == 0) atomicAdd(&cnt[wave][r.digit[g]], r.place[g] >> 8);
        }
    __syncthreads();
    // thread: digit tid / 4, waves 4 (tid % 4) .. + 3
    const int d = tid >> 2, w = 4 * (tid & 3);
    int v[4], sum = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[i] = cnt[w + i][d];
        sum += v[i];
    }
    const int upto = wave_scan(sum);
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int at = upto - sum + first_waves(sums, wave);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        cnt[w + i][d] = at;
        at += v[i];
    }
    __syncthreads();
}

// The tokens' places in order: f(g, place). Advances cnt.
template <class F>
__device__ inline void place_all(const Ranks& r, int (*cnt)[DIGITS], F f) {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int g = 0; g < SI; ++g)
        if (g < r.n && __builtin_amdgcn_ballot_w64(r.digit[g] >= 0)) {
            const int d = r.digit[g];
            if (d >= 0) {
                const int base = cnt[wave][d];
                f(g, base + (r.place[g] & 255));
                if ((r.place[g] & 255) == 0) cnt[wave][d] = base + (r.place[g] >> 8);
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the first lane's count before the next read
            __builtin_amdgcn_wave_barrier();
        }
}

// Block b's ids, `per` of them from b * per (those outside the table count as
// one more, vocab), of up to CHUNK tokens: the block lists its own tokens in
// order, most of what it looks at is not, and sorts the list (16381 tokens of
// 32000 ids with the table's 131 MB, which take 21 us by themselves: 28 us, and 32
// with ranks of all tokens in place; 8190 tokens of 181 ids 6.6 and 8.5). FEW
// tokens are summed right here, a thread's columns over every run in order.
constexpr int FEW = 512;
template <class T, bool SUM>
__global__ __launch_bounds__(ST) void sort_range_k(Sort s, int per, Tokens out, const T* __restrict__ dY, long rs, int cols, float scale) {
    __shared__ int cnt[WAVES][DIGITS], sums[WAVES], start[DIGITS + 1], lower[WAVES], owned[WAVES];
    __shared__ int list[SUM ? FEW : CHUNK];  // token, digit above it
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, lo = blockIdx.x * per;
    const int places = (s.T + ST - 1) / ST, first = wave * 64 * places + lane;
    int id[SI];
#pragma unroll
    for (int g = 0; g < SI; ++g) {
        const int i = first + 64 * g;
        id[g] = g < places && i < s.T ? key_of(s.ids[i], s.vocab) : INT_MAX;
    }
    const int n = min(per, s.vocab - lo);
    begin_rows(s.table + static_cast<long>(lo) * cols, static_cast<long>(n) * cols, s.beta, tid, ST);
    const auto mine = [&](int g) __attribute__((always_inline)) { return static_cast<unsigned>(id[g] - lo) < static_cast<unsigned>(per); };
    int less = 0, own = 0;
#pragma unroll
    for (int g = 0; g < SI; ++g) {
        less += __builtin_popcountll(__builtin_amdgcn_ballot_w64(id[g] < lo));
        own += __builtin_popcountll(__builtin_amdgcn_ballot_w64(mine(g)));
    }
    if (lane == 0) {
        lower[wave] = less;
        owned[wave] = own;
    }
    __syncthreads();
    const int base = first_waves(lower, WAVES), total = first_waves(owned, WAVES);
    int at = first_waves(owned, wave);
#pragma unroll
    for (int g = 0; g < SI; ++g) {
        const unsigned long long m = __builtin_amdgcn_ballot_w64(mine(g));
        if (m) {
            if (mine(g)) list[at + __builtin_popcountll(m & ((1ull << lane) - 1))] = (first + 64 * g) | (id[g] - lo) << 16;
            at += __builtin_popcountll(m);
        }
    }
    __syncthreads();
    if (per > 1) {
        Ranks r;
        r.n = (total + ST - 1) / ST;
        const int from = wave * 64 * r.n + lane;
        int token[SI];
#pragma unroll
        for (int g = 0; g < SI; ++g) {
            const int i = from + 64 * g;
            token[g] = g < r.n && i < total ? list[i] : 0;
            r.digit[g] = g < r.n && i < total ? token[g] >> 16 : -1;
        }
        block_offsets(r, s.bits, cnt, sums);  // behind the list's last reads
        if (tid < DIGITS) start[tid] = cnt[0][tid];
        if (tid == 0) start[DIGITS] = total;
        __syncthreads();
        place_all(r, cnt, [&](int g, int to) {
            if (SUM) {
                list[to] = token[g];
            } else {
                out.id[base + to] = lo + r.digit[g];
                out.at[base + to] = token[g] & 0xFFFF;
            }
        });
    } else {
        if (tid == 0) {
            start[0] = 0;
            start[1] = total;
        }
        if (!SUM)
            for (int i = tid; i < total; i += ST) {
                out.id[base + i] = lo;
                out.at[base + i] = list[i];
            }
    }
    if (!SUM) return;
    __syncthreads();
    for (int i0 = 0, i1; i0 < total; i0 = i1) {
        const int digit = per > 1 ? list[i0] >> 16 : 0;
        i1 = start[digit + 1];
        if (digit >= n) break;  // outside the table
        const auto row = [&](int i) __attribute__((always_inline)) { return dY + (list[i] & 0xFFFF) * rs; };
        for (int c = tid; c < cols; c += ST) {
            float acc = 0.0f;
            int i = i0;
            for (; i + 8 <= i1; i += 8) {
                float f[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] = static_cast<float>(row(i + j)[c]);
#pragma unroll
                for (int j = 0; j < 8; ++j) acc += f[j];
            }
            for (; i < i1; ++i) acc += static_cast<float>(row(i)[c]);
            float* to = s.table + static_cast<long>(lo + digit) * cols + c;
            *to = s.beta == 0.0f ? scale * acc : *to + scale * acc;
        }
    }
}

// More tokens: a digit's counts by chunk, then every chunk's tokens to their
// places. counts[digit * chunks + chunk].
__global__ __launch_bounds__(ST) void sort_count_k(Sort s, int pass, int chunks, const int* src, int* counts) {
    __shared__ int cnt[DIGITS];
    if (static_cast<int>(blockIdx.x) >= chunks) {
        begin_rows(s.table, s.n, s.beta, static_cast<long>(blockIdx.x - chunks) * ST + threadIdx.x, static_cast<long>(gridDim.x - chunks) * ST);
        return;
    }
    const int tid = threadIdx.x, base = blockIdx.x * CHUNK;
    if (tid < DIGITS) cnt[tid] = 0;
    __syncthreads();
    for (int i = tid; i < CHUNK && base + i < s.T; i += ST)
        atomicAdd(&cnt[key_of(src[base + i], s.vocab) >> (pass * s.bits) & ((1 << s.bits) - 1)], 1);
    __syncthreads();
    if (tid < DIGITS) counts[static_cast<long>(tid) * chunks + blockIdx.x] = cnt[tid];
}

__global__ __launch_bounds__(ST) void sort_place_k(Sort s, int pass, int chunks, const int* src_id, const int* src_at, const int* counts,
                                                   Tokens out) {
    __shared__ int cnt[WAVES][DIGITS], sums[WAVES], start[DIGITS];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, base = blockIdx.x * CHUNK;
    Ranks r;
    r.n = (min(s.T - base, CHUNK) + ST - 1) / ST;
    const int first = base + wave * 64 * r.n + lane;
    int id[SI], at[SI];
#pragma unroll
    for (int g = 0; g < SI; ++g) {
        const int i = first + 64 * g;
        const bool has = g < r.n && i < s.T;
        id[g] = has ? key_of(src_id[i], s.vocab) : -1;
        at[g] = has ? (src_at ? src_at[i] : i) : 0;
        r.digit[g] = has ? id[g] >> (pass * s.bits) & ((1 << s.bits) - 1) : -1;
    }
    block_offsets(r, s.bits, cnt, sums);
    // where this chunk's tokens of digit tid / 4 begin: the digits before it, and
    // the chunks before this one of the digit
    int all = 0, before = 0;
    for (int c = tid & 3; c < chunks; c += 4) {
        const int n = counts[static_cast<long>(tid >> 2) * chunks + c];
        all += n;
        before += c < static_cast<int>(blockIdx.x) ? n : 0;
    }
    all += __shfl_xor(all, 1);
    all += __shfl_xor(all, 2);
    before += __shfl_xor(before, 1);
    before += __shfl_xor(before, 2);
    int upto = all;  // over the wave's sixteen digits
#pragma unroll
    for (int o = 4; o < 64; o *= 2) {
        const int x = __shfl_up(upto, o);
        upto += lane >= o ? x : 0;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int from = upto - all + before;
    for (int i = 0; i < wave; ++i) from += sums[i];
    if ((tid & 3) == 0) start[tid >> 2] = from - cnt[0][tid >> 2];
    __syncthreads();
    place_all(r, cnt, [&](int g, int to) {
        to += start[r.digit[g]];
        out.id[to] = id[g];
        out.at[to] = at[g];
    });
}

// ─── sums ───

struct Sums {
    const int *id, *at;  // sorted
    int T, vocab, cols, piece, pieces, chunks;
    float scale, *table;
    bool add;   // the table's rows hold something to add to
    float* part;  // (pieces, 2, cols): a run that began before the piece, one that goes on behind it
};

// A wave walks a piece's tokens for 64 parts of a row, sixteen rows' loads at a
// time: 16381 rows of 1024 bf16 take 14.1 us (34 MB read), 8190 of 768
// floats 9.2 (25 read).
template <class T>
__global__ __launch_bounds__(ET) void embed_sums_k(Sums s, const T* __restrict__ dY, long rs, bool vec) {
    constexpr int E = PART<T>, N = 16;
    const int lane = threadIdx.x & 63;
    const long block = static_cast<long>(blockIdx.y) * gridDim.x + blockIdx.x;
    const long unit = block * (ET / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int piece = static_cast<int>(unit / s.chunks), chunk = static_cast<int>(unit - static_cast<long>(piece) * s.chunks);
    if (piece >= s.pieces) return;
    const int s0 = piece * s.piece, n = min(s.piece, s.T - s0);
    const int c = E * (64 * chunk + lane), nc = max(min(E, s.cols - c), 0);
    const int ids = lane < n ? s.id[s0 + lane] : s.vocab, ats = lane < n ? s.at[s0 + lane] : 0;
    const int prev = s0 > 0 ? s.id[s0 - 1] : -1, next = s0 + n < s.T ? s.id[s0 + n] : -1;
    float acc[E];
#pragma unroll
    for (int k = 0; k < E; ++k) acc[k] = 0.0f;
    int cur = __builtin_amdgcn_readlane(ids, 0);
    bool left = prev == cur;  // the run began before the piece
    const auto put = [&](bool right) __attribute__((always_inline)) {
        float* to;
        if (left || right) {
            to = s.part + (2L * piece + (left ? 0 : 1)) * s.cols + c;
        } else {
            to = s.table + static_cast<long>(cur) * s.cols + c;
#pragma unroll
            for (int i = 0; i < E; ++i) acc[i] *= s.scale;
            if (s.add)
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (i < nc) acc[i] += to[i];
        }
        if (nc == E && (s.cols & 3) == 0 && (reinterpret_cast<size_t>(to) & 15) == 0) {
#pragma unroll
            for (int i = 0; i < E; i += 4) *reinterpret_cast<f32x4*>(to + i) = f32x4{acc[i], acc[i + 1], acc[i + 2], acc[i + 3]};
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i)
                if (i < nc) to[i] = acc[i];
        }
    };
    for (int i0 = 0; i0 < n; i0 += N) {
        Part<T> f[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int i = min(i0 + j, n - 1);
            f[j] = load_part(dY + __builtin_amdgcn_readlane(ats, i) * rs + c, __builtin_amdgcn_readlane(ids, i) < s.vocab ? nc : 0, vec);
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            if (i0 + j >= n) break;
            const int id = __builtin_amdgcn_readlane(ids, i0 + j);
            if (id != cur) {
                put(false);
                cur = id;
                left = false;
#pragma unroll
                for (int k = 0; k < E; ++k) acc[k] = 0.0f;
            }
            if (id == s.vocab) return;  // what follows is outside the table
#pragma unroll
            for (int k = 0; k < E; ++k) acc[k] += static_cast<float>(f[j][k]);
        }
    }
    put(next == cur);
}

// The runs that cross pieces: block (boundary, columns) of the first boundary
// that a run crosses adds its partial rows, each of its waves a stretch of them,
// and the waves' sums in order.
__global__ __launch_bounds__(ET) void embed_join_k(Sums s) {
    constexpr int W = ET / 64;
    __shared__ f32x4 sum[W][64];
    const int p = blockIdx.x + 1, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int id = s.id[p * s.piece];
    if (id == s.vocab || s.id[p * s.piece - 1] != id) return;
    if (p > 1 && s.id[(p - 1) * s.piece - 1] == id) return;
    int last = p;  // the last piece whose first token is of the run
    for (int q = p + 1;; q += 64) {
        const bool in = q + lane < s.pieces && s.id[(q + lane) * s.piece] == id;
        const int more = __builtin_popcountll(__builtin_amdgcn_ballot_w64(in));
        last += more;
        if (more < 64) break;
    }
    // rows 0 (what the run began with) .. m - 1
    const int m = last - p + 2, r0 = static_cast<int>(static_cast<long>(m) * wave / W), r1 = static_cast<int>(static_cast<long>(m) * (wave + 1) / W);
    const int c = 256 * blockIdx.y + 4 * lane, nc = max(min(4, s.cols - c), 0);
    const bool vec = (s.cols & 3) == 0 && nc == 4;
    const auto row = [&](int r) __attribute__((always_inline)) {
        const float* from = s.part + (2L * (p - 1 + r) + (r == 0 ? 1 : 0)) * s.cols + c;
        f32x4 v = f32x4{};
        if (vec) return *reinterpret_cast<const f32x4*>(from);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i < nc) v[i] = from[i];
        return v;
    };
    f32x4 acc = f32x4{};
    int r = r0;
    for (; r + 8 <= r1; r += 8) {
        f32x4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = row(r + i);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc += v[i];
    }
    for (; r < r1; ++r) acc += row(r);
    sum[wave][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
    for (int w = 1; w < W; ++w) acc += sum[w][lane];
    float* to = s.table + static_cast<long>(id) * s.cols + c;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < nc) to[i] = s.add ? to[i] + s.scale * acc[i] : s.scale * acc[i];
}

template <class T>
void lookup(kdec_ctx* ctx, const void* table, long t_rs, const int* ids, void* Y, long y_rs, int rows, int vocab, int cols,
            float scale) {
    constexpr int E = PART<T>;
    const auto ok = [&](const void* p, long rs) { return reinterpret_cast<size_t>(p) % 16 == 0 && rs % E == 0; };
    const bool vec = cols % E == 0 && ok(table, t_rs) && ok(Y, y_rs);
    const unsigned groups = static_cast<unsigned>(cdiv(cols, E));
    const long threads = static_cast<long>(rows) * groups;
    long blocks = cdiv(threads, ET * J);
    if (blocks > 64L * ctx->num_cus) blocks = 64L * ctx->num_cus;
    hipLaunchKernelGGL(embed_k<T>, dim3(static_cast<unsigned>(blocks)), dim3(ET), 0, ctx->stream, static_cast<const T*>(table), t_rs, ids,
                       static_cast<T*>(Y), y_rs, rows, vocab, cols, groups, vec, scale);
}

}  // namespace
}  // namespace kdec

using namespace kdec;

extern "C" {

int kdec_embed_fwd(kdec_ctx* ctx, int dtype, const void* table, long t_rs, const int* ids, int T, int vocab, int cols, float scale,
                   void* Y, long y_rs) {
    if (!ctx) return KDEC_EINVAL;
    const DeviceScope device(ctx);
    KDEC_CHECK(ctx, dtype == KDEC_F32 || dtype == KDEC_BF16, "kdec_embed_fwd: unknown type");
    KDEC_CHECK(ctx, T >= 0 && vocab >= 0 && cols >= 0 && cols <= 0x7FFFFFF0, "kdec_embed_fwd: bad sizes");
    if (T == 0 || cols == 0) return KDEC_OK;
    KDEC_CHECK(ctx, ids && Y && (table || vocab == 0), "kdec_embed_fwd: null tensor");
    KDEC_CHECK(ctx, T == 1 || y_rs >= cols, "kdec_embed_fwd: row stride of Y too small");
    const int es = dtype == KDEC_F32 ? 4 : 2;
    ProfScope ps(ctx, "embed", 0.0, 2.0 * es * T * static_cast<double>(cols));
    if (dtype == KDEC_F32) lookup<float>(ctx, table, t_rs, ids, Y, y_rs, T, vocab, cols, scale);
    else lookup<bf16>(ctx, table, t_rs, ids, Y, y_rs, T, vocab, cols, scale);
    return launch_check(ctx, "kdec_embed_fwd");
}

int kdec_embed_bwd(kdec_ctx* ctx, int dtype, const void* dY, long dy_rs, const int* ids, int T, int vocab, int cols, float scale,
                   float* dtable, float beta) {
    if (!ctx) return KDEC_EINVAL;
    const DeviceScope device(ctx);
    KDEC_CHECK(ctx, dtype == KDEC_F32 || dtype == KDEC_BF16, "kdec_embed_bwd: unknown type");
    KDEC_CHECK(ctx, T >= 0 && T <= INT_MAX - CHUNK && vocab >= 0 && vocab <= INT_MAX - 2 * DIGITS && cols >= 0 && cols <= 0x7FFFFF00,
               "kdec_embed_bwd: bad sizes");
    if (vocab == 0 || cols == 0) return KDEC_OK;
    KDEC_CHECK(ctx, dtable && (T == 0 || (dY && ids)), "kdec_embed_bwd: null tensor");
    const int es = dtype == KDEC_F32 ? 4 : 2, el = 16 / es;
    const long n = static_cast<long>(vocab) * cols;
    ProfScope ps(ctx, "embed", 0.0, es * static_cast<double>(T) * cols + 4.0 * n);

    const auto bits_of = [](unsigned last) { return last ? 32 - __builtin_clz(last) : 0; };  // of the numbers 0 .. last
    const int chunks = static_cast<int>(cdiv(T, CHUNK));
    Sort so{ids, T, vocab, 0, dtable, n, beta};
    // Ids of a block of the one-launch sort: a block a CU, up to a digit's. Past
    // eight blocks a CU, each of which looks at all tokens, the radix sort is
    // quicker (8192 tokens of 64 columns, ids of 500000: 77 us for 90, of a million
    // 131 for 106), as past what a block holds.
    long per = cdiv(static_cast<long>(vocab) + 1, static_cast<long>(ctx->num_cus));
    if (per > DIGITS) per = DIGITS;
    const dim3 ranges(static_cast<unsigned>(cdiv(static_cast<long>(vocab) + 1, per)));
    const bool one = chunks <= 1 && ranges.x <= 8u * static_cast<unsigned>(ctx->num_cus);
    // Few tokens: the sums in the sort's launch (512 tokens as texts have them, 181
    // ids, 512 columns, forward and backward 16.5 us, in launches of their own 21.8;
    // all of one id, 1024 columns, 36 and 22).
    if (one && T <= FEW) {
        so.bits = bits_of(static_cast<unsigned>(per - 1));
        if (dtype == KDEC_F32)
            hipLaunchKernelGGL((sort_range_k<float, true>), ranges, dim3(ST), 0, ctx->stream, so, static_cast<int>(per), Tokens{},
                               static_cast<const float*>(dY), dy_rs, cols, scale);
        else
            hipLaunchKernelGGL((sort_range_k<bf16, true>), ranges, dim3(ST), 0, ctx->stream, so, static_cast<int>(per), Tokens{},
                               static_cast<const bf16*>(dY), dy_rs, cols, scale);
        return launch_check(ctx, "kdec_embed_bwd");
    }
    // Blocks that clear or scale the table beside the first count's, or alone.
    long fill = beta == 1.0f ? 0 : cdiv(n, 16L * ST);
    if (fill > 2L * ctx->num_cus) fill = 2L * ctx->num_cus;
    if (T == 0) {
        if (fill)
            hipLaunchKernelGGL(sort_count_k, dim3(static_cast<unsigned>(fill)), dim3(ST), 0, ctx->stream, so, 0, 0, ids, nullptr);
        return launch_check(ctx, "kdec_embed_bwd");
    }
    Sums s{};
    s.T = T;
    s.vocab = vocab;
    s.cols = cols;
    s.chunks = static_cast<int>(cdiv(cols, 64 * el));
    // Tokens of a piece: a piece leaves up to two partial rows, eight waves a CU are
    // what the loads need (the two cases above with pieces of 8, 16 and 32, sums and
    // join: 23.5 us, 20.0, 20.9 and 14.3, 14.1, 18.3).
    s.piece = 64;
    while (s.piece > 16 && cdiv(T, s.piece) * s.chunks < 8L * ctx->num_cus) s.piece /= 2;
    s.pieces = static_cast<int>(cdiv(T, s.piece));
    s.scale = scale;
    s.table = dtable;
    s.add = beta != 0.0f;
    const long units = static_cast<long>(s.pieces) * s.chunks;
    // Blocks of the sums: past GX in rows of them, so that what a call takes is a
    // matter of memory, and what no launch takes is refused before any is asked for.
    constexpr long GX = 1 << 16;
    const long blocks = cdiv(units, ET / 64);
    const dim3 grid(static_cast<unsigned>(blocks < GX ? blocks : GX), static_cast<unsigned>(cdiv(blocks, GX)));
    KDEC_CHECK(ctx, cdiv(cols, 256) <= 65535, "kdec_embed_bwd: too many columns");
    KDEC_CHECK(ctx, cdiv(blocks, GX) <= 65535 && grid_holds(s.pieces, ET), "kdec_embed_bwd: too many tokens");
    int bits = bits_of(static_cast<unsigned>(vocab));
    const int passes = (bits + 7) / 8;
    const bool two = !one && passes > 1;  // passes that read what the last one wrote
    const size_t part = cdiv(static_cast<long>(s.pieces) * 2 * cols, 4) * 4, ints = cdiv(T, 4) * 4;
    Workspace ws(ctx, (part + (two ? 4 : 2) * ints + static_cast<size_t>(DIGITS) * chunks) * 4);
    if (!ws.p) return KDEC_ENOMEM;
    s.part = ws.as<float>();
    int* room = reinterpret_cast<int*>(s.part + part);
    const Tokens to[2] = {{room, room + ints}, {room + 2 * ints, room + 3 * ints}};
    int* counts = room + (two ? 4 : 2) * ints;
    Tokens from{const_cast<int*>(ids), nullptr};
    if (one) {
        so.bits = bits_of(static_cast<unsigned>(per - 1));
        from = to[0];
        hipLaunchKernelGGL((sort_range_k<float, false>), ranges, dim3(ST), 0, ctx->stream, so, static_cast<int>(per), from, nullptr, 0, cols,
                           scale);
    } else {
        so.bits = (bits + passes - 1) / passes;
        for (int p = 0; p < passes; ++p) {
            hipLaunchKernelGGL(sort_count_k, dim3(static_cast<unsigned>(chunks + (p == 0 ? fill : 0))), dim3(ST), 0, ctx->stream, so, p,
                               chunks, from.id, counts);
            hipLaunchKernelGGL(sort_place_k, dim3(static_cast<unsigned>(chunks)), dim3(ST), 0, ctx->stream, so, p, chunks, from.id, from.at,
                               counts, to[p & 1]);
            from = to[p & 1];
        }
    }
    s.id = from.id;
    s.at = from.at;
    const bool vec = cols % el == 0 && reinterpret_cast<size_t>(dY) % 16 == 0 && dy_rs % el == 0;
    if (dtype == KDEC_F32)
        hipLaunchKernelGGL(embed_sums_k<float>, grid, dim3(ET), 0, ctx->stream, s, static_cast<const float*>(dY), dy_rs, vec);
    else
        hipLaunchKernelGGL(embed_sums_k<bf16>, grid, dim3(ET), 0, ctx->stream, s, static_cast<const bf16*>(dY), dy_rs, vec);
    if (s.pieces > 1)
        hipLaunchKernelGGL(embed_join_k, dim3(static_cast<unsigned>(s.pieces - 1), static_cast<unsigned>(cdiv(cols, 256))), dim3(ET), 0,
                           ctx->stream, s);
    return launch_check(ctx, "kdec_embed_bwd");
}

}  // extern "C"
