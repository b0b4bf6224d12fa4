// Embedding lookup on gfx950, and the gradient of its table by sorted tokens.
//
// Forward: Y[t] = scale * table[ids[t]], a row of zeros where the id is outside
// the table. One lane copies eight columns; bound by memory.
//
// Backward: dtable[v] = beta dtable[v] + scale * sum of dY[t] over the tokens t
// of id v, in ascending t. Tokens are sorted by id first (a stable radix sort:
// ranks within 64 tokens from ballots over the digit's bits, counts by wave and
// digit, one scan), cut into pieces of a fixed number of sorted tokens, and a
// wave walks a piece for a stretch of columns: a run of one id that lies inside
// the piece goes to the table, what a run leaves at a piece's ends goes to a
// partial row, and the partial rows of a run are added in the pieces' order.
// So every piece is the same work however often an id occurs, and every sum has
// one order. The table is cleared (or scaled by beta) by the blocks that the
// sort leaves idle.
#include "kdec_frag.hpp"
#include "kdec_internal.hpp"

#include <climits>

namespace kdec {
namespace {

constexpr int ET = 256;         // threads of the copying and summing blocks
constexpr int ST = 1024;        // threads of a sorting block
constexpr int SI = 16;          // tokens a thread of it holds at most
constexpr int CHUNK = ST * SI;  // tokens a sorting block holds
constexpr int WAVES = ST / 64;
constexpr int DIGITS = 256;

template <class T>
__global__ __launch_bounds__(ET) void embed_k(const T* table, long t_rs, const int* ids, T* Y, long y_rs, int rows, int vocab,
                                              int cols, unsigned groups, bool vec, float scale) {
    const unsigned long long total = static_cast<unsigned long long>(rows) * groups;
    for (unsigned long long e = static_cast<unsigned long long>(blockIdx.x) * ET + threadIdx.x; e < total;
         e += static_cast<unsigned long long>(gridDim.x) * ET) {
        const unsigned row = static_cast<unsigned>(e / groups), g = static_cast<unsigned>(e - static_cast<unsigned long long>(row) * groups);
        const int c = 8 * static_cast<int>(g), n = min(8, cols - c), id = ids[row];
        Frag<T> f = Frag<T>{};
        if (static_cast<unsigned>(id) < static_cast<unsigned>(vocab)) f = load8(table + id * t_rs + c, n, vec);
        T* y = Y + row * y_rs + c;
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = static_cast<T>(scale * static_cast<float>(f[i]));
        if (vec) {
            *reinterpret_cast<Frag<T>*>(y) = f;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < n) y[i] = f[i];
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

__device__ inline void begin_table(const Sort& s, long block, long blocks) {
    if (s.beta == 1.0f) return;
    const bool vec = reinterpret_cast<size_t>(s.table) % 16 == 0;
    const long quads = vec ? s.n / 4 : 0, step = blocks * blockDim.x, first = block * blockDim.x + threadIdx.x;
    f32x4* q = reinterpret_cast<f32x4*>(s.table);
    if (s.beta == 0.0f) {
        for (long i = first; i < quads; i += step) q[i] = f32x4{};
        for (long i = 4 * quads + first; i < s.n; i += step) s.table[i] = 0.0f;
    } else {
        for (long i = first; i < quads; i += step) q[i] *= s.beta;
        for (long i = 4 * quads + first; i < s.n; i += step) s.table[i] *= s.beta;
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
    for (int b = 0; b < bits; ++b) {
        const unsigned long long one = __builtin_amdgcn_ballot_w64(digit >> b & 1);
        same &= (digit >> b & 1) ? one : ~one;
    }
    const int before = __builtin_popcountll(same & ((1ull << lane) - 1));
    place = before | __builtin_popcountll(same) << 8;
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
    int upto = sum;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const int x = __shfl_up(upto, o);
        upto += lane >= o ? x : 0;
    }
    if (lane == 63) sums[wave] = upto;
    __syncthreads();
    int at = upto - sum;
    for (int i = 0; i < wave; ++i) at += sums[i];
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
        if (g < r.n) {
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

// One block sorts up to CHUNK tokens, digit by digit, through shared memory.
// The other blocks begin the table.
__global__ __launch_bounds__(ST) void sort_one_k(Sort s, int passes, Tokens out) {
    __shared__ int cnt[WAVES][DIGITS], sums[WAVES];
    __shared__ int sid[CHUNK], sat[CHUNK];
    if (blockIdx.x > 0) {
        begin_table(s, blockIdx.x - 1, gridDim.x - 1);
        return;
    }
    const int tid = threadIdx.x;
    Ranks r;
    r.n = (s.T + ST - 1) / ST;
    const int first = (tid >> 6) * 64 * r.n + (tid & 63);
    int id[SI], at[SI];
#pragma unroll
    for (int g = 0; g < SI; ++g) {
        at[g] = first + 64 * g;
        id[g] = g < r.n && at[g] < s.T ? key_of(s.ids[at[g]], s.vocab) : -1;
    }
    for (int p = 0; p < passes; ++p) {
#pragma unroll
        for (int g = 0; g < SI; ++g) r.digit[g] = id[g] < 0 ? -1 : id[g] >> (p * s.bits) & ((1 << s.bits) - 1);
        block_offsets(r, s.bits, cnt, sums);
        place_all(r, cnt, [&](int g, int to) {
            sid[to] = id[g];
            sat[to] = at[g];
        });
        __syncthreads();
#pragma unroll
        for (int g = 0; g < SI; ++g)
            if (g < r.n && first + 64 * g < s.T) {
                id[g] = sid[first + 64 * g];
                at[g] = sat[first + 64 * g];
            }
        __syncthreads();
    }
#pragma unroll
    for (int g = 0; g < SI; ++g)
        if (g < r.n && first + 64 * g < s.T) {
            out.id[first + 64 * g] = id[g];
            out.at[first + 64 * g] = at[g];
        }
}

// More tokens: a digit's counts by chunk, then every chunk's tokens to their
// places. counts[digit * chunks + chunk].
__global__ __launch_bounds__(ST) void sort_count_k(Sort s, int pass, int chunks, const int* src, int* counts) {
    __shared__ int cnt[DIGITS];
    if (static_cast<int>(blockIdx.x) >= chunks) {
        begin_table(s, blockIdx.x - chunks, gridDim.x - chunks);
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

// A wave walks a piece's tokens for 512 columns, eight rows' loads at a time.
template <class T>
__global__ __launch_bounds__(ET) void embed_sums_k(Sums s, const T* dY, long rs, bool vec) {
    const int lane = threadIdx.x & 63;
    const long unit = static_cast<long>(blockIdx.x) * (ET / 64) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int piece = static_cast<int>(unit / s.chunks), chunk = static_cast<int>(unit - static_cast<long>(piece) * s.chunks);
    if (piece >= s.pieces) return;
    const int s0 = piece * s.piece, n = min(s.piece, s.T - s0);
    const int c = 512 * chunk + 8 * lane, nc = max(min(8, s.cols - c), 0);
    const int ids = lane < n ? s.id[s0 + lane] : s.vocab, ats = lane < n ? s.at[s0 + lane] : 0;
    const int prev = s0 > 0 ? s.id[s0 - 1] : -1, next = s0 + n < s.T ? s.id[s0 + n] : -1;
    f32x8 acc = f32x8{};
    int cur = __builtin_amdgcn_readlane(ids, 0);
    bool left = prev == cur;  // the run began before the piece
    const auto put = [&](bool right) __attribute__((always_inline)) {
        float* to;
        if (left || right) {
            to = s.part + (2L * piece + (left ? 0 : 1)) * s.cols + c;
        } else {
            to = s.table + static_cast<long>(cur) * s.cols + c;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] *= s.scale;
            if (s.add)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (i < nc) acc[i] += to[i];
        }
        if (nc == 8 && (s.cols & 3) == 0 && (reinterpret_cast<size_t>(to) & 15) == 0) {
            *reinterpret_cast<f32x4*>(to) = acc.lo;
            *reinterpret_cast<f32x4*>(to + 4) = acc.hi;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (i < nc) to[i] = acc[i];
        }
    };
    for (int i0 = 0; i0 < n; i0 += 8) {
        Frag<T> f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int i = min(i0 + j, n - 1);
            f[j] = load8(dY + __builtin_amdgcn_readlane(ats, i) * rs + c, __builtin_amdgcn_readlane(ids, i) < s.vocab ? nc : 0, vec);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (i0 + j >= n) break;
            const int id = __builtin_amdgcn_readlane(ids, i0 + j);
            if (id != cur) {
                put(false);
                cur = id;
                left = false;
                acc = f32x8{};
            }
            if (id == s.vocab) return;  // what follows is outside the table
#pragma unroll
            for (int k = 0; k < 8; ++k) acc[k] += static_cast<float>(f[j][k]);
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
    const int el = 16 / static_cast<int>(sizeof(T));  // elements per 16 bytes
    const auto ok = [&](const void* p, long rs) { return reinterpret_cast<size_t>(p) % 16 == 0 && rs % el == 0; };
    const bool vec = cols % 8 == 0 && ok(table, t_rs) && ok(Y, y_rs);
    const unsigned groups = static_cast<unsigned>(cdiv(cols, 8));
    long blocks = cdiv(static_cast<long>(rows) * groups, ET);
    if (blocks > 32L * ctx->num_cus) blocks = 32L * ctx->num_cus;
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
    KDEC_CHECK(ctx, dtype == KDEC_F32 || dtype == KDEC_BF16, "kdec_embed_bwd: unknown type");
    KDEC_CHECK(ctx, T >= 0 && T <= INT_MAX - CHUNK && vocab >= 0 && vocab < INT_MAX && cols >= 0 && cols <= 0x7FFFFF00,
               "kdec_embed_bwd: bad sizes");
    if (vocab == 0 || cols == 0) return KDEC_OK;
    KDEC_CHECK(ctx, dtable && (T == 0 || (dY && ids)), "kdec_embed_bwd: null tensor");
    const int es = dtype == KDEC_F32 ? 4 : 2, el = 16 / es;
    const long n = static_cast<long>(vocab) * cols;
    ProfScope ps(ctx, "embed", 0.0, es * static_cast<double>(T) * cols + 4.0 * n);

    int bits = 32 - __builtin_clz(static_cast<unsigned>(vocab));  // of the keys 0 .. vocab
    const int passes = (bits + 7) / 8;
    bits = (bits + passes - 1) / passes;
    const int chunks = static_cast<int>(cdiv(T, CHUNK));
    Sums s{};
    s.T = T;
    s.vocab = vocab;
    s.cols = cols;
    s.piece = 32;
    s.pieces = static_cast<int>(cdiv(T, s.piece));
    s.chunks = static_cast<int>(cdiv(cols, 512));
    s.scale = scale;
    s.table = dtable;
    s.add = beta != 0.0f;
    const long units = static_cast<long>(s.pieces) * s.chunks;
    KDEC_CHECK(ctx, cdiv(units, ET / 64) < INT_MAX && cdiv(cols, 256) <= 65535, "kdec_embed_bwd: bad sizes");
    const bool two = chunks > 1 && passes > 1;  // passes that read what the last one wrote
    const size_t part = cdiv(static_cast<long>(s.pieces) * 2 * cols, 4) * 4, ints = cdiv(T, 4) * 4;
    Workspace ws(ctx, (part + (two ? 4 : 2) * ints + static_cast<size_t>(DIGITS) * chunks) * 4);
    if (!ws.p) return KDEC_ENOMEM;
    s.part = ws.as<float>();
    int* room = reinterpret_cast<int*>(s.part + part);
    const Tokens to[2] = {{room, room + ints}, {room + 2 * ints, room + 3 * ints}};
    int* counts = room + (two ? 4 : 2) * ints;

    Sort so{ids, T, vocab, bits, dtable, n, beta};
    long fill = beta == 1.0f ? 0 : cdiv(n, 16L * ST);  // blocks beside the sort's
    if (fill > ctx->num_cus - 1) fill = ctx->num_cus - 1;
    Tokens from{const_cast<int*>(ids), nullptr};
    if (chunks <= 1) {
        from = to[0];
        hipLaunchKernelGGL(sort_one_k, dim3(static_cast<unsigned>(1 + fill)), dim3(ST), 0, ctx->stream, so, passes, from);
    }
    for (int p = 0; chunks > 1 && p < passes; ++p) {
        hipLaunchKernelGGL(sort_count_k, dim3(static_cast<unsigned>(chunks + (p == 0 ? fill : 0))), dim3(ST), 0, ctx->stream, so, p, chunks,
                           from.id, counts);
        hipLaunchKernelGGL(sort_place_k, dim3(static_cast<unsigned>(chunks)), dim3(ST), 0, ctx->stream, so, p, chunks, from.id, from.at,
                           counts, to[p & 1]);
        from = to[p & 1];
    }
    s.id = from.id;
    s.at = from.at;
    if (T > 0) {
        const bool vec = cols % 8 == 0 && reinterpret_cast<size_t>(dY) % 16 == 0 && dy_rs % el == 0;
        const dim3 grid(static_cast<unsigned>(cdiv(units, ET / 64)));
        if (dtype == KDEC_F32)
            hipLaunchKernelGGL(embed_sums_k<float>, grid, dim3(ET), 0, ctx->stream, s, static_cast<const float*>(dY), dy_rs, vec);
        else
            hipLaunchKernelGGL(embed_sums_k<bf16>, grid, dim3(ET), 0, ctx->stream, s, static_cast<const bf16*>(dY), dy_rs, vec);
        if (s.pieces > 1)
            hipLaunchKernelGGL(embed_join_k, dim3(static_cast<unsigned>(s.pieces - 1), static_cast<unsigned>(cdiv(cols, 256))), dim3(ET), 0,
                               ctx->stream, s);
    }
    return launch_check(ctx, "kdec_embed_bwd");
}

}  // extern "C"
