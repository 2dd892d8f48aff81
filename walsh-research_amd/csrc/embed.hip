// Embedding lookup with scaling and dropout, and its gradient:
//     y_r = scale keep(r) W[t_r]          dW_v = scale sum over r with t_r = v of keep(r) gy_r
// with keep() the mask and factor of dropout (rows8.h).  A token outside the
// vocabulary gives a row of NaN and adds to no gradient; nor does padding_idx.
//
// The gradient adds the rows of a token in float32 in a fixed order, which
// depends on the call's tokens and sizes (where a long row is cut): equal calls
// give equal bits.  Three kernels:
//   sort   a workgroup takes a range of up to 256 tokens and walks all N: it
//          counts those below its range, which is where its part of the sorted
//          order begins (no workgroup waits for another), and lists those in
//          it, to count and place them.  What every workgroup repeats, ten
//          instructions for 64 tokens, costs less than a launch would: 6.5 us for
//          8,192 tokens, 8.6 for 16,384, 20 for 65,536, 4 of them the launch.
//          The range with the most tokens places them alone: with frequent
//          tokens side by side in the vocabulary 11, 19 and 72 us.
//   rows   zeros where a token does not occur; else the sum of its tokens' rows,
//          a lane 8 columns, up to 32 of them.  Longer rows are cut where the
//          sorted order is, every 32 places (embed_most), and their pieces summed
//          into a workspace.
//   join   adds the pieces of each long row, in a fixed order.
// Bound by memory: 50,257 x 4,096 bf16 from 16,384 rows (546 MB) take 93 us for
// the rows, 5.9 TB/s, x 512 float32 from 8,192 (120 MB) 18 us, of 108 and 29 in
// all; a character model's 65 x 768 from 16,384 rows 21 us, all of it latency.
// The lookup of 16,384 x 4,096 takes 32 us, of 64 rows 3.0.
#include <type_traits>

#include "rows8.h"

namespace walsh {

constexpr int kEmWaves = 16, kEmRange = 256;

struct EmbedArgs {
    const int64_t *tokens;
    const void *w;
    void *y;
    int64_t V, ldw, ldy;
    int C;
    Blocks g;
    Drop d;
    float f;
};

// Stores of bf16 are streamed, as in dropout (lookup and gradient of 16,384 x
// 4,096 one after the other 142 us instead of 160).
template <typename TW, typename TY, bool DROP, int U>
__global__ __launch_bounds__(256) void embed_kernel(EmbedArgs a) {
    const uint32_t first = blockIdx.x * (256u * U);
    const DropBits bits(a.d);
    BlockAt at[U];
    float v[U][8];
    int64_t t[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
        at[j] = block_at(a.g, first, 256u * j + threadIdx.x);
        t[j] = at[j].row < a.g.rows ? a.tokens[at[j].row] : -1;
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
        const int c = 8 * (int)at[j].col;
        if ((uint64_t)t[j] < (uint64_t)a.V) {
            load8((const TW *)a.w + t[j] * a.ldw + c, a.C - c, v[j]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] = NAN;
        }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
        if (at[j].row < a.g.rows) {
            const int c = 8 * (int)at[j].col;
            if (DROP && (uint64_t)t[j] < (uint64_t)a.V) bits.apply(v[j], at[j].row, at[j].col);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] *= a.f;
            store8<true>((TY *)a.y + at[j].row * a.ldy + c, a.C - c, v[j]);
        }
    }
}

// ---------------------------------------------------------------- gradient
// order[start[v] .. start[v + 1]): the places of token v, in order; token[]: v there.
struct EmbedSort {
    const int64_t *tokens;
    uint32_t V;
    int N, bits;                       // a workgroup's range: 2^bits tokens
    int *start, *order, *token;
};

// A wavefront walks a stretch of steps of 64 tokens, the loads of 8 together,
// and lists those of the range (few of 64, mostly) in LDS, so that counting and
// placing take 64 of them at once.  A list that overflows is counted and begun
// anew, and the stretch walked again for the placing.
constexpr int kEmLoads = 8, kEmList = 1024;
constexpr uint32_t kEmNone = 0xffffffffu;

struct EmbedSortShared {
    int count[kEmWaves][kEmRange], total[kEmRange], below[kEmWaves], sums[kEmRange / 64];
    uint32_t list[kEmWaves][kEmList];  // place in the stretch << 8 | token relative to the range
};

// For a lane whose token is in the range, among the step's lanes with the same
// token: the first, how many lie before the lane, and how many there are.
// Token by token, or bit by bit where there are many.
struct EmbedSame {
    int first, before, n;
};
__device__ __forceinline__ int lanes_below(uint64_t m) {
    return __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0));
}
__device__ __forceinline__ EmbedSame embed_same(uint32_t d, uint64_t left, int bits) {
    EmbedSame s{-1, 0, 0};
    for (int k = 0; left && k < 4; ++k) {
        const int first = __builtin_ctzll(left);
        const bool is = d == (uint32_t)__builtin_amdgcn_readlane((int)d, first);
        const uint64_t m = __ballot(is);
        s = is ? EmbedSame{first, lanes_below(m), (int)__popcll(m)} : s;
        left &= ~m;
    }
    if (left) {
        const bool mine = left >> (threadIdx.x & 63) & 1;
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot(d >> b & 1);
            left &= d >> b & 1 ? set : ~set;
        }
        s = mine ? EmbedSame{(int)__builtin_ctzll(left), lanes_below(left), (int)__popcll(left)} : s;
    }
    return s;
}

__global__ __launch_bounds__(64 * kEmWaves) void embed_sort_kernel(EmbedSort a) {
    extern __shared__ __align__(16) unsigned char em_smem[];
    EmbedSortShared &sh = *(EmbedSortShared *)em_smem;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t lo = blockIdx.x << a.bits, range = min(1u << a.bits, a.V - lo);
    const int steps = (a.N + 64 * kEmWaves - 1) / (64 * kEmWaves);
    const int from = wave * steps * 64, to = min(a.N, from + steps * 64);
    uint32_t *list = sh.list[wave];
    int below = 0, n = 0;
    bool whole = true;
    auto walk = [&](auto flush) {
        below = n = 0;
        uint64_t next[kEmLoads];
        auto load = [&](int i0) {
#pragma unroll
            for (int j = 0; j < kEmLoads; ++j) {
                next[j] = ~0ull;
                if (i0 + 64 * j + lane < to) next[j] = a.tokens[i0 + 64 * j + lane];
            }
        };
        load(from);
        for (int i0 = from; i0 < to; i0 += 64 * kEmLoads) {
            uint64_t t[kEmLoads];
#pragma unroll
            for (int j = 0; j < kEmLoads; ++j) t[j] = next[j];
            load(i0 + 64 * kEmLoads);
            if (n > kEmList - 64 * kEmLoads) {
                flush(n);
                n = 0, whole = false;
            }
#pragma unroll
            for (int j = 0; j < kEmLoads; ++j) {
                const uint32_t x = t[j] >> 32 ? kEmNone : (uint32_t)t[j], d = x - lo;
                below += __popcll(__ballot(x < lo));
                const uint64_t in = __ballot(d < range);
                if (!in) continue;
                if (d < range) list[n + lanes_below(in)] = (uint32_t)(i0 - from + 64 * j + lane) << 8 | d;
                n += __popcll(in);
            }
        }
        flush(n);
    };
    auto tally = [&](int m) {
        wave_lds_fence();
        for (int g = 0; g < m; g += 64) {
            const uint32_t d = g + lane < m ? list[g + lane] & 0xffu : kEmNone;
            // (the first lane's token at once: a frequent one would go one by one)
            const bool is = d == (uint32_t)__builtin_amdgcn_readfirstlane((int)d);
            const int c = __popcll(__ballot(is));
            if (is ? lane == 0 : d != kEmNone) atomicAdd(&sh.count[wave][d], is ? c : 1);
        }
        wave_lds_fence();
    };
    auto place = [&](int m) {
        wave_lds_fence();
        for (int g = 0; g < m; g += 64) {
            const bool there = g + lane < m;
            const uint32_t v = there ? list[g + lane] : 0, d = there ? v & 0xffu : kEmNone;
            const EmbedSame same = embed_same(d, __ballot(there), a.bits);
            int at = 0;                // (a wavefront's LDS operations keep their order)
            if (same.first == lane) at = sh.total[d] + atomicAdd(&sh.count[wave][d], same.n);
            at = __shfl(at, same.first & 63) + same.before;
            if (there) {
                a.order[at] = from + (int)(v >> 8);
                a.token[at] = (int)(lo + d);
            }
        }
        wave_lds_fence();
    };
    for (int i = tid; i < kEmWaves * kEmRange; i += 64 * kEmWaves) (&sh.count[0][0])[i] = 0;
    __syncthreads();
    walk(tally);
    if (lane == 0) sh.below[wave] = below;
    __syncthreads();
    // where each wavefront's tokens of each value go
    int mine = 0, incl = 0;
    if (tid < kEmRange) {
#pragma unroll
        for (int w = 0; w < kEmWaves; ++w) {
            const int c = sh.count[w][tid];
            sh.count[w][tid] = mine;
            mine += c;
        }
        incl = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 63) sh.sums[wave] = incl;
    }
    __syncthreads();
    if (tid < kEmRange) {
        int base = 0;
#pragma unroll
        for (int w = 0; w < kEmWaves; ++w) base += sh.below[w];
        for (int w = 0; w < wave; ++w) base += sh.sums[w];
        const int at = base + incl - mine;
        sh.total[tid] = at;
        if ((uint32_t)tid < range) a.start[lo + tid] = at;
        // the end of the last range is the end of all
        if ((uint32_t)tid == range - 1 && lo + range == a.V) a.start[a.V] = base + incl;
    }
    __syncthreads();
    if (whole) place(n);
    else walk(place);
}

struct EmbedBwd {
    const int *start, *order, *token;
    const void *gy;
    void *dw;
    float *parts;                      // [2 per chunk][C]: of the row that a chunk begins with, and ends with
    int64_t V, ldg, ldw;
    int pad;                           // a row that stays zeros (-1: none)
    int C, most;                       // most: tokens of a row that one lane adds, places of a chunk
    Blocks rows, places, chunks;       // rows of dW (16 bytes), places of the sorted order, chunks of those
    uint32_t chunk_groups, head_groups;
    Drop d;
    float f;
};

// Sum of the gradients at places s .. e of the sorted order: U rows' loads
// together, the places of the next U on their way.
template <typename TG, bool DROP>
__device__ __forceinline__ void embed_add(const EmbedBwd &a, const DropBits &bits, int s, int e, uint32_t col, float (&acc)[8]) {
    constexpr int U = 4;
    const int c = 8 * (int)col;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    if (s >= e) return;
    const TG *g = (const TG *)a.gy + c;
    int r[U];
#pragma unroll
    for (int j = 0; j < U; ++j) r[j] = a.order[min(s + j, e - 1)];
    for (int k = s; k < e; k += U) {
        int now[U];
#pragma unroll
        for (int j = 0; j < U; ++j) now[j] = r[j];
        float v[8];
        if (a.C - c >= 8) {
            Raw8<TG> raw[U];
#pragma unroll
            for (int j = 0; j < U; ++j) raw[j].template load<false>(g + now[j] * a.ldg);
#pragma unroll
            for (int j = 0; j < U; ++j) r[j] = a.order[min(k + U + j, e - 1)];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                raw[j].unpack(v);
                if (DROP) bits.apply(v, now[j], col);
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] = k + j < e ? acc[i] + v[i] : acc[i];
            }
        } else {
#pragma unroll
            for (int j = 0; j < U; ++j) r[j] = a.order[min(k + U + j, e - 1)];
            for (int j = 0; j < min(U, e - k); ++j) {
                const int at = a.order[k + j];
                load8(g + at * a.ldg, a.C - c, v);
                if (DROP) bits.apply(v, at, col);
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] += v[i];
            }
        }
    }
}

// Workgroups by what they do, the longest chains of loads first:
//   chunks  the pieces of long rows
//   heads   the rows of tokens that occur, at the first place of each in the
//           sorted order: U blocks of a lane, their first tokens' rows loaded together
//   rest    zeros in the rows of those that do not: F blocks of 16 bytes of a lane
// SS: stores are streamed, of a gradient that the caches do not hold (50,257 x
// 4,096 bf16: 107 us instead of 129 in all, x 2,048 float32 100 instead of 132;
// with a pass over the gradient and the weights behind it 378 and 376 instead of
// 390 and 399).
template <typename TG, typename TW, bool DROP, int U, int F, bool SS> __global__ __launch_bounds__(256) void embed_rows_kernel(EmbedBwd a) {
    const DropBits bits(a.d);
    const int all = a.start[a.V];
    if (blockIdx.x < a.chunk_groups) {
        float acc[8];
        const BlockAt at = block_at(a.chunks, blockIdx.x * 256u, threadIdx.x);
        const int s = (int)at.row * a.most, e = min(all, s + a.most);
        if (at.row >= a.chunks.rows || s >= all) return;
        const int t0 = a.token[s], t1 = a.token[e - 1];
        const int c = 8 * (int)at.col, e0 = a.start[t0 + 1], s1 = a.start[t1];
        const bool long0 = t0 != a.pad && e0 - a.start[t0] > a.most;
        const bool long1 = t1 != t0 && t1 != a.pad && a.start[t1 + 1] - s1 > a.most;
#pragma unroll 1
        for (int k = 0; k < 2; ++k) {
            if (!(k ? long1 : long0)) continue;
            embed_add<TG, DROP>(a, bits, k ? s1 : s, k ? e : min(e, e0), at.col, acc);
            store8(a.parts + (2 * (int64_t)at.row + k) * a.C + c, a.C - c, acc);
        }
    } else if (blockIdx.x < a.chunk_groups + a.head_groups) {
        BlockAt at[U];
        int t[U], n[U], r[U];
        float v[U][8];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            at[j] = block_at(a.places, (blockIdx.x - a.chunk_groups) * (256u * U), 256u * j + threadIdx.x);
            const int k = min((int)at[j].row, all - 1);
            t[j] = r[j] = -1;
            if (k >= 0) {
                const int before = a.token[max(k - 1, 0)];
                t[j] = a.token[k], r[j] = a.order[k];
                if ((int)at[j].row >= all || (k > 0 && before == t[j])) t[j] = -1;
            }
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int c = 8 * (int)at[j].col;
            n[j] = 0;
            if (t[j] >= 0) {
                load8((const TG *)a.gy + r[j] * a.ldg + c, a.C - c, v[j]);
                n[j] = t[j] == a.pad ? 0 : a.start[t[j] + 1] - (int)at[j].row;
            }
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (n[j] < 1 || n[j] > a.most) continue;
            const int c = 8 * (int)at[j].col;
            if (DROP) bits.apply(v[j], r[j], at[j].col);
            if (n[j] > 1) {
                float acc[8];
                embed_add<TG, DROP>(a, bits, (int)at[j].row + 1, (int)at[j].row + n[j], at[j].col, acc);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j][i] += acc[i];
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) v[j][i] *= a.f;
            store8<SS>((TW *)a.dw + t[j] * a.ldw + c, a.C - c, v[j]);
        }
    } else {
        constexpr int E = 16 / sizeof(TW);
        BlockAt at[F];
        bool none[F];
#pragma unroll
        for (int j = 0; j < F; ++j) {
            at[j] = block_at(a.rows, (blockIdx.x - a.chunk_groups - a.head_groups) * (256u * F), 256u * j + threadIdx.x);
            const bool there = at[j].row < a.rows.rows;
            const uint32_t v = there ? at[j].row : 0;
            none[j] = there && (a.start[v + 1] == a.start[v] || (int)v == a.pad);
        }
#pragma unroll
        for (int j = 0; j < F; ++j) {
            const int c = E * (int)at[j].col;
            TW *p = (TW *)a.dw + at[j].row * a.ldw + c;
            if (!none[j]) continue;
            if (a.C - c >= E) {
                store16<SS>(p, u32x4{0, 0, 0, 0});
            } else {
                for (int i = 0; i < a.C - c; ++i) p[i] = 0;
            }
        }
    }
}

// A workgroup takes 32 blocks of the columns of a chunk's long row, if one
// begins there: its eighths take every eighth piece, then their sums are added.
constexpr int kEmSlab = 32;
template <typename TW> __global__ __launch_bounds__(256) void embed_join_kernel(EmbedBwd a, uint32_t slabs) {
    __shared__ float sum[8][8][kEmSlab + 1];
    const uint32_t chunk = blockIdx.x / slabs, slab = blockIdx.x - chunk * slabs;
    const int all = a.start[a.V], s = (int)chunk * a.most, e = min(all, s + a.most);
    if (s >= all) return;
    const int64_t t = a.token[e - 1];
    const int first = a.start[t], last = a.start[t + 1] - 1;
    if (first < s || last - first < a.most || t == a.pad) return;
    const int lane = threadIdx.x % kEmSlab, part = threadIdx.x / kEmSlab;
    const uint32_t col = slab * kEmSlab + lane;
    const bool there = col < a.chunks.per_row;
    const int c = 8 * (int)col, q1 = last / a.most;
    float acc[8] = {};
    if (there) {
#pragma unroll 4
        for (int q = (int)chunk + part; q <= q1; q += 8) {
            float v[8];
            load8(a.parts + (2 * (int64_t)q + (q == (int)chunk && first != s)) * a.C + c, a.C - c, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] += v[i];
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[part][i][lane] = acc[i];
    __syncthreads();
    if (part || !there) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
        for (int k = 1; k < 8; ++k) acc[i] += sum[k][i][lane];
        acc[i] *= a.f;
    }
    store8((TW *)a.dw + t * a.ldw + c, a.C - c, acc);
}

// Places of a chunk: fewer than 32 where that leaves too few lanes for the chip
// (16,384 x 768 in chunks of 16 instead of 32: 30 us instead of 34 in all, 4,096 x
// 384 in 8 17 instead of 26; 16,384 x 4,096 in 8 133 instead of 126), more
// where the longest row would have more than 1,024 pieces.
static int64_t embed_most(int64_t N, int64_t C) {
    int64_t most = 8;
    while (most < 32 && N * ceil_div(C, 8) > most * 131072) most *= 2;
    while (most * 1024 < N) most *= 2;
    return most;
}
static int64_t embed_chunks(int64_t N, int64_t C) { return ceil_div(N, embed_most(N, C)); }
// start, order, token, parts: each from a multiple of 16 bytes on
static int64_t embed_start_bytes(int64_t V) { return ceil_div(4 * (V + 1), 16) * 16; }
static int64_t embed_order_bytes(int64_t N) { return ceil_div(4 * N, 16) * 16; }

// Sizes that a call takes.
static bool embed_sizes(int64_t N, int64_t V, int64_t C) {
    return N >= 0 && C >= 0 && V >= 1 && C <= 0x7fffffff - 8 && N < 1 << 28 && V <= 0x7fffffff - 2048 &&
           N * ceil_div(C, 8) <= kMaxBlocks;
}

static int embed_check(const char *fn, int64_t N, int64_t V, int64_t C, int drop, const int64_t *seed, int64_t rng_stream,
                       int dt0, int dt1) {
    if (!embed_sizes(N, V, C))
        return set_error(WALSH_ENOTSUP, "%s: N=%lld tokens, V=%lld rows of C=%lld", fn, (long long)N, (long long)V, (long long)C);
    if (drop < 0 || drop > 65536 || rng_stream < 0 || rng_stream > 0xffffffffll)
        return set_error(WALSH_EINVAL, "%s: drop %d (0 to 65536), stream %lld (32 bits)", fn, drop, (long long)rng_stream);
    for (int dt : {dt0, dt1})
        if (dt != WALSH_F32 && dt != WALSH_BF16) return set_error(WALSH_ENOTSUP, "%s: dtype %d", fn, dt);
    if (drop && !seed) return set_error(WALSH_EINVAL, "%s: null pointer", fn);
    return WALSH_OK;
}

// f(a, b, drop) with two of float / uint16_t in place of the types and DROP.
template <typename F> static void embed_types(int dt0, int dt1, int drop, F f) {
    auto with = [&](auto x, auto y) {
        if (drop) f(x, y, std::integral_constant<bool, true>{});
        else f(x, y, std::integral_constant<bool, false>{});
    };
    if (dt0 == WALSH_BF16 && dt1 == WALSH_BF16) with(uint16_t{}, uint16_t{});
    else if (dt0 == WALSH_BF16) with(uint16_t{}, float{});
    else if (dt1 == WALSH_BF16) with(float{}, uint16_t{});
    else with(float{}, float{});
}

}  // namespace walsh

using namespace walsh;

WALSH_EXPORT int walsh_embedding_fwd(const int64_t *tokens, int64_t N, const void *weight, int64_t ldw, int64_t V, int64_t C,
                                     float scale, int drop, const int64_t *seed, int64_t rng_stream, void *y, int64_t ldy,
                                     int wdtype, int ydtype, void *stream) {
    const char *fn = "walsh_embedding_fwd";
    const int rc = embed_check(fn, N, V, C, drop, seed, rng_stream, wdtype, ydtype);
    if (rc) return rc;
    if (N == 0 || C == 0) return WALSH_OK;
    if (!tokens || !weight || !y) return set_error(WALSH_EINVAL, "%s: null pointer", fn);
    if ((V > 1 && ldw < C) || (N > 1 && ldy < C)) return set_error(WALSH_EINVAL, "%s: rows of %lld overlap", fn, (long long)C);
    constexpr int U = 2;
    const EmbedArgs a{tokens, weight, y, V, ldw, ldy, (int)C, make_blocks(N, C),
                      Drop{(const uint64_t *)seed, (uint32_t)rng_stream, (uint32_t)drop},
                      (float)((double)scale * kept_factor(drop))};
    const dim3 G((unsigned)ceil_div(N * a.g.per_row, 256 * U)), B(256);
    embed_types(wdtype, ydtype, drop, [&](auto w, auto o, auto d) {
        launch(embed_kernel<decltype(w), decltype(o), decltype(d)::value, U>, G, B, 0, (hipStream_t)stream, a);
    });
    return check_hip(hipGetLastError(), fn);
}

WALSH_EXPORT int64_t walsh_embedding_bwd_workspace_bytes(int64_t N, int64_t V, int64_t C) {
    if (!embed_sizes(N, V, C)) return 0;
    return embed_start_bytes(V) + 2 * embed_order_bytes(N) + 2 * embed_chunks(N, C) * C * 4;
}

WALSH_EXPORT int walsh_embedding_bwd(const int64_t *tokens, int64_t N, const void *gy, int64_t ldg, int64_t V, int64_t C,
                                     float scale, int64_t padding_idx, int drop, const int64_t *seed, int64_t rng_stream,
                                     void *dw, int64_t ldw, int gdtype, int wdtype, void *work, int64_t work_bytes,
                                     void *stream) {
    const char *fn = "walsh_embedding_bwd";
    int rc = embed_check(fn, N, V, C, drop, seed, rng_stream, gdtype, wdtype);
    if (rc) return rc;
    if (C == 0) return WALSH_OK;
    const Blocks rows = make_blocks(V, wdtype == WALSH_BF16 ? C : 2 * C), chunks = make_blocks(embed_chunks(N, C), C);
    if (V * (int64_t)rows.per_row > kMaxBlocks)
        return set_error(WALSH_ENOTSUP, "%s: V=%lld rows of C=%lld", fn, (long long)V, (long long)C);
    if ((N && (!tokens || !gy)) || !dw || !work) return set_error(WALSH_EINVAL, "%s: null pointer", fn);
    if ((V > 1 && ldw < C) || (N > 1 && ldg < C)) return set_error(WALSH_EINVAL, "%s: rows of %lld overlap", fn, (long long)C);
    if (work_bytes < walsh_embedding_bwd_workspace_bytes(N, V, C) || (uintptr_t)work % 16)
        return set_error(WALSH_EINVAL, "%s: workspace of %lld bytes (16-aligned), needs %lld", fn, (long long)work_bytes,
                         (long long)walsh_embedding_bwd_workspace_bytes(N, V, C));
    const hipStream_t s = (hipStream_t)stream;
    int *start = (int *)work, *order = (int *)((char *)work + embed_start_bytes(V));
    int *token = (int *)((char *)order + embed_order_bytes(N));
    float *parts = (float *)((char *)token + embed_order_bytes(N));
    // ranges small enough for a workgroup to every CU, where the vocabulary has as many
    int bits = 0;
    while (bits < 8 && ceil_div(V, 1 << bits) > device_info().cu_count) ++bits;
    const EmbedSort so{tokens, (uint32_t)V, (int)N, bits, start, order, token};
    launch(embed_sort_kernel, dim3((unsigned)ceil_div(V, 1 << bits)), dim3(64 * kEmWaves), (uint32_t)sizeof(EmbedSortShared), s,
           so);
    rc = check_hip(hipGetLastError(), fn);
    if (rc) return rc;
    constexpr int U = 1, F = 4;
    const uint32_t head_groups = (uint32_t)ceil_div(N * chunks.per_row, 256 * U);
    const uint32_t rest_groups = (uint32_t)ceil_div(V * rows.per_row, 256 * F);
    const int64_t most = embed_most(N, C);         // (up to so many tokens no row is long)
    const uint32_t chunk_groups = N > most ? (uint32_t)ceil_div((int64_t)chunks.rows * chunks.per_row, 256) : 0;
    const EmbedBwd a{start, order, token, gy, dw, parts, V, ldg, ldw,
                     (int)(padding_idx >= 0 && padding_idx < V ? padding_idx : -1), (int)C, (int)most, rows, make_blocks(N, C),
                     chunks, chunk_groups, head_groups, Drop{(const uint64_t *)seed, (uint32_t)rng_stream, (uint32_t)drop},
                     (float)((double)scale * kept_factor(drop))};
    embed_types(gdtype, wdtype, drop, [&](auto g, auto w, auto d) {
        const dim3 G(chunk_groups + head_groups + rest_groups), B(256);
        if (V * C * (int64_t)sizeof(w) >= kCacheBytes)
            launch(embed_rows_kernel<decltype(g), decltype(w), decltype(d)::value, U, F, true>, G, B, 0, s, a);
        else
            launch(embed_rows_kernel<decltype(g), decltype(w), decltype(d)::value, U, F, false>, G, B, 0, s, a);
    });
    rc = check_hip(hipGetLastError(), fn);
    if (rc || !chunk_groups) return rc;
    const uint32_t slabs = (uint32_t)ceil_div(chunks.per_row, kEmSlab);
    const dim3 G(chunks.rows * slabs), B(256);
    if (wdtype == WALSH_BF16) launch(embed_join_kernel<uint16_t>, G, B, 0, s, a, slabs);
    else launch(embed_join_kernel<float>, G, B, 0, s, a, slabs);
    return check_hip(hipGetLastError(), fn);
}
