// Embedding lookup with scaling and dropout, and its gradient:
//     y_r = scale keep(r) W[t_r]          dW_v = scale sum over r with t_r = v of keep(r) gy_r
// with keep() the mask and factor of dropout (rows8.h).  A token outside the
// vocabulary gives a row of NaN and adds to no gradient; nor does padding_idx.
//
// The gradient adds the rows of a token in their order, in float32, so equal
// calls give equal bits.  Three kernels:
//   sort   a workgroup takes a range of up to 256 tokens and walks all N: it
//          counts those below its range, which is where its part of the sorted
//          order begins (no workgroup waits for another), and those in it by
//          token; a second walk puts them in place.
//   rows   a lane takes 8 columns of a row of dW and adds its tokens' rows up
//          to kEmLong of them; rows without tokens are zeros.  Longer rows are
//          cut where the sorted order is, every kEmLong places, and their
//          pieces summed into a workspace.
//   join   adds the pieces of each long row, in order.
#include <type_traits>

#include "rows8.h"

namespace walsh {

constexpr int kEmWaves = 16, kEmRange = 256;
constexpr int kEmLong = 32;            // tokens of a row that one lane adds

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
            store8((TY *)a.y + at[j].row * a.ldy + c, a.C - c, v[j]);
        }
    }
}

// ---------------------------------------------------------------- gradient
// order[start[v] .. start[v + 1]): the places of token v, in order.
struct EmbedSort {
    const int64_t *tokens;
    int64_t V, pad;                    // pad: a token that counts as outside (-1: none)
    int N, bits;                       // a workgroup's range: 2^bits tokens
    int *start, *order;
};

__global__ __launch_bounds__(64 * kEmWaves) void embed_sort_kernel(EmbedSort a) {
    __shared__ int count[kEmWaves][kEmRange], total[kEmRange], below_of[kEmWaves], sums[kEmRange / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int range = 1 << a.bits;
    const int64_t lo = (int64_t)blockIdx.x << a.bits;
    for (int i = tid; i < kEmWaves * kEmRange; i += 64 * kEmWaves) (&count[0][0])[i] = 0;
    __syncthreads();
    // a wavefront walks a stretch of whole steps of 64
    const int steps = (a.N + 64 * kEmWaves - 1) / (64 * kEmWaves);
    const int from = wave * steps * 64, to = min(a.N, from + steps * 64);
    auto token = [&](int i) {
        const int64_t t = i < to ? a.tokens[i] : -1;
        return t >= 0 && t < a.V && t != a.pad ? t : (int64_t)-1;
    };
    int below = 0;
#pragma unroll 8
    for (int i = from + lane; i - lane < to; i += 64) {
        const int64_t t = token(i);
        below += t >= 0 && t < lo;
        const int64_t r = t - lo;
        if (t >= lo && r < range) atomicAdd(&count[wave][(int)r], 1);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) below += __shfl_xor(below, o);
    if (lane == 0) below_of[wave] = below;
    __syncthreads();
    // where each wavefront's tokens of each value go
    int mine = 0, incl = 0;
    if (tid < kEmRange) {
        for (int w = 0; w < kEmWaves; ++w) {
            const int c = count[w][tid];
            count[w][tid] = mine;
            mine += c;
        }
        incl = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int v = __shfl_up(incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 63) sums[wave] = incl;
    }
    __syncthreads();
    if (tid < kEmRange) {
        int base = 0;
        for (int w = 0; w < kEmWaves; ++w) base += below_of[w];
        for (int w = 0; w < wave; ++w) base += sums[w];
        const int at = base + incl - mine;
        total[tid] = at;
        if (tid < range && lo + tid <= a.V) a.start[lo + tid] = at;
        // the end of the last range is the end of all
        if (tid == range - 1 && lo + range >= a.V) a.start[a.V] = base + incl;
    }
    __syncthreads();
    for (int i0 = from; i0 < to; i0 += 64) {
        const int64_t t = token(i0 + lane), r = t - lo;
        const bool in = t >= lo && r < range;
        uint64_t same = __ballot(in);
        if (!same) continue;
        const int d = in ? (int)r : 0;
        for (int b = 0; b < a.bits; ++b) {
            const uint64_t set = __ballot(d >> b & 1);
            same &= d >> b & 1 ? set : ~set;
        }
        if (in) {
            const int before = __popcll(same & ((1ull << lane) - 1));
            const int at = count[wave][d] + before;
            wave_lds_fence();
            if (before == 0) count[wave][d] = at + __popcll(same);
            a.order[total[d] + at] = i0 + lane;
        }
        wave_lds_fence();
    }
}

struct EmbedBwd {
    const int64_t *tokens;
    const int *start, *order;
    const void *gy;
    void *dw;
    float *parts;                      // [2 per chunk][C]: of the row that a chunk begins with, and ends with
    int64_t V, ldg, ldw;
    int C;
    Blocks rows, chunks;               // rows of dW, chunks of the sorted order
    uint32_t row_groups;               // workgroups that take rows
    Drop d;
    float f;
};

// sum of the gradients at places s .. e of the sorted order
template <typename TG, bool DROP>
__device__ __forceinline__ void embed_add(const EmbedBwd &a, const DropBits &bits, int s, int e, uint32_t col, float (&acc)[8]) {
    const int c = 8 * (int)col;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    constexpr int U = 4;
    for (int k = s; k < e; k += U) {
        int r[U];
        float v[U][8];
#pragma unroll
        for (int j = 0; j < U; ++j) r[j] = a.order[min(k + j, e - 1)];
#pragma unroll
        for (int j = 0; j < U; ++j) load8((const TG *)a.gy + r[j] * a.ldg + c, a.C - c, v[j]);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (DROP) bits.apply(v[j], r[j], col);
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] = k + j < e ? acc[i] + v[j][i] : acc[i];
        }
    }
}

template <typename TG, typename TW, bool DROP> __global__ __launch_bounds__(256) void embed_rows_kernel(EmbedBwd a) {
    const DropBits bits(a.d);
    float acc[8];
    if (blockIdx.x < a.row_groups) {
        const BlockAt at = block_at(a.rows, blockIdx.x * 256u, threadIdx.x);
        if (at.row >= a.rows.rows) return;
        const int s = a.start[at.row], e = a.start[at.row + 1], c = 8 * (int)at.col;
        if (e - s > kEmLong) return;
        embed_add<TG, DROP>(a, bits, s, e, at.col, acc);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] *= a.f;
        store8((TW *)a.dw + at.row * a.ldw + c, a.C - c, acc);
        return;
    }
    const BlockAt at = block_at(a.chunks, (blockIdx.x - a.row_groups) * 256u, threadIdx.x);
    const int all = a.start[a.V], s = (int)at.row * kEmLong, e = min(all, s + kEmLong);
    if (at.row >= a.chunks.rows || s >= all) return;
    const int64_t t0 = a.tokens[a.order[s]], t1 = a.tokens[a.order[e - 1]];
    const int c = 8 * (int)at.col;
    if (a.start[t0 + 1] - a.start[t0] > kEmLong) {
        embed_add<TG, DROP>(a, bits, s, min(e, a.start[t0 + 1]), at.col, acc);
        store8(a.parts + 2 * (int64_t)at.row * a.C + c, a.C - c, acc);
    }
    if (t1 != t0 && a.start[t1 + 1] - a.start[t1] > kEmLong) {
        embed_add<TG, DROP>(a, bits, a.start[t1], e, at.col, acc);
        store8(a.parts + (2 * (int64_t)at.row + 1) * a.C + c, a.C - c, acc);
    }
}

template <typename TW> __global__ __launch_bounds__(256) void embed_join_kernel(EmbedBwd a) {
    const BlockAt at = block_at(a.chunks, blockIdx.x * 256u, threadIdx.x);
    const int all = a.start[a.V], s = (int)at.row * kEmLong, e = min(all, s + kEmLong);
    if (at.row >= a.chunks.rows || s >= all) return;
    // the long row that begins in this chunk
    const int64_t t = a.tokens[a.order[e - 1]];
    const int first = a.start[t], last = a.start[t + 1] - 1;
    if (first < s || last - first < kEmLong) return;
    const int c = 8 * (int)at.col;
    float acc[8], v[8];
    load8((const float *)a.parts + (2 * (int64_t)at.row + (first == s ? 0 : 1)) * a.C + c, a.C - c, acc);
    for (int q = (int)at.row + 1; q <= last / kEmLong; ++q) {
        load8((const float *)a.parts + 2 * (int64_t)q * a.C + c, a.C - c, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += v[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] *= a.f;
    store8((TW *)a.dw + t * a.ldw + c, a.C - c, acc);
}

static int64_t embed_chunks(int64_t N) { return ceil_div(N, kEmLong); }
// start, order, parts: each from a multiple of 16 bytes on
static int64_t embed_start_bytes(int64_t V) { return ceil_div(4 * (V + 1), 16) * 16; }
static int64_t embed_order_bytes(int64_t N) { return ceil_div(4 * N, 16) * 16; }

static int embed_check(const char *fn, int64_t N, int64_t V, int64_t C, int drop, const int64_t *seed, int64_t rng_stream,
                       int dt0, int dt1) {
    if (N < 0 || C < 0 || V < 1 || C > 0x7fffffff - 8 || N > 0x7fffffff - 2048 || V > 0x7fffffff - 2048 ||
        N * ceil_div(C, 8) > kMaxBlocks)
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
    if (N < 0 || V < 1 || C < 0) return 0;
    return embed_start_bytes(V) + embed_order_bytes(N) + 2 * embed_chunks(N) * C * 4;
}

WALSH_EXPORT int walsh_embedding_bwd(const int64_t *tokens, int64_t N, const void *gy, int64_t ldg, int64_t V, int64_t C,
                                     float scale, int64_t padding_idx, int drop, const int64_t *seed, int64_t rng_stream,
                                     void *dw, int64_t ldw, int gdtype, int wdtype, void *work, int64_t work_bytes,
                                     void *stream) {
    const char *fn = "walsh_embedding_bwd";
    int rc = embed_check(fn, N, V, C, drop, seed, rng_stream, gdtype, wdtype);
    if (rc) return rc;
    if (C == 0) return WALSH_OK;
    const Blocks rows = make_blocks(V, C), chunks = make_blocks(embed_chunks(N), C);
    if (V * (int64_t)rows.per_row > kMaxBlocks)
        return set_error(WALSH_ENOTSUP, "%s: V=%lld rows of C=%lld", fn, (long long)V, (long long)C);
    if ((N && (!tokens || !gy)) || !dw || !work) return set_error(WALSH_EINVAL, "%s: null pointer", fn);
    if ((V > 1 && ldw < C) || (N > 1 && ldg < C)) return set_error(WALSH_EINVAL, "%s: rows of %lld overlap", fn, (long long)C);
    if (work_bytes < walsh_embedding_bwd_workspace_bytes(N, V, C) || (uintptr_t)work % 16)
        return set_error(WALSH_EINVAL, "%s: workspace of %lld bytes (16-aligned), needs %lld", fn, (long long)work_bytes,
                         (long long)walsh_embedding_bwd_workspace_bytes(N, V, C));
    const hipStream_t s = (hipStream_t)stream;
    int *start = (int *)work, *order = (int *)((char *)work + embed_start_bytes(V));
    float *parts = (float *)((char *)order + embed_order_bytes(N));
    // ranges small enough for a workgroup to every CU, where the vocabulary has as many
    int bits = 0;
    while (bits < 8 && ceil_div(V, 1 << bits) > device_info().cu_count) ++bits;
    const EmbedSort so{tokens, V, padding_idx >= 0 && padding_idx < V ? padding_idx : -1, (int)N, bits, start, order};
    launch(embed_sort_kernel, dim3((unsigned)ceil_div(V, 1 << bits)), dim3(64 * kEmWaves), 0, s, so);
    rc = check_hip(hipGetLastError(), fn);
    if (rc) return rc;
    const uint32_t row_groups = (uint32_t)ceil_div(V * rows.per_row, 256);
    const uint32_t chunk_groups = (uint32_t)ceil_div((int64_t)chunks.rows * chunks.per_row, 256);
    const EmbedBwd a{tokens, start, order, gy, dw, parts, V, ldg, ldw, (int)C, rows, chunks, row_groups,
                     Drop{(const uint64_t *)seed, (uint32_t)rng_stream, (uint32_t)drop},
                     (float)((double)scale * kept_factor(drop))};
    embed_types(gdtype, wdtype, drop, [&](auto g, auto w, auto d) {
        launch(embed_rows_kernel<decltype(g), decltype(w), decltype(d)::value>, dim3(row_groups + chunk_groups), dim3(256), 0,
               s, a);
    });
    rc = check_hip(hipGetLastError(), fn);
    if (rc || N <= kEmLong) return rc;
    if (wdtype == WALSH_BF16) launch(embed_join_kernel<uint16_t>, dim3(chunk_groups), dim3(256), 0, s, a);
    else launch(embed_join_kernel<float>, dim3(chunk_groups), dim3(256), 0, s, a);
    return check_hip(hipGetLastError(), fn);
}
