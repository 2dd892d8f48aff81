// Log probabilities of given tokens, with the entropy of every row of logits
// and its n most probable tokens:
//     m = max l,  S = sum exp(l - m),  L = m + log S
//     logprob = l_t - L,   H = log S - sum exp(l - m) (l - m) / S
//     alternatives: the n largest l, of equal ones the lowest indexes first
// and the gradient, for G = g_logprob + sum g_top:
//     dl_i = [i = t] g_logprob + sum_j [i = top_j] g_top_j - p_i (G + g_H (log p_i + H))
// A row with a negative token is not counted: it is not read, and gives zeros
// (no alternatives).  -inf has no weight; a row of nothing else has logprob
// -inf, entropy and gradient 0.  NaN or +inf make a row's numbers NaN.
//
// One workgroup per row, one pass over it: every lane keeps a running maximum
// and sums relative to it, in float32, moved when a step of its values brings a
// larger one; lanes and wavefronts are joined at the end.
//
// Alternatives: the lanes' maxima, taken together over the wavefronts, are the
// largest of 64 groups of tokens.  The n-th largest of them is a bound that at
// least n tokens reach, and few more: only lanes whose own maximum does look
// at their tokens again.  Those go to a list in LDS and are ranked there by
// value and index.  Where there are too many (thousands of equal ones) or a
// group has none, the row is walked once for every alternative instead.
#include "rows8.h"

namespace walsh {

constexpr int kLpTop = 64;             // most alternatives
constexpr int kLpList = 1024;
constexpr float kLpLowest = -3.402823466e38f;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

struct LogprobArgs {
    const void *logits;
    const int64_t *tokens;
    int64_t ld;
    int V, n;
    float *logprob, *entropy, *top;    // [N], [N], [N][n]
    int64_t *top_index;
    f32x4 *stats;                      // (m, S, H, 0) of every row, or null
};

// Sums over tokens relative to a maximum m, in powers of two: s = sum w,
// e = sum w log2 w for w = 2^((l - m) log2(e)).
struct LpSums {
    float m, s, e;
    // a larger maximum: at most 2^1000 below, where nothing is left of s
    __device__ __forceinline__ void move(float to) {
        const float d = fmaxf((m - to) * kLog2e, -1000.f), c = __builtin_amdgcn_exp2f(d);
        e = c * (e + d * s);
        s *= c;
        m = to;
    }
    __device__ __forceinline__ void add(float x) {
        const float t = (x - m) * kLog2e, w = __builtin_amdgcn_exp2f(t);
        s += w;
        e = fmaf(w, fmaxf(t, -1000.f), e);         // (0 times -inf)
    }
};

// Tokens in order of preference: larger values first, then lower indexes.
__device__ __forceinline__ uint64_t lp_key(float x, int i) {
    const uint32_t b = __float_as_uint(fmaxf(x, -INFINITY) + 0.f);
    return (uint64_t)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (uint32_t)~i;
}
__device__ __forceinline__ float lp_value(uint64_t key) {
    const uint32_t b = (uint32_t)(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ uint64_t lp_xor(uint64_t v, int o) {
    return (uint64_t)(uint32_t)__shfl_xor((int)(v >> 32), o) << 32 | (uint32_t)__shfl_xor((int)(uint32_t)v, o);
}

template <int NT> struct LpShared {
    f32x4 part[NT / 64];
    float group[NT / 64][64];
    uint64_t list[kLpList], best[NT / 64];
    int n;
};

template <typename T, int NT, bool TOP> __global__ __launch_bounds__(NT) void logprobs_kernel(LogprobArgs a) {
    constexpr int W = NT / 64, U = 4;
    __shared__ LpShared<NT> sh;
    const int64_t row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t t = a.tokens[row];
    if (t < 0) {
        if (tid == 0) {
            a.logprob[row] = a.entropy[row] = 0.f;
            if (a.stats) a.stats[row] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        if (TOP && tid < a.n) a.top[row * a.n + tid] = -INFINITY, a.top_index[row * a.n + tid] = -1;
        return;
    }
    const T *p = (const T *)a.logits + row * a.ld;
    const int blocks = a.V / 8, rest = a.V & 7;
    // each(f): f(first index, values), 8 at a time
    LpSums q{kLpLowest, 0.f, 0.f};
    for (int b0 = tid; b0 < blocks; b0 += NT * U) {
        Raw8<T> r[U];
        float x[U][8], top = kLpLowest;
#pragma unroll
        for (int j = 0; j < U; ++j) {
            r[j].fill(-INFINITY);
            if (b0 + j * NT < blocks) r[j].load(p + 8 * (b0 + j * NT));
        }
#pragma unroll
        for (int j = 0; j < U; ++j) {
            r[j].unpack(x[j]);
#pragma unroll
            for (int i = 0; i < 8; ++i) top = fmaxf(top, x[j][i]);
        }
        if (top > q.m) q.move(top);
#pragma unroll
        for (int j = 0; j < U; ++j)
#pragma unroll
            for (int i = 0; i < 8; ++i) q.add(x[j][i]);
    }
    const int last = 8 * blocks + tid;             // the row's last tokens, one to a lane
    if (tid < rest) {
        const float x = Act<T>::load(p + last);
        if (x > q.m) q.move(x);
        q.add(x);
    }
    const float own = q.m;
    // the wavefront's, then the row's
    float m = own;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    q.move(m);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) q.s += __shfl_xor(q.s, o), q.e += __shfl_xor(q.e, o);
    if (lane == 0) sh.part[wave] = f32x4{q.m, q.s, q.e, 0.f};
    if constexpr (TOP) {
        sh.group[wave][lane] = own;
        if (tid == 0) sh.n = 0;
    }
    __syncthreads();
    LpSums all{sh.part[0].x, sh.part[0].y, sh.part[0].z};
#pragma unroll
    for (int w = 1; w < W; ++w) m = fmaxf(m, sh.part[w].x);
    m = fmaxf(m, all.m);
    all.move(m);
#pragma unroll
    for (int w = 1; w < W; ++w) {
        LpSums o{sh.part[w].x, sh.part[w].y, sh.part[w].z};
        o.move(m);
        all.s += o.s, all.e += o.e;
    }
    const float logs = __builtin_amdgcn_logf(all.s) * kLn2;
    const bool nothing = all.s == 0.f;             // (not where it is NaN)
    auto logprob = [&](float x) { return nothing ? -INFINITY : (x - m) - logs; };
    if (tid == 0) {
        const float h = nothing ? 0.f : logs - all.e / all.s * kLn2;
        a.logprob[row] = t < a.V ? logprob(Act<T>::load(p + t)) : NAN;
        a.entropy[row] = h;
        if (a.stats) a.stats[row] = f32x4{m, all.s, h, 0.f};
    }
    if constexpr (!TOP) return;

    float *top = a.top + row * a.n;
    int64_t *index = a.top_index + row * a.n;
    // the n-th largest of the groups' maxima
    float g = sh.group[0][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) g = fmaxf(g, sh.group[w][lane]);
    int rank = 0;
#pragma unroll
    for (int j = 0; j < 64; ++j) {
        const float o = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(g), j));
        rank += o > g || (o == g && j < lane);
    }
    const uint64_t nth = __ballot(rank == a.n - 1);
    const float bound = __shfl(g, (int)__ffsll((long long)nth) - 1);
    if (bound > kLpLowest) {
        auto put = [&](float x, int i) {
            if (x >= bound) {
                const int at = atomicAdd(&sh.n, 1);
                if (at < kLpList) sh.list[at] = lp_key(x, i);
            }
        };
        if (own >= bound) {
            for (int b = tid; b < blocks; b += NT) {
                Raw8<T> r;
                float x[8];
                r.load(p + 8 * b);
                r.unpack(x);
#pragma unroll
                for (int i = 0; i < 8; ++i) put(x[i], 8 * b + i);
            }
            if (tid < rest) put(Act<T>::load(p + last), last);
        }
        __syncthreads();
        const int count = sh.n;
        if (count <= kLpList) {
            for (int i = tid; i < count; i += NT) {
                const uint64_t k = sh.list[i];
                int before = 0;
                for (int j = 0; j < count; ++j) before += sh.list[j] > k;
                if (before < a.n) top[before] = logprob(lp_value(k)), index[before] = (int64_t)(uint32_t)~(uint32_t)k;
            }
            return;
        }
    }
    uint64_t prev = ~0ull;
    for (int j = 0; j < a.n; ++j) {
        uint64_t k = 0;
        for (int i = tid; i < a.V; i += NT) {
            const uint64_t c = lp_key(Act<T>::load(p + i), i);
            if (c < prev && c > k) k = c;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint64_t c = lp_xor(k, o);
            if (c > k) k = c;
        }
        __syncthreads();
        if (lane == 0) sh.best[wave] = k;
        __syncthreads();
        prev = sh.best[0];
        for (int w = 1; w < W; ++w)
            if (sh.best[w] > prev) prev = sh.best[w];
        if (tid == 0) top[j] = logprob(lp_value(prev)), index[j] = (int64_t)(uint32_t)~(uint32_t)prev;
    }
}

// ---------------------------------------------------------------- gradient
struct LogprobBwd {
    const void *logits;
    const int64_t *tokens, *top_index;
    const f32x4 *stats;
    const float *g_logprob, *g_entropy, *g_top;    // [N], [N], [N][n], or null
    void *dlogits;
    int64_t ld, ldd;
    int V, n, parts, per;              // parts of a row, blocks of 8 in each
};

// A workgroup writes a part of a row by the formula without its first two
// terms, then the tokens that have one of them again, whole.
template <typename T> __global__ __launch_bounds__(256) void logprobs_bwd_kernel(LogprobBwd a) {
    const int64_t row = blockIdx.x / (uint32_t)a.parts;
    const int part = blockIdx.x % (uint32_t)a.parts, tid = threadIdx.x, lane = tid & 63;
    const int blocks = a.V / 8, b1 = min(blocks, (part + 1) * a.per);
    const int rest = part == a.parts - 1 ? a.V & 7 : 0, last = 8 * blocks + tid;
    const T *p = (const T *)a.logits + row * a.ld;
    T *d = (T *)a.dlogits + row * a.ldd;
    const int64_t t = a.tokens[row];
    const f32x4 st = a.stats[row];
    const float m = st.x, S = st.y, h = st.z;
    if (t < 0 || S == 0.f) {
        Raw8<T> z;
        z.fill(0.f);
        for (int b = part * a.per + tid; b < b1; b += 256) z.store(d + 8 * b);
        if (tid < rest) Act<T>::store(d + last, 0.f);
        return;
    }
    float G = a.g_top && lane < a.n ? a.g_top[row * a.n + lane] : 0.f;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) G += __shfl_xor(G, o);
    const float g = a.g_logprob ? a.g_logprob[row] : 0.f, gh = a.g_entropy ? a.g_entropy[row] : 0.f;
    G += g;
    const float inv = t < a.V ? 1.f / S : NAN, logs = __builtin_amdgcn_logf(S) * kLn2, hs = h - logs;
    auto grad = [&](float x) {
        const float t = x - m, w = __builtin_amdgcn_exp2f(t * kLog2e) * inv;
        return -w * (G + gh * (fmaxf(t, -1000.f) + hs));
    };
    for (int b = part * a.per + tid; b < b1; b += 256) {
        Raw8<T> r;
        float x[8];
        r.load(p + 8 * b);
        r.unpack(x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = grad(x[i]);
        r.pack(x);
        r.store(d + 8 * b);
    }
    if (tid < rest) Act<T>::store(d + last, grad(Act<T>::load(p + last)));
    __syncthreads();
    // the token's lane is n, the alternatives' 0 .. n - 1
    if (tid > a.n) return;
    const int64_t i = tid < a.n ? a.top_index[row * a.n + tid] : t;
    const int64_t from = 8 * (int64_t)part * a.per, to = part == a.parts - 1 ? a.V : 8 * (int64_t)b1;
    if (i < from || i >= to) return;
    float add = tid < a.n ? (a.g_top ? a.g_top[row * a.n + tid] : 0.f) : g;
    if (tid < a.n) {
        if (i == t) add += g;
    } else {
        for (int j = 0; j < a.n; ++j)
            if (a.top_index[row * a.n + j] == t) return;
    }
    Act<T>::store(d + i, add + grad(Act<T>::load(p + i)));
}

static int logprobs_check(const char *fn, int64_t N, int64_t V, int64_t n, int64_t ld, int dtype) {
    if (N < 0 || N > 0x7fffff || V < 1 || V > 0x7fffffff / 2 || n < 0 || n > kLpTop || n > V)
        return set_error(WALSH_EINVAL, "%s: N=%lld rows (below 2^23) of V=%lld, %lld alternatives (up to 64 and V)", fn,
                         (long long)N, (long long)V, (long long)n);
    if (dtype != WALSH_F32 && dtype != WALSH_BF16) return set_error(WALSH_ENOTSUP, "%s: dtype %d", fn, dtype);
    if (N > 1 && ld < V) return set_error(WALSH_EINVAL, "%s: row stride %lld for %lld logits", fn, (long long)ld, (long long)V);
    return WALSH_OK;
}

}  // namespace walsh

using namespace walsh;

WALSH_EXPORT int walsh_token_logprobs_fwd(const void *logits, int64_t ld, int64_t N, int64_t V, const int64_t *tokens,
                                          int64_t n, float *logprob, float *entropy, float *top, int64_t *top_index,
                                          float *stats, int dtype, void *stream) {
    const char *fn = "walsh_token_logprobs_fwd";
    const int rc = logprobs_check(fn, N, V, n, ld, dtype);
    if (rc) return rc;
    if (N == 0) return WALSH_OK;
    if (!logits || !tokens || !logprob || !entropy || (n && (!top || !top_index)))
        return set_error(WALSH_EINVAL, "%s: null pointer", fn);
    if ((uintptr_t)stats % 16) return set_error(WALSH_EINVAL, "%s: stats 16-byte aligned", fn);
    const LogprobArgs a{logits, tokens, ld, (int)V, (int)n, logprob, entropy, top, top_index, (f32x4 *)stats};
    auto go = [&](auto kernel, int nt) { launch(kernel, dim3((unsigned)N), dim3(nt), 0, (hipStream_t)stream, a); };
    if (dtype == WALSH_BF16) {
        if (n) go(logprobs_kernel<uint16_t, 1024, true>, 1024);
        else go(logprobs_kernel<uint16_t, 256, false>, 256);
    } else {
        if (n) go(logprobs_kernel<float, 1024, true>, 1024);
        else go(logprobs_kernel<float, 256, false>, 256);
    }
    return check_hip(hipGetLastError(), fn);
}

WALSH_EXPORT int walsh_token_logprobs_bwd(const void *logits, int64_t ld, int64_t N, int64_t V, const int64_t *tokens,
                                          int64_t n, const int64_t *top_index, const float *stats, const float *g_logprob,
                                          const float *g_entropy, const float *g_top, void *dlogits, int64_t ldd, int dtype,
                                          void *stream) {
    const char *fn = "walsh_token_logprobs_bwd";
    const int rc = logprobs_check(fn, N, V, n, ld < ldd ? ld : ldd, dtype);
    if (rc) return rc;
    if (N == 0) return WALSH_OK;
    if (!logits || !tokens || !stats || !dlogits || (n && !top_index)) return set_error(WALSH_EINVAL, "%s: null pointer", fn);
    if ((uintptr_t)stats % 16) return set_error(WALSH_EINVAL, "%s: stats 16-byte aligned", fn);
    const int64_t blocks = V / 8, parts = blocks ? ceil_div(blocks, 1024) : 1, per = ceil_div(blocks, parts);
    if (N * parts > kMaxBlocks / 256)
        return set_error(WALSH_ENOTSUP, "%s: N=%lld rows of V=%lld", fn, (long long)N, (long long)V);
    const LogprobBwd a{logits, tokens, top_index, (const f32x4 *)stats, g_logprob, g_entropy, n ? g_top : nullptr, dlogits,
                       ld, ldd, (int)V, (int)n, (int)parts, (int)per};
    const dim3 G((unsigned)(N * parts)), B(256);
    if (dtype == WALSH_BF16) launch(logprobs_bwd_kernel<uint16_t>, G, B, 0, (hipStream_t)stream, a);
    else launch(logprobs_bwd_kernel<float>, G, B, 0, (hipStream_t)stream, a);
    return check_hip(hipGetLastError(), fn);
}
