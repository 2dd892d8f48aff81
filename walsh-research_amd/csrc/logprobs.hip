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
// larger one; lanes and wavefronts are joined at the end.  Four wavefronts take
// a row; sixteen where rows of more than 8,192 tokens are no more than CUs, so
// that a row is not left to a quarter of its CU (50,257 tokens: one row 5.8 us
// instead of 6.0, with 5 alternatives 9 to 10, 256 rows 7.1 instead of 7.6; at
// 512 rows sixteen take 18.2, four 12).  Rows are not split over workgroups, of
// which the last to arrive could join the others' sums in the same launch: 64
// float32 rows take 7.1 us, with 20 alternatives 12.8, where a copy of their
// bytes would take 2.5.
//
// Alternatives: the lanes' maxima, taken together over the wavefronts, are the
// largest of 256 groups of tokens.  A search by their bits finds a bound that
// at least n of them reach and few more, so at least n tokens do; lanes whose
// own maximum does read again those of their steps whose maximum does.  Those
// tokens go to a list in LDS and are ranked there by value and index.  Where
// there are too many (thousands of equal ones), or fewer are not masked than are
// asked for, the row is walked once for each further value.
//
// Bound by memory: 8,192 rows of 50,257 bf16 logits take 129 us (6.4 TB/s), with
// 5 and 20 alternatives 152 to 175 and 172 to 186 by how many lie near them, with
// float32 logits 257 (6.4), 269, 304.
// Of 10 instructions a token the exponential takes the time of four.  Their
// gradient, 823 MB read and as many written, takes 292 us (5.6 TB/s), in
// float32 582 (5.7, where a copy reaches 5.1).
#include <type_traits>

#include "rows8.h"

namespace walsh {

constexpr int kLpTop = 64;             // most alternatives
constexpr int kLpList = 1024;
constexpr float kLpLowest = -3.402823466e38f;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

// 16 bytes of logits.  What is read or written once and is more than the caches
// hold is streamed: 823 MB of bf16 logits are read in 129 us instead of 142, and
// with a gradient to come, whose kernel finds the last of them there, forward
// and gradient take 414 us instead of 446 (float32 828, 896), with the product
// that reads the gradient 987 instead of 996.  A gradient that fits beside its
// logits is better left there (8,192 x 4,096: 42 us, streamed 44), one that does
// not is streamed (2,048 rows: 97 us, not 109).
template <typename T> struct LpBlock {
    static constexpr int E = 16 / sizeof(T);
    u32x4 a;
    template <bool STREAM> __device__ __forceinline__ void load(const T *p) {
        a = load16<STREAM>(p);
    }
    template <bool STREAM> __device__ __forceinline__ void store(T *p) const {
        store16<STREAM>(p, a);
    }
    __device__ __forceinline__ void unpack(float (&v)[E]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (E == 8) v[2 * i] = __uint_as_float(a[i] << 16), v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
            else v[i] = __uint_as_float(a[i]);
        }
    }
    __device__ __forceinline__ void pack(const float (&v)[E]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (E == 8) a[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
            else a[i] = __float_as_uint(v[i]);
        }
    }
    __device__ __forceinline__ void fill(float v) {
        const uint32_t w = E == 8 ? pack_bf16x2(v, v) : __float_as_uint(v);
        a = u32x4{w, w, w, w};
    }
};

struct LogprobArgs {
    const void *logits;
    const int64_t *tokens;
    int64_t ld;
    int V, n;
    float *logprob, *entropy, *top;    // [N], [N], [N][n]
    int64_t *top_index;
    f32x4 *stats;                      // (m, S, H, 0) of every row, or null
};

// Sums over tokens, in powers of two: s = sum w, e = sum w log2 w for
// w = 2^(l log2(e) - r), with r the rounded product of a maximum m.  What its
// rounding leaves out is a factor common to all (taken back at the end), so a
// weight costs one multiply-add besides the exponential.  Lanes begin below
// every usual logit; a row where that, or an infinity or NaN, spoils the sums
// shows in them (`usual`) and is walked again with the distances l - m
// themselves (LpExact).
struct LpSums {
    float m, r, s, e;
    __device__ __forceinline__ LpSums() : m(-1e30f), r(-1e30f * kLog2e), s(0.f), e(0.f) {}
    __device__ __forceinline__ LpSums(f32x4 v) : m(v.x), r(v.x * kLog2e), s(v.y), e(v.z) {}
    // a larger maximum: at most 2^1000 below, where nothing is left of s
    __device__ __forceinline__ void move(float to) {
        const float rt = to * kLog2e, d = fmaxf(r - rt, -1000.f), c = __builtin_amdgcn_exp2f(d);
        e = c * (e + d * s);
        s *= c;
        m = to, r = rt;
    }
    __device__ __forceinline__ void add(float x) {
        const float t = fmaf(x, kLog2e, -r), w = __builtin_amdgcn_exp2f(t);
        s += w;
        e = fmaf(w, fmaxf(t, -1000.f), e);         // (0 times -inf)
    }
    __device__ __forceinline__ bool usual() const { return m < 2e38f && s > 0.f && s < INFINITY && fabsf(e) < INFINITY; }
};
struct LpExact {
    float m, s, e;
    __device__ __forceinline__ LpExact(float m_, float s_, float e_) : m(m_), s(s_), e(e_) {}
    __device__ __forceinline__ LpExact(f32x4 v) : m(v.x), s(v.y), e(v.z) {}
    // the sums of q relative to m itself: r off by d makes w 2^d times as large
    __device__ __forceinline__ explicit LpExact(const LpSums &q) : m(q.m) {
        const float d = fmaf(q.m, kLog2e, -q.r), c = __builtin_amdgcn_exp2f(-d);
        s = c * q.s, e = c * (q.e - d * q.s);
    }
    __device__ __forceinline__ void move(float to) {
        const float d = fmaxf((m - to) * kLog2e, -1000.f), c = __builtin_amdgcn_exp2f(d);
        e = c * (e + d * s);
        s *= c;
        m = to;
    }
    __device__ __forceinline__ void add(float x) {
        const float t = (x - m) * kLog2e, w = __builtin_amdgcn_exp2f(t);
        s += w;
        e = fmaf(w, fmaxf(t, -1000.f), e);
    }
};

// Over the lanes of a wavefront (ROWS 4) or of its first 16 (ROWS 1), in a
// fixed order; the result in every lane.
template <int CTRL, int MASK> __device__ __forceinline__ float lp_dpp(float none, float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(none), __float_as_int(v), CTRL, MASK, 0xf, false));
}
template <int ROWS, typename F> __device__ __forceinline__ float lp_reduce(float v, float none, F f) {
    v = f(v, lp_dpp<0x111, 0xf>(none, v));         // 1, 2, 4, 8 lanes to the left in the row of 16
    v = f(v, lp_dpp<0x112, 0xf>(none, v));
    v = f(v, lp_dpp<0x114, 0xf>(none, v));
    v = f(v, lp_dpp<0x118, 0xf>(none, v));
    if (ROWS > 1) {
        v = f(v, lp_dpp<0x142, 0xa>(none, v));     // the row before's last lane, the second row's last
        v = f(v, lp_dpp<0x143, 0xc>(none, v));
    }
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 16 * ROWS - 1));
}
template <int ROWS> __device__ __forceinline__ float lp_max(float v) {
    return lp_reduce<ROWS>(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}
template <int ROWS> __device__ __forceinline__ float lp_sum(float v) {
    return lp_reduce<ROWS>(v, 0.f, [](float a, float b) { return a + b; });
}

// Tokens in order of preference: larger values first (NaN as -inf), then lower indexes.
__device__ __forceinline__ uint32_t lp_order(float x) {
    const uint32_t b = __float_as_uint(fmaxf(x, -INFINITY) + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ uint64_t lp_key(float x, int i) { return (uint64_t)lp_order(x) << 32 | (uint32_t)~i; }
__device__ __forceinline__ float lp_value(uint64_t key) {
    const uint32_t b = (uint32_t)(key >> 32);
    return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
constexpr int kLpSlots = 16;           // of the steps' maxima
template <int NT, bool TOP> struct LpShared {
    f32x4 part[NT / 64];
    float step[TOP ? kLpSlots : 1][NT];            // a lane's largest of steps i, i + kLpSlots ...
    float group[TOP ? NT / 64 : 1][64];
    uint64_t list[TOP ? kLpList : 1];
    uint32_t most[NT / 64], many[NT / 64], first[NT / 64];
    int n;
};

// The lanes' sums joined: over the wavefront, through LDS, over the wavefronts.
template <int NT, typename Q, typename S> __device__ __forceinline__ Q lp_join(S &sh, Q q, int lane, int wave) {
    constexpr int W = NT / 64;
    q.move(lp_max<4>(q.m));
    q.s = lp_sum<4>(q.s), q.e = lp_sum<4>(q.e);
    if (lane == 0) sh.part[wave] = f32x4{q.m, q.s, q.e, 0.f};
    __syncthreads();
    const f32x4 v = sh.part[lane & (W - 1)];
    q = Q(v);
    if (lane >= W) q.s = q.e = 0.f;
    q.move(lp_max<1>(q.m));
    q.s = lp_sum<1>(q.s), q.e = lp_sum<1>(q.e);
    return q;
}

// A lane takes U blocks of E tokens in a step.
template <typename T, int NT, bool TOP, bool STREAM> __global__ __launch_bounds__(NT) void logprobs_kernel(LogprobArgs a) {
    constexpr int W = NT / 64, E = LpBlock<T>::E, U = 32 / E;
    __shared__ LpShared<NT, TOP> sh;
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
    // Blocks begin at a multiple of 4 bytes: of rows that begin between two
    // (bf16, odd strides) 16-byte loads reach 4.7 TB/s, else 5.7.  What is left
    // at both ends of the row goes to a lane each, as token `last`.
    const T *p = (const T *)a.logits + row * a.ld;
    const int lead = (uintptr_t)p & 3 ? 1 : 0;
    const int blocks = (a.V - lead) / E, rest = (a.V - lead) % E;
    const T *body = p + lead;
    const int last = tid < rest ? lead + E * blocks + tid : 0;
    LpSums q;
    const float end = tid < rest + lead ? Act<T>::load(p + last) : -INFINITY;
    // up to U blocks of the lane's step from block b on; what there is not is -inf
    auto load = [&](LpBlock<T> (&r)[U], int b) {
        if (b + (U - 1) * NT < blocks) {
#pragma unroll
            for (int j = 0; j < U; ++j) r[j].template load<STREAM>(body + E * (int64_t)(b + j * NT));
        } else {
#pragma unroll
            for (int j = 0; j < U; ++j) {
                r[j].fill(-INFINITY);
                if (b + j * NT < blocks) r[j].template load<STREAM>(body + E * (int64_t)(b + j * NT));
            }
        }
    };
    auto take = [&](const auto &r, auto n) {       // the sums of n blocks; their maximum
        float x[decltype(n)::value][E], top = -INFINITY;
#pragma unroll
        for (int j = 0; j < n; ++j) {
            r[j].unpack(x[j]);
#pragma unroll
            for (int i = 0; i < E; ++i) top = fmaxf(top, x[j][i]);
        }
        if (top > q.m) q.move(top);
#pragma unroll
        for (int j = 0; j < n; ++j)
#pragma unroll
            for (int i = 0; i < E; ++i) q.add(x[j][i]);
        return top;
    };
    if constexpr (TOP) {
#pragma unroll
        for (int i = 0; i < kLpSlots; ++i) sh.step[i][tid] = -INFINITY;
    }
    int step = 0;
    for (int b = tid; b < blocks; b += NT * U, ++step) {
        float top;
        LpBlock<T> r[U];
        if (b + NT < blocks) {
            load(r, b);
            top = take(r, std::integral_constant<int, U>{});
        } else {
            r[0].template load<STREAM>(body + E * (int64_t)b);
            top = take(r, std::integral_constant<int, 1>{});
        }
        if constexpr (TOP) {
            float &slot = sh.step[step % kLpSlots][tid];
            slot = step < kLpSlots ? top : fmaxf(slot, top);
        }
    }
    if (end > q.m) q.move(end);
    q.add(end);
    const float own = q.m;
    if constexpr (TOP) {
        sh.group[wave][lane] = own;
        if (tid == 0) sh.n = 0;
    }
    q = lp_join<NT>(sh, q, lane, wave);
    LpExact all(q);
    if (!q.usual()) {
        all = LpExact(kLpLowest, 0.f, 0.f);
        for (int i = tid; i < a.V; i += NT) {
            const float x = Act<T>::load(p + i);
            if (x > all.m) all.move(x);
            all.add(x);
        }
        __syncthreads();
        all = lp_join<NT>(sh, all, lane, wave);
    }
    const bool nothing = all.s == 0.f;             // (not where it is NaN)
    // the largest logit's own weight is 1: what rounding leaves below that would
    // make log probabilities positive
    if (all.s < 1.f && !nothing) all.s = 1.f;
    const float m = all.m, logs = __builtin_amdgcn_logf(all.s) * kLn2;
    auto logprob = [&](float x) { return nothing ? -INFINITY : (x - m) - logs; };
    if (tid == 0) {
        const float sum = logs - all.e / all.s * kLn2;
        const float h = nothing || sum < 0.f ? 0.f : sum;          // (NaN stays)
        a.logprob[row] = t < a.V ? logprob(Act<T>::load(p + t)) : NAN;
        a.entropy[row] = h;
        if (a.stats) a.stats[row] = f32x4{m, all.s, h, 0.f};
    }
    if constexpr (!TOP) return;

    float *top = a.top + row * a.n;
    int64_t *index = a.top_index + row * a.n;
    // a bound that at least n of the groups' maxima reach, and few more
    constexpr int K = 4, PER = W / K;
    uint32_t key[K];
    float least = INFINITY, most = -INFINITY;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        float g = sh.group[k * PER][lane];
#pragma unroll
        for (int w = 1; w < PER; ++w) g = fmaxf(g, sh.group[k * PER + w][lane]);
        key[k] = lp_order(g);
        least = fminf(least, g), most = fmaxf(most, g);
    }
    uint32_t lo = lp_order(-lp_max<4>(-least)), hi = lp_order(lp_max<4>(most)) + 1;
    for (int reach = 64 * K; reach > a.n + a.n / 4 + 2 && hi - lo > 1;) {
        const uint32_t mid = lo + (hi - lo) / 2;
        int c = 0;
#pragma unroll
        for (int k = 0; k < K; ++k) c += __popcll(__ballot(key[k] >= mid));
        if (c >= a.n) lo = mid, reach = c;
        else hi = mid;
    }
    // (what lies at -1e30 or below is taken from the whole row, further down)
    lo = max(lo, lp_order(-1e30f) + 1);
    const float bound = lp_value((uint64_t)lo << 32);
    auto put = [&](float x, int i) {
        if (x >= bound) {
            const int at = atomicAdd(&sh.n, 1);
            if (at < kLpList) sh.list[at] = lp_key(x, i);
        }
    };
    if (own >= bound) {
        step = 0;
        for (int b = tid; b < blocks; b += NT * U, ++step) {
            if (sh.step[step % kLpSlots][tid] < bound) continue;
            LpBlock<T> r[U];
            load(r, b);
#pragma unroll
            for (int j = 0; j < U; ++j) {
                float x[E];
                r[j].unpack(x);
#pragma unroll
                for (int i = 0; i < E; ++i) put(x[i], lead + E * (b + j * NT) + i);
            }
        }
        put(end, last);
    }
    __syncthreads();
    int got = 0;
    uint32_t below = 0xffffffffu;      // tokens of lower order are still to be looked at
    if (sh.n <= kLpList) {
        const int count = sh.n;
        for (int i = tid; i < count; i += NT) {
            const uint64_t k = sh.list[i];
            int before = 0;
            for (int j = 0; j < count; ++j) before += sh.list[j] > k;
            if (before < a.n) top[before] = logprob(lp_value(k)), index[before] = (int64_t)(uint32_t)~(uint32_t)k;
        }
        got = min(count, a.n), below = lo;
    }
    // too many for the list, or fewer than asked for: one value after the other,
    // each with as many of its tokens as are wanted, the lowest first
    while (got < a.n) {
        uint32_t most = 0, n = 0, at = 0;          // the lane's largest, how many, the first
        auto look = [&](float x, int i) {
            const uint32_t k = lp_order(x);
            if (k >= below || k < most) return;
            n = k > most ? 1 : n + 1;
            at = k > most ? i : min(at, (uint32_t)i);
            most = k;
        };
        for (int b = tid; b < blocks; b += NT) {
            LpBlock<T> r;
            float x[E];
            r.template load<STREAM>(body + E * (int64_t)b);
            r.unpack(x);
#pragma unroll
            for (int i = 0; i < E; ++i) look(x[i], lead + E * b + i);
        }
        if (tid < rest + lead) look(end, last);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const uint32_t k = (uint32_t)__shfl_xor((int)most, o), c = (uint32_t)__shfl_xor((int)n, o);
            const uint32_t i = (uint32_t)__shfl_xor((int)at, o);
            at = k > most ? i : k < most ? at : min(at, i);
            n = k > most ? c : k < most ? n : n + c;
            most = max(most, k);
        }
        __syncthreads();
        if (lane == 0) sh.most[wave] = most, sh.many[wave] = n, sh.first[wave] = at;
        __syncthreads();
        most = n = at = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const uint32_t k = sh.most[w];
            at = k > most ? sh.first[w] : k < most ? at : min(at, sh.first[w]);
            n = k > most ? sh.many[w] : k < most ? n : n + sh.many[w];
            most = max(most, k);
        }
        if (!n) break;
        const int want = min((int)n, a.n - got);
        const float v = logprob(lp_value((uint64_t)most << 32));
        if (want == 1) {
            if (tid == 0) top[got] = v, index[got] = at;
        } else {
            for (int base = (int)at, found = 0; found < want && base < a.V; base += NT) {
                const int i = base + tid;
                const bool is = i < a.V && lp_order(Act<T>::load(p + i)) == most;
                const uint64_t who = __ballot(is);
                __syncthreads();
                if (lane == 0) sh.many[wave] = (uint32_t)__popcll(who);
                __syncthreads();
                int before = found + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
                for (int w = 0; w < W; ++w) {
                    if (w < wave) before += (int)sh.many[w];
                    found += (int)sh.many[w];
                }
                if (is && before < want) top[got + before] = v, index[got + before] = i;
            }
        }
        got += want, below = most;
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
    int V, n, parts, per;              // parts of a row, blocks of 16 bytes in each
};

// A workgroup writes a part of a row by the formula without its first two
// terms, then the tokens that have one of them again, whole.
// SL, SS: loads and stores are streamed.
template <typename T, bool SL, bool SS> __global__ __launch_bounds__(256) void logprobs_bwd_kernel(LogprobBwd a) {
    constexpr int E = LpBlock<T>::E;
    const int64_t row = blockIdx.x / (uint32_t)a.parts;
    const int part = blockIdx.x % (uint32_t)a.parts, tid = threadIdx.x, lane = tid & 63;
    const int blocks = a.V / E, b1 = min(blocks, (part + 1) * a.per);
    const int rest = part == a.parts - 1 ? a.V % E : 0, last = E * blocks + tid;
    const T *p = (const T *)a.logits + row * a.ld;
    T *d = (T *)a.dlogits + row * a.ldd;
    const int64_t t = a.tokens[row];
    const f32x4 st = a.stats[row];
    const float m = st.x, S = st.y, h = st.z;
    if (t < 0 || S == 0.f) {
        LpBlock<T> z;
        z.fill(0.f);
        for (int b = part * a.per + tid; b < b1; b += 256) z.template store<SS>(d + E * b);
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
        LpBlock<T> r;
        float x[E];
        r.template load<SL>(p + E * b);
        r.unpack(x);
#pragma unroll
        for (int i = 0; i < E; ++i) x[i] = grad(x[i]);
        r.pack(x);
        r.template store<SS>(d + E * b);
    }
    if (tid < rest) Act<T>::store(d + last, grad(Act<T>::load(p + last)));
    __syncthreads();
    // the token's lane is n, the alternatives' 0 .. n - 1
    if (tid > a.n) return;
    const int64_t i = tid < a.n ? a.top_index[row * a.n + tid] : t;
    const int64_t from = E * (int64_t)part * a.per, to = part == a.parts - 1 ? a.V : E * (int64_t)b1;
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

template <typename T> static void logprobs_launch(const LogprobArgs &a, int64_t N, hipStream_t s) {
    auto go = [&](auto kernel, int nt) { launch(kernel, dim3((unsigned)N), dim3(nt), 0, s, a); };
    // four wavefronts to a row, or sixteen where there are few long ones
    if (N <= device_info().cu_count && a.V > 8192) {
        if (a.n) go(logprobs_kernel<T, 1024, true, false>, 1024);
        else go(logprobs_kernel<T, 1024, false, false>, 1024);
    } else if (!a.stats && N * a.V * (int64_t)sizeof(T) > kCacheBytes) {
        if (a.n) go(logprobs_kernel<T, 256, true, true>, 256);
        else go(logprobs_kernel<T, 256, false, true>, 256);
    } else {
        if (a.n) go(logprobs_kernel<T, 256, true, false>, 256);
        else go(logprobs_kernel<T, 256, false, false>, 256);
    }
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
    if (dtype == WALSH_BF16) logprobs_launch<uint16_t>(a, N, (hipStream_t)stream);
    else logprobs_launch<float>(a, N, (hipStream_t)stream);
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
    const int64_t blocks = V / (dtype == WALSH_BF16 ? 8 : 4), parts = blocks ? ceil_div(blocks, 1024) : 1, per = ceil_div(blocks, parts);
    if (N * parts > 0xffffffffll / 256)
        return set_error(WALSH_ENOTSUP, "%s: N=%lld rows of V=%lld", fn, (long long)N, (long long)V);
    const LogprobBwd a{logits, tokens, top_index, (const f32x4 *)stats, g_logprob, g_entropy, n ? g_top : nullptr, dlogits,
                       ld, ldd, (int)V, (int)n, (int)parts, (int)per};
    auto go = [&](auto kernel) { launch(kernel, dim3((unsigned)(N * parts)), dim3(256), 0, (hipStream_t)stream, a); };
    auto pick = [&](auto t) {
        using T = decltype(t);
        const int64_t bytes = N * V * (int64_t)sizeof(T);
        if (bytes > kCacheBytes) go(logprobs_bwd_kernel<T, true, true>);
        else if (2 * bytes > kCacheBytes) go(logprobs_bwd_kernel<T, false, true>);
        else go(logprobs_bwd_kernel<T, false, false>);
    };
    if (dtype == WALSH_BF16) pick(uint16_t{});
    else pick(float{});
    return check_hip(hipGetLastError(), fn);
}
