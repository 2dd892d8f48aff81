// The next token of every row of logits, from a given uniform number u:
//     z_i = l_i / T,   w_i = exp(z_i - max z)
//   top-k   the k largest l (of equal ones the lowest indexes first)
//   top-p   of these, in the same order, a token stays while the weight before
//           it is below p of their sum (the first always stays)
//   min-p   of these, w_i >= min_p
//   draw    the first index whose running sum of remaining weights, in index
//           order, exceeds u times their sum
// T <= 0 takes the largest logit.  NaN counts as -inf; a row without a finite
// or infinite maximum gives -1.
//
// No sorting: the tokens that top-k and top-p keep are those above a threshold
// logit, and the first r of those equal to it.  The threshold is found from a
// histogram of counts and weights over the distance from the maximum (2048
// bins, 64 to a factor of two), and within its bin exactly, by the bits of the
// logits (sm_select).
//
// Weights are float32, with 1 / T in two parts so that its rounding does not
// tilt them all to one side; all sums are 64-bit integers of 2^-44, exact in
// any order, so equal calls give equal tokens and borders are met as in exact
// arithmetic up to the weights' own rounding.
//
// One workgroup of 16 wavefronts per row; wavefront w walks the indexes from
// w * ceil(V / 1024) * 64 on, 64 at a time.  The row is read for its maximum,
// for the histogram, and once more to keep the tokens that the histogram
// leaves in question, each wavefront's in a list in LDS; what follows works on
// the lists, or, where one overflows (nothing filtered, or thousands kept), on
// the row again, out of the L2.
#include "common.h"

namespace walsh {

constexpr int kSmWaves = 16;
constexpr int kSmThreads = 64 * kSmWaves;
constexpr int kSmBins = 2048, kSmList = 2048;
constexpr int kSmKept = 512;                    // tokens of a wavefront's list
constexpr int kSmParts = 8;                     // parts of a wavefront's walk with sums of their own
constexpr float kSmBinsPer2 = 64.f;             // bins to a factor of two

struct SampleArgs {
    const void *logits;
    int64_t ld, V;
    const float *u, *temperature, *top_p, *min_p;   // [B], or null and the value below
    const int *top_k;
    float temperature0, top_p0, min_p0;
    int top_k0;
    int64_t *out;
};

// Order-preserving integer of a float (no NaN); -0 counts as 0.
__device__ __forceinline__ uint32_t sm_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct SmShared {
    unsigned long long mass[kSmBins];
    uint32_t count[kSmBins];
    uint32_t list[kSmList];                     // keys of a bin
    uint2 kept[kSmWaves][kSmKept];              // (key, index) of the tokens in question, by wavefront
    unsigned long long wsum[kSmWaves], part[kSmWaves][kSmParts];
    uint32_t wcnt[kSmWaves];
    float wmax[kSmWaves];
    // results of a search
    uint32_t n, kmin, kmax, before;
    unsigned long long mbefore;
    int bin, over;
};

__device__ __forceinline__ unsigned long long shfl64(unsigned long long v, int src) {
    return ((unsigned long long)(uint32_t)__shfl((int)(v >> 32), src) << 32) | (uint32_t)__shfl((int)(uint32_t)v, src);
}
// Inclusive sums over the wavefront's lanes.
__device__ __forceinline__ void wave_scan(uint32_t &c, unsigned long long &m, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t oc = (uint32_t)__shfl_up((int)c, o);
        const unsigned long long om = ((unsigned long long)(uint32_t)__shfl_up((int)(m >> 32), o) << 32) |
                                      (uint32_t)__shfl_up((int)(uint32_t)m, o);
        if (lane >= o) c += oc, m += om;
    }
}
__device__ __forceinline__ unsigned long long wave_sum64(unsigned long long v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1)
        v += ((unsigned long long)(uint32_t)__shfl_xor((int)(v >> 32), o) << 32) |
             (uint32_t)__shfl_xor((int)(uint32_t)v, o);
    return v;
}

__device__ __forceinline__ float sm_value(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

// The row's weights.
struct SmWeights {
    float m, chi, clo;     // log2(e) / T in two parts
    bool one;              // only the maximum counts (T <= 0 or tiny, or an infinite maximum)
    __device__ __forceinline__ float log2_of(float x) const {       // -inf .. 0
        const float s = x - m;
        return fmaf(s, chi, s * clo);
    }
    __device__ __forceinline__ float of(float x) const {
        return one ? (x == m ? 1.f : 0.f) : x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(log2_of(x));
    }
    // of() in units of 2^-44, by the addition of 1.5 * 2^8: 44 fraction bits are left below it
    static __device__ __forceinline__ unsigned long long fixed(float w) {
        return (unsigned long long)__double_as_longlong((double)w + 384.0) - 0x4078000000000000ull;
    }
    __device__ __forceinline__ unsigned long long mass(float x) const { return fixed(of(x)); }
    __device__ __forceinline__ int bin(float x) const {             // monotone in x
        if (one) return x == m ? 0 : kSmBins - 1;
        const float y = (x - m) * chi * -kSmBinsPer2;
        return y < (float)(kSmBins - 1) ? (int)y : kSmBins - 1;
    }
};

// The tokens that a wavefront walks, 64 at a time and in index order:
// each(f) calls f(step, there, value) with every lane.
template <typename T> struct SmRow {
    const T *p;
    int base, n, end;      // first index of the lane, steps, past the last index
    __device__ __forceinline__ SmRow(const T *row, int V, int wave, int lane) {
        n = (V + kSmThreads - 1) / kSmThreads;
        p = row;
        base = wave * n * 64 + lane;
        end = min(V, (wave + 1) * n * 64);
    }
    __device__ __forceinline__ int index(int i) const { return base + 64 * i; }
    template <typename F> __device__ __forceinline__ void each(int i0, int i1, F f) const {
        constexpr int U = 8;                                        // loads on their way together
        for (int i = i0; i < i1; i += U) {
            float v[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int at = index(i + j);
                v[j] = i + j < i1 && at < end ? Act<T>::load(p + at) : -INFINITY;
            }
#pragma unroll
            for (int j = 0; j < U; ++j)
                if (i + j < i1) f(i + j, index(i + j) < end, v[j] == v[j] ? v[j] : -INFINITY);
        }
    }
    template <typename F> __device__ __forceinline__ void each(F f) const { each(0, n, f); }
};
struct SmKeptRow {
    const uint2 *p;
    int lane, n, end;
    __device__ __forceinline__ SmKeptRow(const uint2 *list, int count, int lane_) {
        p = list, lane = lane_, end = count, n = (count + 63) / 64;
    }
    __device__ __forceinline__ int index(int i) const { return (int)p[lane + 64 * i].y; }
    template <typename F> __device__ __forceinline__ void each(int i0, int i1, F f) const {
        for (int i = i0; i < i1; ++i) {
            const bool there = lane + 64 * i < end;
            f(i, there, there ? sm_value(p[lane + 64 * i].x) : -INFINITY);
        }
    }
    template <typename F> __device__ __forceinline__ void each(F f) const { each(0, n, f); }
};

// A threshold: tokens with a larger key stay, and the first `ties` of those
// with this key.
struct SmCut {
    uint32_t key, ties;
};
// What a search looks for: the place where the count (or, by_mass, the
// weight) before a token, in descending order, reaches `need`.
__device__ __forceinline__ uint32_t sm_ties(bool by_mass, uint32_t need, uint32_t before, unsigned long long mneed,
                                            unsigned long long mbefore, unsigned long long w) {
    if (!by_mass) return need - before;
    const unsigned long long left = mneed - mbefore;                // > 0; w > 0, or nothing would be left to reach
    return w ? (uint32_t)((left + w - 1) / w) : 1u;
}

// The first bin, in order from the maximum, at whose end the running count or
// weight reaches the need; with what lies before it.  All threads.
__device__ __forceinline__ void sm_find_bin(SmShared &sh, int nbins, bool by_mass, uint32_t need,
                                            unsigned long long mneed) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = nbins / kSmThreads > 0 ? nbins / kSmThreads : 1;   // 2 for the histogram, 1 for 256 digits
    uint32_t c = 0;
    unsigned long long m = 0;
    const bool mine = tid * per < nbins;
    if (mine)
        for (int i = 0; i < per; ++i) c += sh.count[tid * per + i], m += sh.mass[tid * per + i];
    uint32_t ci = c;
    unsigned long long mi = m;
    wave_scan(ci, mi, lane);
    if (lane == 63) sh.wcnt[wave] = ci, sh.wsum[wave] = mi;
    __syncthreads();
    uint32_t c0 = ci - c;
    unsigned long long m0 = mi - m;
    for (int w = 0; w < wave; ++w) c0 += sh.wcnt[w], m0 += sh.wsum[w];
    if (mine && (by_mass ? m0 < mneed && mneed <= m0 + m : c0 < need && need <= c0 + c)) {   // one thread
        for (int i = 0; i < per; ++i) {
            const uint32_t cb = sh.count[tid * per + i];
            const unsigned long long mb = sh.mass[tid * per + i];
            if (by_mass ? mneed <= m0 + mb : need <= c0 + cb) {
                sh.bin = tid * per + i, sh.before = c0, sh.mbefore = m0;
                break;
            }
            c0 += cb, m0 += mb;
        }
    }
    __syncthreads();
}

// The cut within bin `sh.bin`, among the tokens of it that `in` admits.  All threads.
template <typename Row, typename In>
__device__ __forceinline__ SmCut sm_select(SmShared &sh, const Row &row, const SmWeights &wt, bool by_mass, uint32_t need,
                                           unsigned long long mneed, In in) {
    const int tid = threadIdx.x, bin = sh.bin;
    uint32_t before = sh.before;
    unsigned long long mbefore = sh.mbefore;
    __syncthreads();
    if (tid == 0) sh.n = 0, sh.kmin = 0xffffffffu, sh.kmax = 0;
    __syncthreads();
    row.each([&](int, bool there, float x) {
        if (there && wt.bin(x) == bin) {
            const uint32_t k = sm_key(x);
            if (in(k)) {
                const uint32_t at = atomicAdd(&sh.n, 1u);
                if (at < kSmList) sh.list[at] = k;
                atomicMin(&sh.kmin, k);
                atomicMax(&sh.kmax, k);
            }
        }
    });
    __syncthreads();
    const uint32_t n = sh.n;
    uint32_t lo = sh.kmin;                                          // the cut's key lies in lo .. lo + 2^bits - 1
    int bits = lo == sh.kmax ? 0 : 32 - __clz((int)(sh.kmax - lo));
    while (bits > 0) {
        const int d = bits < 8 ? bits : 8, sft = bits - d;          // the next digit, its largest value first
        __syncthreads();
        if (tid < 256) sh.count[tid] = 0, sh.mass[tid] = 0;
        __syncthreads();
        auto put = [&](uint32_t k) {
            const uint32_t o = k - lo;
            if (k < lo || (o >> sft) >= (1u << d)) return;
            const uint32_t q = ((1u << d) - 1) - (o >> sft);
            atomicAdd(&sh.count[q], 1u);
            if (by_mass) atomicAdd(&sh.mass[q], wt.mass(sm_value(k)));
        };
        if (n <= kSmList) {
            for (uint32_t i = tid; i < n; i += kSmThreads) put(sh.list[i]);
        } else {
            row.each([&](int, bool there, float x) {
                if (there && wt.bin(x) == bin) {
                    const uint32_t k = sm_key(x);
                    if (in(k)) put(k);
                }
            });
        }
        __syncthreads();
        sm_find_bin(sh, 256, by_mass, need - before, mneed - mbefore);
        before += sh.before, mbefore += sh.mbefore;
        lo += (uint32_t)(((1u << d) - 1) - sh.bin) << sft;
        bits = sft;
    }
    return SmCut{lo, sm_ties(by_mass, need, before, mneed, mbefore, wt.mass(sm_value(lo)))};
}

// The sum of the histogram's weights.  All threads.
__device__ __forceinline__ unsigned long long sm_total(SmShared &sh) {
    const int tid = threadIdx.x;
    unsigned long long s = 0, total = 0;
    for (int i = tid; i < kSmBins; i += kSmThreads) s += sh.mass[i];
    s = wave_sum64(s);
    if ((tid & 63) == 0) sh.wsum[tid >> 6] = s;
    __syncthreads();
    for (int w = 0; w < kSmWaves; ++w) total += sh.wsum[w];
    __syncthreads();
    return total;
}
// The weight that top-p asks for.
__device__ __forceinline__ unsigned long long sm_share(float p, unsigned long long total) {
    const double t = ceil((double)p * (double)total);
    return t >= (double)total ? total : t > 1. ? (unsigned long long)t : 1ull;
}

// From the first search's bin (sh.bin, sh.before, sh.mbefore) to the token, on
// the whole row or on the lists.
template <typename Row>
__device__ __forceinline__ void sm_finish(SmShared &sh, const Row &row, const SmWeights &wt, bool by_k, bool by_p,
                                          uint32_t k, float top_p, unsigned long long need, float min_p, float u,
                                          int64_t *out) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    SmCut cut{0u, 0u};
    if (by_k) {
        cut = sm_select(sh, row, wt, false, k, 0ull, [](uint32_t) { return true; });
        if (by_p) {
            // the histogram of what top-k keeps; the ties at its cut weigh the
            // same, so any of them stand for the first ones
            __syncthreads();
            for (int i = tid; i < kSmBins; i += kSmThreads) sh.count[i] = 0, sh.mass[i] = 0;
            __syncthreads();
            row.each([&](int, bool there, float x) {
                if (there && sm_key(x) > cut.key) atomicAdd(&sh.mass[wt.bin(x)], wt.mass(x));
            });
            if (tid == 0) {
                const float x = sm_value(cut.key);
                atomicAdd(&sh.mass[wt.bin(x)], wt.mass(x) * cut.ties);
            }
            __syncthreads();
            need = sm_share(top_p, sm_total(sh));
            sm_find_bin(sh, kSmBins, true, 0u, need);
        }
    }
    if (by_p) {
        const uint32_t least = cut.key;
        const SmCut c = sm_select(sh, row, wt, true, 0u, need, [&](uint32_t q) { return q >= least; });
        if (!by_k || c.key > cut.key) cut = c;
        else cut.ties = min(cut.ties, c.ties);
    }
    const bool cutting = by_k || by_p;
    uint32_t tie = 0;                                               // ties at the cut before this wavefront
    __syncthreads();
    if (cutting) {
        uint32_t t = 0;
        row.each([&](int, bool there, float x) { t += __popcll(__ballot(there && sm_key(x) == cut.key)); });
        if (lane == 0) sh.wcnt[wave] = t;
        __syncthreads();
        for (int w = 0; w < wave; ++w) tie += sh.wcnt[w];
    }
    // the weight that a token keeps (0: it is gone); `seen` counts the ties on
    auto rest = [&](bool there, float x, uint32_t &seen) {
        if (cutting) {
            const uint32_t q = sm_key(x);
            const unsigned long long eq = __ballot(there && q == cut.key);
            const uint32_t r = seen + __popcll(eq & ((1ull << lane) - 1));
            there = there && (q > cut.key || (q == cut.key && r < cut.ties));
            seen += __popcll(eq);
        }
        const float w = wt.of(x);
        return there && w >= min_p ? SmWeights::fixed(w) : 0ull;
    };
    // sums of the parts of the walk, then of wavefronts
    const int step = (row.n + kSmParts - 1) / kSmParts;
    unsigned long long mine = 0;
    uint32_t seen = tie;
    for (int j = 0; j < kSmParts; ++j) {
        unsigned long long s = 0;
        if (j * step < row.n) {
            if (lane == 0) sh.part[wave][j] = 0;
            const uint32_t at = seen;
            row.each(j * step, min(row.n, (j + 1) * step), [&](int, bool there, float x) { s += rest(there, x, seen); });
            s = wave_sum64(s);
            if (lane == 0) sh.part[wave][j] = s;
            if (lane == 0) sh.list[wave * kSmParts + j] = at;       // ties before the part
        }
        mine += s;
    }
    if (lane == 0) sh.wsum[wave] = mine;
    __syncthreads();
    unsigned long long all = 0, run = 0;
    for (int w = 0; w < kSmWaves; ++w) {
        if (w == wave) run = all;
        all += sh.wsum[w];
    }
    if (all == 0) {                                                 // min_p above 1, or not a number
        if (tid == 0) *out = -1;
        return;
    }
    const double ut = (double)(u > 0.f ? u : 0.f) * (double)all;
    unsigned long long thr = ut < (double)all ? (unsigned long long)ut : all - 1;   // the first running sum above this
    if (thr >= all) thr = all - 1;
    if (thr < run || thr >= run + mine) return;                     // another wavefront's
    int j = 0;
    while (run + sh.part[wave][j] <= thr) run += sh.part[wave][j++];
    seen = sh.list[wave * kSmParts + j];
    bool found = false;
    row.each(j * step, min(row.n, (j + 1) * step), [&](int i, bool there, float x) {
        unsigned long long s = rest(there, x, seen);
        if (found || !__any(s != 0)) return;
        uint32_t none = 0;
        wave_scan(none, s, lane);
        const unsigned long long hit = __ballot(run + s > thr);
        if (hit) {
            if (lane == (int)__ffsll((long long)hit) - 1) *out = row.index(i);
            found = true;
        }
        run += shfl64(s, 63);
    });
}

template <typename T> __global__ __launch_bounds__(kSmThreads) void sample_kernel(SampleArgs a) {
    extern __shared__ __align__(16) unsigned char sm_smem[];
    SmShared &sh = *(SmShared *)sm_smem;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float temp = a.temperature ? a.temperature[b] : a.temperature0;
    const float top_p = a.top_p ? a.top_p[b] : a.top_p0, min_p = a.min_p ? a.min_p[b] : a.min_p0;
    const int top_k = a.top_k ? a.top_k[b] : a.top_k0;
    const float u = a.u[b];
    const SmRow<T> row((const T *)a.logits + b * a.ld, (int)a.V, wave, lane);

    float m = -INFINITY;
    row.each([&](int, bool, float x) { m = fmaxf(m, x); });
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (lane == 0) sh.wmax[wave] = m;
    for (int i = tid; i < kSmBins; i += kSmThreads) sh.count[i] = 0, sh.mass[i] = 0;
    if (tid == 0) sh.over = 0;
    __syncthreads();
    m = sh.wmax[0];
    for (int w = 1; w < kSmWaves; ++w) m = fmaxf(m, sh.wmax[w]);
    if (m == -INFINITY) {
        if (tid == 0) a.out[b] = -1;
        return;
    }
    const bool greedy = !(temp > 0.f);
    const double c = greedy ? 0. : 1.4426950408889634074 / (double)temp;
    const SmWeights wt{m, (float)c, (float)(c - (double)(float)c), greedy || m == INFINITY || !(c < 1e30)};
    const bool by_k = greedy || (top_k > 0 && top_k < a.V), by_p = !greedy && top_p < 1.f;
    const uint32_t k = greedy ? 1u : (uint32_t)top_k;
    unsigned long long need = 0;
    if (by_k || by_p) {
        row.each([&](int, bool there, float x) {
            if (there) {
                const int q = wt.bin(x);
                if (by_k) atomicAdd(&sh.count[q], 1u);
                else atomicAdd(&sh.mass[q], wt.mass(x));
            }
        });
        __syncthreads();
        if (!by_k) need = sm_share(top_p, sm_total(sh));
        sm_find_bin(sh, kSmBins, !by_k, k, need);
    }
    // the tokens still in question: down to the search's bin, or to min_p
    const int last = by_k || by_p ? sh.bin : kSmBins;
    int kept = 0;
    if (last < kSmBins || min_p > 0.f) {
        row.each([&](int i, bool there, float x) {
            const bool in = there && (last < kSmBins ? wt.bin(x) <= last : wt.of(x) >= min_p);
            const unsigned long long who = __ballot(in);
            const int at = kept + __popcll(who & ((1ull << lane) - 1));
            if (in && at < kSmKept) sh.kept[wave][at] = make_uint2(sm_key(x), (uint32_t)row.index(i));
            kept += __popcll(who);
        });
        if (kept > kSmKept && lane == 0) sh.over = 1;
    } else if (tid == 0) {
        sh.over = 1;
    }
    __syncthreads();
    if (sh.over) sm_finish(sh, row, wt, by_k, by_p, k, top_p, need, min_p, u, a.out + b);
    else sm_finish(sh, SmKeptRow(sh.kept[wave], kept, lane), wt, by_k, by_p, k, top_p, need, min_p, u, a.out + b);
}

}  // namespace walsh

using namespace walsh;

WALSH_EXPORT int walsh_sample(const void *logits, int64_t ld, int64_t B, int64_t V, const float *u,
                              const float *temperature, float temperature0, const int *top_k, int top_k0,
                              const float *top_p, float top_p0, const float *min_p, float min_p0, int64_t *out, int dtype,
                              void *stream) {
    const char *fn = "walsh_sample";
    if (B < 0 || B > INT32_MAX || V < 1 || V > (1 << 20))
        return set_error(WALSH_EINVAL, "%s: bad shape B=%lld V=%lld (1 to 2^20)", fn, (long long)B, (long long)V);
    if (dtype != WALSH_F32 && dtype != WALSH_BF16) return set_error(WALSH_ENOTSUP, "%s: dtype %d", fn, dtype);
    if (B == 0) return WALSH_OK;
    if (!logits || !u || !out) return set_error(WALSH_EINVAL, "%s: null pointer", fn);
    if (B > 1 && ld < V) return set_error(WALSH_EINVAL, "%s: row stride %lld for %lld logits", fn, (long long)ld, (long long)V);
    const SampleArgs a{logits, ld, V, u, temperature, top_p, min_p, top_k, temperature0, top_p0, min_p0, top_k0, out};
    const dim3 G((unsigned)B), N(kSmThreads);
    hipStream_t s = (hipStream_t)stream;
    const uint32_t lds = (uint32_t)sizeof(SmShared);
    if (dtype == WALSH_BF16) launch(sample_kernel<uint16_t>, G, N, lds, s, a);
    else launch(sample_kernel<float>, G, N, lds, s, a);
    return check_hip(hipGetLastError(), fn);
}
