// The next token of every row of logits, from a given uniform number u:
//     z_i = l_i / T,   w_i = exp(z_i - max z)
//   top-k   the k largest l (of equal ones the lowest indexes first)
//   top-p   of these, in the same order, a token stays while the weight before
//           it is below p of their sum (the first always stays, p <= 0: alone)
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
// w * ceil(V / 1024) * 64 on, 64 at a time, held in registers up to 57,344
// tokens.  Three walks over the row: its maximum, the histogram, and the
// tokens that the histogram leaves in question, each wavefront's into a list
// in LDS; what follows works on the lists, or, where one overflows (nothing
// filtered, or thousands kept), on the row again, out of the L2.
// Bound by that chain, not by memory: 50,257 logits in bf16 with top-k 50 and
// top-p 0.95 take 24 us for one row (load and maximum 5, histogram 5, search 2,
// the rest, half of it, lists, cut and draw) and 56 us for 256 rows of float32
// with every filter, one row to a CU.  Past the registers a row is read again
// at every walk: 65,536 and 131,072 logits take 38 and 58 us.  top-p without
// top-k adds the weights of all tokens in 64 bits: 50 to 62 us, 131 to 179 for
// 131,072.
#include "common.h"

namespace walsh {

constexpr int kSmWaves = 16;
constexpr int kSmThreads = 64 * kSmWaves;
constexpr int kSmBins = 2048, kSmList = 2048;
constexpr int kSmKept = 512;                    // tokens of a wavefront's list
constexpr int kSmStep = 8;                      // steps of a walk between its marks
constexpr int kSmParts = 16;                    // parts of a wavefront's walk with sums of their own
constexpr float kSmBinsPer2 = 64.f;             // bins to a factor of two

typedef unsigned long long u64;

struct SampleArgs {
    const void *logits;
    int64_t ld, V;
    const float *u, *temperature, *top_p, *min_p;   // [B], or null and the value below
    const int *top_k;
    float temperature0, top_p0, min_p0;
    int top_k0;
    int64_t *out;
};

// Order-preserving integer of a float (no NaN; -0 counts as 0), and back.
__device__ __forceinline__ uint32_t sm_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float sm_value(uint32_t key) {
    return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
}

struct SmShared {
    u64 mass[kSmBins];
    uint32_t count[kSmBins];
    uint32_t list[kSmList];                     // keys of a bin
    uint2 kept[kSmWaves][kSmKept];              // (key, index) of the tokens in question, by wavefront
    u64 wsum[kSmWaves], part[kSmWaves][kSmParts];
    uint32_t wcnt[kSmWaves];
    float wmax[kSmWaves];
    // results of a search
    uint32_t n, kmin, kmax, before;
    u64 mbefore;
    int bin, over[2], edge;
};

__device__ __forceinline__ u64 shfl64(u64 v, int src) {
    return ((u64)(uint32_t)__shfl((int)(v >> 32), src) << 32) | (uint32_t)__shfl((int)(uint32_t)v, src);
}
__device__ __forceinline__ u64 xor64(u64 v, int o) {
    return ((u64)(uint32_t)__shfl_xor((int)(v >> 32), o) << 32) | (uint32_t)__shfl_xor((int)(uint32_t)v, o);
}
// Inclusive sums over the wavefront's lanes.
__device__ __forceinline__ void wave_scan(uint32_t &c, u64 &m, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t oc = (uint32_t)__shfl_up((int)c, o);
        const u64 om = ((u64)(uint32_t)__shfl_up((int)(m >> 32), o) << 32) | (uint32_t)__shfl_up((int)(uint32_t)m, o);
        if (lane >= o) c += oc, m += om;
    }
}
__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += xor64(v, o);
    return v;
}
// What the wavefronts left in wcnt / wsum: before this one, and in all.
__device__ __forceinline__ void waves_before(const SmShared &sh, int wave, int lane, uint32_t &c, u64 &m, u64 &all) {
    const int w = lane & (kSmWaves - 1);
    uint32_t ci = w < wave ? sh.wcnt[w] : 0;
    u64 ms = sh.wsum[w], mi = w < wave ? ms : 0;
#pragma unroll
    for (int o = 1; o < kSmWaves; o <<= 1) ci += (uint32_t)__shfl_xor((int)ci, o), mi += xor64(mi, o), ms += xor64(ms, o);
    c = ci, m = mi, all = ms;
}

// The row's weights.
struct SmWeights {
    float m, chi, clo;     // the maximum (finite); log2(e) / T in two parts
    __device__ __forceinline__ float of(float x) const {            // 0 .. 1
        const float s = x - m;
        // (far below what counts the two parts might pass float32 with opposite signs)
        return s * chi > -150.f ? __builtin_amdgcn_exp2f(fmaf(s, chi, s * clo)) : 0.f;
    }
    // of() in units of 2^-44, by the addition of 1.5 * 2^8: 44 fraction bits are left below it
    static __device__ __forceinline__ u64 fixed(float w) {
        return (u64)__double_as_longlong((double)w + 384.0) - 0x4078000000000000ull;
    }
    __device__ __forceinline__ u64 mass(float x) const { return fixed(of(x)); }
    __device__ __forceinline__ int bin(float x) const {             // monotone in x; what is no number (0 times -inf): last
        const float y = (x - m) * (chi * -kSmBinsPer2);
        return y < (float)(kSmBins - 1) ? (int)y : kSmBins - 1;
    }
    // a value that every token of bins 0 .. q lies at or above
    __device__ __forceinline__ float floor_of(int q) const {
        const float r = ((float)q + 1.5f) / (chi * kSmBinsPer2);
        return q >= kSmBins - 1 ? -INFINITY : m - r - 1e-5f * (r + fabsf(m));
    }
    // and one that no token of bin q lies above
    __device__ __forceinline__ float ceiling_of(int q) const {
        const float r = fmaxf((float)q - 0.5f, 0.f) / (chi * kSmBinsPer2);
        return q == 0 ? INFINITY : m - r + 1e-5f * (r + fabsf(m));
    }
};

// The tokens that a wavefront walks, 64 at a time and in index order.
// each(f, mark): f(step, there, value) with every lane, mark(steps done) after
// every kSmStep steps and the last.  What is not there has no number as value.
template <typename T, int U> struct SmRow {                          // U: loads on their way together
    const T *p;
    int base, n, end;      // first index of the lane, steps, past the last index
    bool inf;              // the maximum is infinite: it counts as 0, the rest as -inf
    __device__ __forceinline__ SmRow(const T *row, int V, int wave, int lane) {
        n = (V + kSmThreads - 1) / kSmThreads;
        p = row;
        base = wave * n * 64 + lane;
        end = min(V, (wave + 1) * n * 64);
        inf = false;
    }
    __device__ __forceinline__ int index(int i) const { return base + 64 * i; }
    __device__ __forceinline__ int index_anew(int i) const {        // not kept in a register from an earlier use
        int at = base;
        asm volatile("" : "+v"(at));
        return at + 64 * i;
    }
    __device__ __forceinline__ float value(float v) const {          // what is no number counts as -inf
        v = fmaxf(v, -INFINITY);
        return inf ? (v == INFINITY ? 0.f : -INFINITY) : v;
    }
    // some element of the row, whether or not step i has one: no branch around the load
    __device__ __forceinline__ float some(int i) const { return Act<T>::load(p + max(0, min(index(i), end - 1))); }
    template <typename F, typename M> __device__ __forceinline__ void each(int i0, int i1, F f, M mark) const {
        for (int i = i0; i < i1; i += U) {
            float v[U];
#pragma unroll
            for (int j = 0; j < U; ++j) v[j] = some(i + j);
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const float x = index(i + j) < end ? value(v[j]) : NAN;
                if (i + j < i1) f(i + j, x == x, x);
                if (i + j < i1 && ((i + j + 1) % kSmStep == 0 || i + j + 1 == i1)) mark(i + j + 1);
            }
        }
    }
};
struct SmKeptRow {
    const uint2 *p;
    int lane, n, end;
    __device__ __forceinline__ SmKeptRow(const uint2 *list, int count, int lane_) {
        p = list, lane = lane_, end = count, n = (count + 63) / 64;
    }
    __device__ __forceinline__ int index(int i) const { return lane + 64 * i < end ? (int)p[lane + 64 * i].y : 0; }
    __device__ __forceinline__ int index_anew(int i) const { return index(i); }
    template <typename F, typename M> __device__ __forceinline__ void each(int i0, int i1, F f, M mark) const {
        for (int i = i0; i < i1; ++i) {
            const bool there = lane + 64 * i < end;
            f(i, there, there ? sm_value(p[lane + 64 * i].x) : NAN);
        }
        if (i1 > i0) mark(i1);
    }
};

// A threshold: tokens with a larger key stay, and the first `ties` of the
// `equal` ones with this key.
struct SmCut {
    uint32_t key, ties, equal;
};

// The first bin, in order from the maximum, at whose end the running count or
// weight reaches the need; with what lies before it.  by_mass with share >= 0:
// the need is that share of the whole.  Returns the need.  All threads.
__device__ __forceinline__ u64 sm_find_bin(SmShared &sh, int nbins, bool by_mass, uint32_t need, u64 mneed, float share) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = nbins > kSmThreads ? nbins / kSmThreads : 1;
    uint32_t c = 0;
    u64 m = 0;
    const bool mine = tid * per < nbins;
    if (mine)
        for (int i = 0; i < per; ++i) c += sh.count[tid * per + i], m += sh.mass[tid * per + i];
    uint32_t ci = c, c0;
    u64 mi = m, m0, all;
    wave_scan(ci, mi, lane);
    if (lane == 63) sh.wcnt[wave] = ci, sh.wsum[wave] = mi;
    __syncthreads();
    waves_before(sh, wave, lane, c0, m0, all);
    if (by_mass && share >= 0.f) {
        const double t = ceil((double)share * (double)all);
        mneed = t >= (double)all ? all : t > 1. ? (u64)t : 1ull;
    }
    c0 += ci - c, m0 += mi - m;
    if (mine && (by_mass ? m0 < mneed && mneed <= m0 + m : c0 < need && need <= c0 + c)) {   // one thread
        for (int i = 0; i < per; ++i) {
            const uint32_t cb = sh.count[tid * per + i];
            const u64 mb = sh.mass[tid * per + i];
            if (by_mass ? mneed <= m0 + mb : need <= c0 + cb) {
                sh.bin = tid * per + i, sh.before = c0, sh.mbefore = m0;
                break;
            }
            c0 += cb, m0 += mb;
        }
    }
    __syncthreads();
    return mneed;
}

// The tokens of the search's bin: their number, range and, as far as they fit,
// a list of their keys.  sm_open before, by all threads; then sm_put of each.
__device__ __forceinline__ void sm_open(SmShared &sh) {
    if (threadIdx.x == 0) sh.n = 0, sh.kmin = 0xffffffffu, sh.kmax = 0;
    __syncthreads();
}
__device__ __forceinline__ void sm_put(SmShared &sh, uint32_t key) {
    const uint32_t at = atomicAdd(&sh.n, 1u);
    if (at < kSmList) sh.list[at] = key;
    atomicMin(&sh.kmin, key);
    atomicMax(&sh.kmax, key);
}

// The cut within bin `sh.bin`, among the tokens put (where they overflow the
// list, again those of the bin from key `least` on).  All threads.
template <typename Row>
__device__ __forceinline__ SmCut sm_select(SmShared &sh, const Row &row, const SmWeights &wt, bool by_mass, uint32_t need,
                                           u64 mneed, uint32_t least) {
    const int tid = threadIdx.x, bin = sh.bin;
    uint32_t before = sh.before;
    u64 mbefore = sh.mbefore;
    const uint32_t n = sh.n;
    uint32_t lo = sh.kmin, equal = n;                               // the cut's key lies in lo .. lo + 2^bits - 1
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
            row.each(0, row.n, [&](int, bool there, float x) {
                if (there && wt.bin(x) == bin && sm_key(x) >= least) put(sm_key(x));
            }, [](int) {});
        }
        __syncthreads();
        sm_find_bin(sh, 256, by_mass, need - before, mneed - mbefore, -1.f);
        before += sh.before, mbefore += sh.mbefore;
        lo += (uint32_t)(((1u << d) - 1) - sh.bin) << sft;
        equal = sh.count[sh.bin];
        bits = sft;
    }
    // equal ones before the need is reached (w > 0, or nothing would be left to reach)
    const u64 w = wt.mass(sm_value(lo)), left = mneed - mbefore;
    const uint32_t ties = by_mass ? (w ? (uint32_t)((left + w - 1) / w) : 1u) : need - before;
    return SmCut{lo, ties, equal};
}

// From the first search's bin (sh.bin, sh.before, sh.mbefore) to the token.
// walk: row.each of everything, or the same out of registers; listed: tokens
// that hold all of the first search's bin, if so_listed.
template <typename Row, typename Walk>
__device__ __forceinline__ void sm_finish(SmShared &sh, const Row &row, Walk walk, const SmKeptRow &listed,
                                          bool so_listed, const SmWeights &wt, bool by_k, bool by_p, uint32_t k, float top_p, u64 need,
                                          float min_p, float u, int64_t *out) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    auto nothing = [](int) {};
    // the keys of the search's bin from `least` on
    auto collect = [&](const auto &from, uint32_t least) {
        const int bin = sh.bin;
        const float lo = wt.floor_of(bin);
        sm_open(sh);
        from.each(0, from.n, [&](int, bool there, float x) {
            if (!__any(x >= lo)) return;
            if (there && wt.bin(x) == bin && sm_key(x) >= least) sm_put(sh, sm_key(x));
        }, nothing);
        __syncthreads();
    };
    SmCut cut{0u, 0u, 0u};
    if (by_k || by_p) {
        if (so_listed) collect(listed, 0u);
        else collect(row, 0u);
    }
    if (by_k) {
        cut = sm_select(sh, row, wt, false, k, 0ull, 0u);
        if (by_p) {
            // the histogram of what top-k keeps; the ties at its cut weigh the
            // same, so any of them stand for the first ones
            __syncthreads();
            for (int i = tid; i < kSmBins; i += kSmThreads) sh.count[i] = 0, sh.mass[i] = 0;
            __syncthreads();
            row.each(0, row.n, [&](int, bool there, float x) {
                if (there && sm_key(x) > cut.key) atomicAdd(&sh.mass[wt.bin(x)], wt.mass(x));
            }, nothing);
            if (tid == 0) {
                const float x = sm_value(cut.key);
                atomicAdd(&sh.mass[wt.bin(x)], wt.mass(x) * cut.ties);
            }
            __syncthreads();
            need = sm_find_bin(sh, kSmBins, true, 0u, 0ull, top_p);
            collect(row, cut.key);
        }
    }
    if (by_p) {
        const SmCut c = sm_select(sh, row, wt, true, 0u, need, cut.key);
        if (!by_k || c.key > cut.key) cut = c;
        else cut.ties = min(cut.ties, c.ties);
    }
    // What stays: values above xc, and those equal to it below index `edge`.
    const bool all_stay = !by_k && !by_p;
    const float xc = all_stay ? -INFINITY : sm_value(cut.key);
    int edge = 0x7fffffff;
    if (!all_stay && cut.ties < cut.equal) {
        // the index of the first equal one that goes
        uint32_t t = 0, before;
        walk([&](int, bool there, float x) { t += __popcll(__ballot(there && x == xc)); }, nothing);
        __syncthreads();
        if (lane == 0) sh.wcnt[wave] = t, sh.wsum[wave] = 0;
        __syncthreads();
        u64 m0, m1;
        waves_before(sh, wave, lane, before, m0, m1);
        if (before <= cut.ties && cut.ties < before + t) {          // one wavefront's
            row.each(0, row.n, [&](int i, bool there, float x) {
                const u64 eq = __ballot(there && x == xc);
                const uint32_t here = __popcll(eq & ((1ull << lane) - 1));
                if (there && x == xc && before + here == cut.ties) sh.edge = row.index(i);
                before += __popcll(eq);
            }, nothing);
        }
        __syncthreads();
        edge = sh.edge;
    }
    auto rest = [&](int i, bool there, float x) {
        const float w = wt.of(x);
        bool stay = there && x >= xc && w >= min_p;
        if (edge != 0x7fffffff) stay = stay && (x > xc || row.index_anew(i) < edge);
        return stay ? SmWeights::fixed(w) : 0ull;
    };
    // sums of the parts of the walk, then of wavefronts
    const int step = kSmStep * ((row.n + kSmStep * kSmParts - 1) / (kSmStep * kSmParts));
    u64 mine = 0, s = 0;
    walk([&](int i, bool there, float x) { s += rest(i, there, x); },
         [&](int done) {
             if (done % step && done < row.n) return;
             s = wave_sum64(s);
             if (lane == 0) sh.part[wave][(done - 1) / step] = s;
             mine += s;
             s = 0;
         });
    __syncthreads();
    if (lane == 0) sh.wsum[wave] = mine;
    __syncthreads();
    uint32_t c0;
    u64 run, all;
    waves_before(sh, wave, lane, c0, run, all);
    if (all == 0) {                                                 // min_p above 1, or not a number
        if (tid == 0) *out = -1;
        return;
    }
    const double ut = (double)(u > 0.f ? u : 0.f) * (double)all;
    u64 thr = ut < (double)all ? (u64)ut : all - 1;                 // the first running sum above this
    if (thr >= all) thr = all - 1;
    if (thr < run || thr >= run + mine) return;                     // another wavefront's
    int j = 0;
    while (run + sh.part[wave][j] <= thr) run += sh.part[wave][j++];
    bool found = false;
    row.each(j * step, min(row.n, (j + 1) * step), [&](int i, bool there, float x) {
        if (found) return;
        u64 v = rest(i, there, x);
        if (!__any(v != 0)) return;
        uint32_t none = 0;
        wave_scan(none, v, lane);
        const u64 hit = __ballot(run + v > thr);
        if (hit) {
            if (lane == (int)__ffsll((long long)hit) - 1) *out = row.index(i);
            found = true;
        }
        run += shfl64(v, 63);
    }, nothing);
}

// NPT: values that a lane holds in registers (V <= NPT * 1024), or 0.
template <typename T, int NPT> __global__ __launch_bounds__(kSmThreads) void sample_kernel(SampleArgs a) {
    extern __shared__ __align__(16) unsigned char sm_smem[];
    SmShared &sh = *(SmShared *)sm_smem;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    SmRow<T, NPT ? 4 : 16> row((const T *)a.logits + b * a.ld, (int)a.V, wave, lane);
    float v[NPT ? NPT : 1];
    if constexpr (NPT > 0) {
#pragma unroll
        for (int i = 0; i < NPT; ++i) {
            v[i] = row.some(i);
            if (i % kSmStep == kSmStep - 1) __builtin_amdgcn_sched_barrier(0);   // (addresses one after the other)
        }
    }
    const float temp = a.temperature ? a.temperature[b] : a.temperature0;
    const float share = a.top_p ? a.top_p[b] : a.top_p0, min_p = a.min_p ? a.min_p[b] : a.min_p0;
    const float top_p = share < 0.f ? 0.f : share;                  // (what is no number keeps all)
    const int top_k = a.top_k ? a.top_k[b] : a.top_k0;
    const float u = a.u[b];
    for (int i = tid; i < kSmBins; i += kSmThreads) sh.count[i] = 0, sh.mass[i] = 0;
    if (tid == 0) sh.over[0] = sh.over[1] = 0;
    auto walk = [&](auto f, auto mark) {
        if constexpr (NPT > 0) {
#pragma unroll
            for (int g = 0; g < NPT; g += kSmStep) {
                if (g < row.n) {                                    // the last steps may lie past the row
#pragma unroll
                    for (int j = 0; j < kSmStep; ++j) {
                        float x = v[g + j];
                        asm volatile("" : "+v"(x));                 // (whether it is there is found anew, not kept)
                        f(g + j, x == x, x);
                    }
                    mark(min(g + kSmStep, row.n));
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
            row.each(0, row.n, f, mark);
        }
    };
    auto nothing = [](int) {};

    float m = -INFINITY;
    if constexpr (NPT > 0) {
        // from here on what lies past the row is no number
        int base = row.base;
        asm volatile("" : "+v"(base));                              // (the addresses are not kept for this)
#pragma unroll
        for (int i = 0; i < NPT; ++i) {
            v[i] = i < row.n && base + 64 * i < row.end ? row.value(v[i]) : NAN;
            m = fmaxf(m, v[i]);
            if (i % kSmStep == kSmStep - 1) __builtin_amdgcn_sched_barrier(0);
        }
    } else {
        walk([&](int, bool, float x) { m = fmaxf(m, x); }, nothing);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (lane == 0) sh.wmax[wave] = m;
    __syncthreads();
    m = sh.wmax[lane & (kSmWaves - 1)];
#pragma unroll
    for (int o = 1; o < kSmWaves; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (m == -INFINITY) {
        if (tid == 0) a.out[b] = -1;
        return;
    }
    if (m == INFINITY) {                                            // the infinite ones share the weight
        row.inf = true;
        m = 0.f;
        if constexpr (NPT > 0) {
#pragma unroll
            for (int i = 0; i < NPT; ++i) v[i] = v[i] == v[i] ? row.value(v[i]) : v[i];
        }
    }
    const bool greedy = !(temp > 0.f);
    const double c = greedy ? 1. : fmin(1.4426950408889634074 / (double)temp, 1e30);   // (1e30: only the maximum counts)
    const SmWeights wt{m, (float)c, (float)(c - (double)(float)c)};
    const bool by_k = greedy || (top_k > 0 && top_k < a.V), by_p = !greedy && top_p < 1.f;
    const uint32_t k = greedy ? 1u : (uint32_t)top_k;
    u64 need = 0;
    float least = -INFINITY;                                        // no token that may stay lies below
    if (by_k || by_p) {
        if (by_k)
            walk([&](int, bool there, float x) {
                if (there) atomicAdd(&sh.count[wt.bin(x)], 1u);
            }, nothing);
        else
            walk([&](int, bool there, float x) {
                if (there) atomicAdd(&sh.mass[wt.bin(x)], wt.mass(x));
            }, nothing);
        __syncthreads();
        need = sm_find_bin(sh, kSmBins, !by_k, k, 0ull, top_p);
        least = wt.floor_of(sh.bin);
    } else if (min_p > 0.f) {
        least = wt.floor_of((int)fminf(ceilf(-log2f(min_p) * kSmBinsPer2), (float)(kSmBins - 1)));
    }
    // the tokens still in question into the wavefronts' lists; where a list
    // overflows, those of the search's bin alone
    float most = INFINITY;
    int kept = 0, pass = 0;
    for (; pass < 2 && least > -INFINITY; ++pass) {
        kept = 0;
        walk([&](int i, bool, float x) {
            const u64 who = __ballot(x >= least && x <= most);
            if (!who) return;
            const int at = kept + __popcll(who & ((1ull << lane) - 1));
            if (x >= least && x <= most && at < kSmKept) sh.kept[wave][at] = make_uint2(sm_key(x), (uint32_t)row.index_anew(i));
            kept += __popcll(who);
        }, nothing);
        if (kept > kSmKept && lane == 0) sh.over[pass] = 1;
        __syncthreads();
        if (!sh.over[pass]) break;
        if (!by_k && !by_p) pass = 1;
        else if (pass == 0) least = wt.floor_of(sh.bin), most = wt.ceiling_of(sh.bin);
    }
    const SmKeptRow mine(sh.kept[wave], min(kept, kSmKept), lane);
    const bool listed = pass < 2 && least > -INFINITY;
    if (listed && pass == 0)
        sm_finish(sh, mine, [&](auto f, auto mark) { mine.each(0, mine.n, f, mark); }, mine, true, wt, by_k, by_p, k, top_p,
                  need, min_p, u, a.out + b);
    else
        sm_finish(sh, row, walk, mine, listed, wt, by_k, by_p, k, top_p, need, min_p, u, a.out + b);
}

template <typename T> static void sample_launch(const SampleArgs &a, unsigned rows, hipStream_t s) {
    const dim3 G(rows), N(kSmThreads);
    const uint32_t lds = (uint32_t)sizeof(SmShared);
    // registers for as many values as leave 16 wavefronts on a CU
    if (a.V <= 16 * kSmThreads) launch(sample_kernel<T, 16>, G, N, lds, s, a);
    else if (a.V <= 56 * kSmThreads) launch(sample_kernel<T, 56>, G, N, lds, s, a);
    else launch(sample_kernel<T, 0>, G, N, lds, s, a);
}

}  // namespace walsh

using namespace walsh;

WALSH_EXPORT int walsh_sample(const void *logits, int64_t ld, int64_t B, int64_t V, const float *u,
                              const float *temperature, float temperature0, const int *top_k, int top_k0,
                              const float *top_p, float top_p0, const float *min_p, float min_p0, int64_t *out, int dtype,
                              void *stream) {
    const char *fn = "walsh_sample";
    if (B < 0 || B >= (1 << 22) || V < 1 || V >= (1 << 20))   // (2^20 weights of 2^44 would pass 64 bits)
        return set_error(WALSH_EINVAL, "%s: bad shape B=%lld (below 2^22) V=%lld (1 to 2^20 - 1)", fn, (long long)B, (long long)V);
    if (dtype != WALSH_F32 && dtype != WALSH_BF16) return set_error(WALSH_ENOTSUP, "%s: dtype %d", fn, dtype);
    if (B == 0) return WALSH_OK;
    if (!logits || !u || !out) return set_error(WALSH_EINVAL, "%s: null pointer", fn);
    if (B > 1 && ld < V) return set_error(WALSH_EINVAL, "%s: row stride %lld for %lld logits", fn, (long long)ld, (long long)V);
    const SampleArgs a{logits, ld, V, u, temperature, top_p, min_p, top_k, temperature0, top_p0, min_p0, top_k0, out};
    if (dtype == WALSH_BF16) sample_launch<uint16_t>(a, (unsigned)B, (hipStream_t)stream);
    else sample_launch<float>(a, (unsigned)B, (hipStream_t)stream);
    return check_hip(hipGetLastError(), fn);
}
