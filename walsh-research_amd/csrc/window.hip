// Attention over a sliding window and a few first tokens, forward and
// backward.  Query i of Tq stands at position p = i + Tk - Tq of its sequence
// and sees the keys
//     j <= p  and  (j > p - W  or  j < S)
// (W the window, S the number of first tokens that stay visible; W <= 0: no
// window), and a position at or past the sequence's length sees nothing.
//     o = softmax(c q K^T) V,      lse = log sum exp(c q K^T)
// A row that sees nothing gives zeros and lse = -inf.  The backward rebuilds
// P = exp(c q K^T - lse) tile by tile:
//     Delta = rowsum(do o),  dV = P^T do,  dS = c P (do V^T - Delta),
//     dQ = dS K,  dK = dS^T Q
// with query heads h sharing the keys and values of head h / (H / G).
//
// Matrix layout.  Everything is a 32x32 product tile over 16 (bf16:
// v_mfma_f32_32x32x16_bf16; float32: eight v_mfma_f32_32x32x2_f32), operands
// eight consecutive elements per lane.  Scores are formed transposed to the
// operand that stays in registers, so a lane holds 16 scores of ONE query
// (forward, dQ) or ONE key (dK, dV) and the softmax weights are, as they come
// out, the second operand of the next product.  A tile of 32-bit results has
// its rows at 8 g + 4 hi + i (hi the lane's half), so product slot 8 hi + e
// stands for row 16 t + 4 hi + e (e < 4) or 16 t + 8 + 4 hi + e - 4, and the
// first operand is read in that order: bf16 with the transposing LDS load
// (four rows of a column per lane), float32 with single loads.  One LDS copy
// of a tile, row-major, so serves both the products over its columns and over
// its rows.
//
// Roundings.  Scores, maxima, sums, lse, Delta and all accumulators are
// float32.  bf16 tensors have their weights P and dS rounded to bf16 for the
// second products (the matrix cores' operand type; off by up to 2^-8 each, the
// size of the inputs' own rounding), and dQ at D <= 32 takes dS in two parts.
// A row is normalised by the sum of its rounded weights, lse by that of the
// unrounded ones: o is then a mean of the values, and a vector common to them
// passes through unchanged.  (Normalised by the unrounded sum it came out
// (1 + 2^-9 or so) times as large, which Delta carried into dS: values within 1
// of 4 in every element, and a gradient of o with a mean of 1, had dQ 1.0 to
// 3.6e-2 and dK 0.5 to 3.7e-2 off.  It costs 2 to 6% of the forward where lse is
// asked for, nothing measurable where it is not.)  Relative errors are
// 2.2e-3 for o and 2.3 to 2.4e-3 for the gradients, where the rounding of the
// results alone leaves 1.6 to 1.7e-3.  Two parts everywhere reach those, for
// 23 to 34% more time of the forward and 18 to 32% of the backward (2 x 32
// heads of 128, 4,096 tokens, window 1,024: 185 us and 228, 547 and 680).
#include "tiles.h"

namespace walsh {

// ---------------------------------------------------------------- arguments
struct WinTensor {
    int64_t sb, sh, st;   // element (b, h, t, d) at b*sb + h*sh + t*st + d
};
struct WinArgs {
    const void *q, *k, *v;
    const int *lengths;   // [B] or null
    void *o;
    float *lse;           // [B, H, Tq]
    void *rest;           // [B, H, Tq, D] or null (bf16): what rounding took from o
    WinTensor sq, skv, so;
    int B, H, G, Tq, Tk, W, S;
    float sl2;            // scale * log2(e)
    // backward
    const void *go;
    void *dq, *dk, *dv;   // dense [B, H, Tq, D], [B, G, Tk, D]
    WinTensor sgo;
    float *stat;          // [2][B, H, Tq]: lse * log2(e) (inf for rows that see nothing), Delta
    float scale;
    float *part;          // partial dK, dV of key blocks whose queries are split
    int nb, nsb, nn, ns;  // key blocks; those with first tokens; splits of the others' and of their queries
};

// Key positions of a sequence: all of Tk, or its length within it.
__device__ __forceinline__ int win_len(const WinArgs &a, int b) {
    return a.lengths ? uniform(max(0, min(a.lengths[b], a.Tk))) : a.Tk;
}
// The chunks of ROWS keys that positions p0 .. p1 see: n chunks, the first ns
// of them the first tokens' (chunks 0 ..), the rest from chunk lo.
struct Chunks {
    int lo, ns, n;
    __device__ __forceinline__ int at(int i) const { return i < ns ? i : lo + i - ns; }
};
template <int ROWS> __device__ __forceinline__ Chunks win_chunks(const WinArgs &a, int p0, int p1) {
    Chunks c;
    c.lo = a.W > 0 && p0 >= a.W ? (p0 - a.W + 1) / ROWS : 0;
    c.ns = min((a.S + ROWS - 1) / ROWS, c.lo);
    c.n = p1 < 0 ? 0 : c.ns + p1 / ROWS - c.lo + 1;
    return c;
}
// How keys k0 .. k0 + n - 1 look to positions pa .. pb: 0 hidden from all, 2 seen by all, 1 mixed.
__device__ __forceinline__ int win_kind(const WinArgs &a, int k0, int n, int pa, int pb) {
    if (k0 > pb || (a.W > 0 && k0 + n <= pa - a.W + 1 && k0 >= a.S)) return 0;
    return k0 + n - 1 <= pa && (a.W <= 0 || k0 > pb - a.W || k0 + n <= a.S) ? 2 : 1;
}
// Of 32 consecutive keys from k0 the ones that position p sees, and of 32
// consecutive positions from p0 the ones that see key j, as bits; and scores
// by such bits: row 8 (r / 4) + 4 hi + r % 4 of a result is bit 8 (r / 4) + r % 4
// of bits >> 4 hi.  (Three instructions a score; comparing positions took eight.)
__device__ __forceinline__ uint32_t bits_below(int n) { return (uint32_t)((1ull << max(0, min(n, 32))) - 1); }
__device__ __forceinline__ uint32_t win_keys(const WinArgs &a, int p, int k0) {
    const int n = p - k0 + 1, W = a.W > 0 ? a.W : 1 << 29;
    return (bits_below(n) & ~bits_below(n - W)) | bits_below(min(n, a.S - k0));
}
__device__ __forceinline__ uint32_t win_rows(const WinArgs &a, int p0, int j) {
    const int n = j - p0, W = a.W > 0 ? a.W : 1 << 29;
    return ~bits_below(n) & (j < a.S ? ~0u : bits_below(n + W));
}
__device__ __forceinline__ void win_hide(f32x16 &s, uint32_t seen, int hi) {
    const uint32_t hidden = ~seen >> (4 * hi);
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const uint32_t all = (uint32_t)((int)(hidden << (31 - 8 * (r >> 2) - (r & 3))) >> 31);   // the bit, 32 times
        s[r] = __uint_as_float((all & 0xff800000u) | (~all & __float_as_uint(s[r])));
    }
}

// Four values of an output row, zeros where the row sees nothing, and what
// their rounding took from them.
template <typename T> __device__ __forceinline__ void win_store(const WinArgs &a, T *o, int64_t dense, f32x4 v, bool live) {
    v = live ? v : f32x4{0.f, 0.f, 0.f, 0.f};
    store4(o, v);
    if constexpr (sizeof(T) == 2) {
        if (a.rest) {
            const uint32_t u0 = pack_bf16x2(v.x, v.y), u1 = pack_bf16x2(v.z, v.w);
            store4((T *)a.rest + dense, v - f32x4{__uint_as_float(u0 << 16), __uint_as_float(u0 & 0xffff0000u),
                                                  __uint_as_float(u1 << 16), __uint_as_float(u1 & 0xffff0000u)});
        }
    }
}

// Work item of this workgroup: workgroups go to the 8 XCDs in turn, so XCD x
// takes items x n/8 ..: neighbouring items, which share keys, share an L2.
// Returns -1 past the last one (the grid is a multiple of 8).
__device__ __forceinline__ int xcd_item(int n) {
    const int per = (n + 7) / 8, id = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
    return ((int)blockIdx.x >> 3) < per && id < n ? id : -1;
}

// ---------------------------------------------------------------- forward
// A workgroup takes 128 queries of a head, 32 per wavefront, over the tiles of
// keys that any of them sees, two tiles of K and V in LDS at a time; blocks of
// 32 keys that none of a wavefront's queries sees are passed over, and only
// those seen in part are masked.  Bound by the matrix products and the
// softmax's vector instructions, which two wavefronts per SIMD overlap in part:
// 2 x 32 heads of 128, 8,192 tokens, window 1,024, bf16: 350 to 390 us alone
// (from one card to another) and 480 in a row, at the clock that the card holds
// then: 740 to 660 and 540 TFLOP/s of what is visible (a large product reaches
// 1,210).  A block's scores, softmax and second products depend on each other,
// and blocks follow one another strictly: the branch around the rescaling ends
// the compiler's schedule.  Of 362 us without the loads' present order, 51 went
// without the softmax, 54 without the tiles' loads.  256 queries on a tile took 394 us, 64 queries per wavefront (each
// LDS operand used twice, at twice the accumulators) 680, three to four tiles
// on their way 440.  Heads of 16: 28 to 31 us for 8 x 32 heads, 1,024 tokens, window
// 256, the exponentials and masks of short products.  float32,
// of which the matrix cores do an eighth of bf16's (154 TFLOP/s in a large
// product): heads of 128, 64, 32 and 16 reach 103, 99, 82 and 43 TFLOP/s (2 x 32
// heads of 64, 4,096 tokens, window 1,024: 608 us).
constexpr int kWinWaves = 4;
constexpr int kWinQ = 32 * kWinWaves;   // queries (or keys, dK and dV) per workgroup
template <typename T, int D> struct WinCfg {
    static constexpr int KC = sizeof(T) == 4 && D == 128 ? 32 : 64;   // rows of a tile: four of them, 64 KB at most
    static constexpr int NK = D / 16;                                 // products over D
    static constexpr int ND = (D + 31) / 32;                          // 32-wide blocks of D
};

template <typename T, int D, bool LSE>
__global__ __launch_bounds__(64 * kWinWaves, sizeof(T) == 4 && D == 128 ? 1 : 2) void window_fwd_kernel(WinArgs a) {
    constexpr bool EXACT = LSE || sizeof(T) == 4, ROUNDED = sizeof(T) == 2;   // sums of the weights in use
    constexpr int KC = WinCfg<T, D>::KC, NK = WinCfg<T, D>::NK, ND = WinCfg<T, D>::ND, NJ = KC / 32;
    typedef Tile<T, D, KC> L;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int nqt = (a.Tq + kWinQ - 1) / kWinQ;
    const int id = xcd_item(nqt * a.H * a.B);
    if (id < 0) return;
    const int bh = uniform(id / nqt), qt = nqt - 1 - (id - bh * nqt);
    const int b = uniform(bh / a.H), h = bh - b * a.H, g = uniform(h / (a.H / a.G));
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 31, hi = lane >> 5;
    const int len = win_len(a, b), off = a.Tk - a.Tq;
    const int qi = qt * kWinQ + 32 * wave + n, p = qi + off;   // this lane's query and its position
    // positions of the workgroup and of the wavefront that have an output
    const int wlo = max(0, qt * kWinQ + off), whi = min(min(qt * kWinQ + kWinQ, a.Tq) - 1 + off, len - 1);
    const int pa = max(0, qt * kWinQ + 32 * wave + off), pb = min(qt * kWinQ + 32 * wave + 31 + off, len - 1);

    const bool live = p >= 0 && p < len;

    Frag<T> qf[NK];
    {
        const T *qp = (const T *)a.q + b * a.sq.sb + h * a.sq.sh + (int64_t)min(qi, a.Tq - 1) * a.sq.st;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) qf[kk] = load_frag(qp + 16 * kk + 8 * hi);
    }
    f32x16 acc[ND];
#pragma unroll
    for (int c = 0; c < ND; ++c) acc[c] = f32x16{};
    float m = kNoScore, l = 0.f, lr = 0.f;        // lr: of the weights as the products take them

    const T *kb = (const T *)a.k + b * a.skv.sb + g * a.skv.sh, *vb = (const T *)a.v + b * a.skv.sb + g * a.skv.sh;
    const Chunks ch = wlo <= whi ? win_chunks<KC>(a, wlo, whi) : Chunks{0, 0, 0};
    const typename L::template Loads<kWinWaves> loads(a.skv.st, wave, lane);
    auto fetch_k = [&](int i) { loads.go(smem + (i & 1) * 2 * L::BYTES, kb, a.skv.st, ch.at(i) * KC, len, wave); };
    auto fetch_v = [&](int i) { loads.go(smem + (i & 1) * 2 * L::BYTES + L::BYTES, vb, a.skv.st, ch.at(i) * KC, len, wave); };
    // a row's operands' addresses, held: worked out between the paced reads they cost a tenth of the time
    uint32_t ka[NK], va = L::col_base(smem + L::BYTES, lane);
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) ka[kk] = L::row_base(smem, n, hi) ^ L::row_step(kk);
    if (ch.n > 0) fetch_k(0), fetch_v(0);
    for (int i = 0; i < ch.n; ++i) {
        tiles_ready();
        const int k0 = ch.at(i) * KC;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int kind = pa <= pb ? win_kind(a, k0 + 32 * j, 32, pa, pb) : 0;
            // the next tile's loads in two bursts, each behind a product's
            if (i + 1 < ch.n) {
                if (j == 0) fetch_k(i + 1);
                if (j == NJ - 1) fetch_v(i + 1);
            }
            if (kind == 0) continue;
            f32x16 s = f32x16{};
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) mma(s, L::row_from(ka[kk] + 32 * j * L::ROWB, 0), qf[kk]);
            if constexpr (sizeof(T) == 2 && NK > 4) pace<1, NK, 4>();
            if (kind == 1) win_hide(s, win_keys(a, p, k0 + 32 * j), hi);
            float mx = s[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
            mx = half_max(mx);
            // the maximum moves only when some row of the wavefront would pass
            // 2^8: weights and sums stay within float32 and the rescaling of the
            // accumulators is rare
            if (__any(live && (mx - m) * a.sl2 > 8.f)) {
                const float mn = fmaxf(m, mx), al = __builtin_amdgcn_exp2f((m - mn) * a.sl2);
                m = mn;
                l *= al;
                lr *= al;
#pragma unroll
                for (int c = 0; c < ND; ++c) acc[c] *= al;
            }
            const float mo = -m * a.sl2;
            float w[16];
            [[maybe_unused]] float l0 = 0.f, l1 = 0.f;
#pragma unroll
            for (int r = 0; r < 16; ++r) w[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.sl2, mo));
            if constexpr (EXACT) {
#pragma unroll
                for (int r = 0; r < 16; r += 2) {
                    l0 += w[r];
                    l1 += w[r + 1];
                }
                l += l0 + l1;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                Frag<T> pf;
                pack(pf, w + 8 * t);
                if constexpr (ROUNDED) lr = add_all(lr, pf);
#pragma unroll
                for (int c = 0; c < ND; ++c) mma(acc[c], L::col_from(va, 32 * j + 16 * t, c), pf);
            }
        }
        const int other = i & 1 ? -2 * L::BYTES : 2 * L::BYTES;          // the next tile's buffer
        va += other;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) ka[kk] += other;
    }
    l = half_sum(l);
    lr = ROUNDED ? half_sum(lr) : l;
    if (qi >= a.Tq) return;
    const float inv = 1.f / lr;                   // (no row that sees a key has none but infinite scores' sum 0)
    T *op = (T *)a.o + b * a.so.sb + h * a.so.sh + (int64_t)qi * a.so.st;
#pragma unroll
    for (int c = 0; c < ND; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int d = 32 * c + 8 * t + 4 * hi;
            if (D % 32 && d >= D) continue;
            const f32x4 v = f32x4{acc[c][4 * t], acc[c][4 * t + 1], acc[c][4 * t + 2], acc[c][4 * t + 3]} * inv;
            win_store(a, op + d, (((int64_t)b * a.H + h) * a.Tq + qi) * D + d, v, live);
        }
    if (LSE && hi == 0)
        a.lse[((int64_t)b * a.H + h) * a.Tq + qi] = live ? (m * a.sl2 + log2f(l)) * (1.f / kLog2e) : -INFINITY;
}

// The same for grids that would leave most of the chip idle (a short part of a
// prompt, few heads): 32 queries per workgroup, whose four wavefronts take
// every fourth block of 32 keys, each with its own maximum, sum and
// accumulators, joined at the end.  Nothing is shared on the way: a wavefront
// reads its K rows straight into operands and V into LDS of its own, the next
// block's while it works on one.  777 queries of 8 heads of 64 in float32 on
// 1,301 keys, window 256: 41 us by four times 32 queries, 15 us so.
template <typename T, int D> struct WinSplitCfg {
    static constexpr int VB = Tile<T, D, 32>::BYTES;
    static constexpr int WAVE = 2 * VB > 32 * D * 4 ? 2 * VB : 32 * D * 4;   // two V tiles; at the end 32 rows of D
};
template <typename T, int D>
__global__ __launch_bounds__(64 * kWinWaves, sizeof(T) == 4 && D == 128 ? 1 : 2) void window_fwd_split_kernel(WinArgs a) {
    constexpr int NK = D / 16, ND = (D + 31) / 32;
    typedef Tile<T, D, 32> L;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ float stat[kWinWaves][3][32];      // maximum, both sums
    const int nqt = (a.Tq + 31) / 32;
    const int id = xcd_item(nqt * a.H * a.B);
    if (id < 0) return;
    const int bh = uniform(id / nqt), qt = nqt - 1 - (id - bh * nqt);
    const int b = uniform(bh / a.H), h = bh - b * a.H, g = uniform(h / (a.H / a.G));
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 31, hi = lane >> 5;
    const int len = win_len(a, b), off = a.Tk - a.Tq;
    const int qi = qt * 32 + n, p = qi + off;
    const int pa = max(0, qt * 32 + off), pb = min(min(qt * 32 + 32, a.Tq) - 1 + off, len - 1);

    Frag<T> qf[NK], kf[NK];
    {
        const T *qp = (const T *)a.q + b * a.sq.sb + h * a.sq.sh + (int64_t)min(qi, a.Tq - 1) * a.sq.st;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) qf[kk] = load_frag(qp + 16 * kk + 8 * hi);
    }
    f32x16 acc[ND];
#pragma unroll
    for (int c = 0; c < ND; ++c) acc[c] = f32x16{};
    float m = kNoScore, l = 0.f, lr = 0.f;
    const T *kb = (const T *)a.k + b * a.skv.sb + g * a.skv.sh, *vb = (const T *)a.v + b * a.skv.sb + g * a.skv.sh;
    const Chunks ch = pa <= pb ? win_chunks<32>(a, pa, pb) : Chunks{0, 0, 0};
    unsigned char *vl = smem + wave * WinSplitCfg<T, D>::WAVE;
    auto fetch = [&](int i, int buf) {
        const int k0 = ch.at(i) * 32;
        const T *kp = kb + (int64_t)min(k0 + n, len - 1) * a.skv.st + 8 * hi;   // (past the end: a row that is masked)
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) kf[kk] = load_frag(kp + 16 * kk);
        L::template fetch<1>(vl + buf * WinSplitCfg<T, D>::VB, vb, a.skv.st, k0, 0, len, 0, lane);
    };
    int i = wave, buf = 0;
    if (i < ch.n) fetch(i, 0);
    for (; i < ch.n; i += kWinWaves, buf ^= 1) {
        const int k0 = ch.at(i) * 32;
        wait_loads();
        f32x16 s = f32x16{};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) mma(s, kf[kk], qf[kk]);
        if (i + kWinWaves < ch.n) fetch(i + kWinWaves, buf ^ 1);
        if (win_kind(a, k0, 32, pa, pb) != 2) win_hide(s, win_keys(a, p, k0), hi);
        float mx = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[r]);
        mx = half_max(mx);
        if (__any(p >= 0 && p < len && (mx - m) * a.sl2 > 8.f)) {
            const float mn = fmaxf(m, mx), al = __builtin_amdgcn_exp2f((m - mn) * a.sl2);
            m = mn;
            l *= al;
            lr *= al;
#pragma unroll
            for (int c = 0; c < ND; ++c) acc[c] *= al;
        }
        const float mo = -m * a.sl2;
        float w[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            w[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.sl2, mo));
            l += w[r];
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            Frag<T> pf;
            pack(pf, w + 8 * t);
            if constexpr (sizeof(T) == 2) lr = add_all(lr, pf);
#pragma unroll
            for (int c = 0; c < ND; ++c) mma(acc[c], L::col(vl + buf * WinSplitCfg<T, D>::VB, 16 * t, c, lane), pf);
        }
    }
    l = half_sum(l);
    lr = sizeof(T) == 2 ? half_sum(lr) : l;
    // the wavefronts' parts: o = sum_w acc_w e^(m_w - m) / sum_w lr_w e^(m_w - m)
    wait_loads();
    float *av = (float *)vl;   // [32 queries][D] of this wavefront (its V is used up)
#pragma unroll
    for (int c = 0; c < ND; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int d = 32 * c + 8 * t + 4 * hi;
            if (D % 32 && d >= D) continue;
            store4(av + n * D + d, f32x4{acc[c][4 * t], acc[c][4 * t + 1], acc[c][4 * t + 2], acc[c][4 * t + 3]});
        }
    if (hi == 0) stat[wave][0][n] = m, stat[wave][1][n] = l, stat[wave][2][n] = lr;
    __syncthreads();
    for (int e = threadIdx.x; e < 32 * (D / 4); e += 64 * kWinWaves) {
        const int r = e / (D / 4), d = e % (D / 4) * 4, q = qt * 32 + r, pos = q + off;
        if (q >= a.Tq) break;
        const bool live = pos >= 0 && pos < len;
        float mm = stat[0][0][r], ll = 0.f, lt = 0.f;
#pragma unroll
        for (int w = 1; w < kWinWaves; ++w) mm = fmaxf(mm, stat[w][0][r]);
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < kWinWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f((stat[w][0][r] - mm) * a.sl2);
            v += load4((const float *)(smem + w * WinSplitCfg<T, D>::WAVE) + r * D + d) * f;
            ll += stat[w][1][r] * f;
            lt += stat[w][2][r] * f;
        }
        win_store(a, (T *)a.o + b * a.so.sb + h * a.so.sh + (int64_t)q * a.so.st + d,
                  (((int64_t)b * a.H + h) * a.Tq + q) * D + d, v * (1.f / lt), live);
        if (a.lse && d == 0)
            a.lse[((int64_t)b * a.H + h) * a.Tq + q] = live ? (mm * a.sl2 + log2f(ll)) * (1.f / kLog2e) : -INFINITY;
    }
}

// ---------------------------------------------------------------- backward: queries
// dQ of 32 queries per wavefront, over the keys they see; also the rows' lse
// and Delta as the keys' kernel reads them.  Delta is formed from the output and
// what its rounding to bf16 took: the rounded one alone shifts a row's dS all
// to one side, and leaves dQ and dK 2.5 to 2.65e-3 off instead of 2.4e-3 (one
// rounding of the results alone: 1.66e-3), for 4% less time.  Tiles and bounds
// as in the forward, three products where that has two: 32 heads on 8 of 128,
// 2 x 4,096 padded tokens, window 1,024, 16 first tokens, bf16: 205 to 231 us
// from one card to another (the forward 151, with lse and what rounding took 170
// to 190).
//
// A row's dS sum to 0, so a vector common to its keys cancels from dQ.  Rounded
// to bf16, and with a Delta that is, they leave a rest of the sum, which such a
// vector multiplies (keys within 1 of it, 4 in every element: dQ 1.5e-2 off).
// The rest is summed as the products took dS and goes back, with its sign
// turned, in even parts to keys at the end of the row's range: 2.4e-3, as
// without a common vector, for 1 to 2.5% of the backward's time at D >= 64 and
// 5 to 6% below.  In float32 the same holds of the steps of large scores (keys
// and queries at 3, spread by 0.25: dQ 7 to 32e-6 off, 3 to 17e-6 so, as dK and
// dV), for 1 to 2%.
template <typename T, int D>
__global__ __launch_bounds__(64 * kWinWaves, sizeof(T) == 4 && D == 128 ? 1 : 2) void window_bwd_q_kernel(WinArgs a) {
    constexpr int KC = WinCfg<T, D>::KC, NK = WinCfg<T, D>::NK, ND = WinCfg<T, D>::ND, NJ = KC / 32;
    typedef Tile<T, D, KC> L;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int nqt = (a.Tq + kWinQ - 1) / kWinQ;
    const int id = xcd_item(nqt * a.H * a.B);
    if (id < 0) return;
    const int bh = uniform(id / nqt), qt = nqt - 1 - (id - bh * nqt);
    const int b = uniform(bh / a.H), h = bh - b * a.H, g = uniform(h / (a.H / a.G));
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 31, hi = lane >> 5;
    const int len = win_len(a, b), off = a.Tk - a.Tq;
    const int qi = qt * kWinQ + 32 * wave + n, p = qi + off, qc = min(qi, a.Tq - 1);
    const int wlo = max(0, qt * kWinQ + off), whi = min(min(qt * kWinQ + kWinQ, a.Tq) - 1 + off, len - 1);
    const int pa = max(0, qt * kWinQ + 32 * wave + off), pb = min(qt * kWinQ + 32 * wave + 31 + off, len - 1);
    const bool live = p >= 0 && p < len && qi < a.Tq;

    Frag<T> qf[NK], gf[NK];
    float delta = 0.f;
    {
        const T *qp = (const T *)a.q + b * a.sq.sb + h * a.sq.sh + (int64_t)qc * a.sq.st;
        const T *gp = (const T *)a.go + b * a.sgo.sb + h * a.sgo.sh + (int64_t)qc * a.sgo.st;
        const T *op = (const T *)a.o + b * a.so.sb + h * a.so.sh + (int64_t)qc * a.so.st;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
            qf[kk] = load_frag(qp + 16 * kk + 8 * hi);
            gf[kk] = load_frag(gp + 16 * kk + 8 * hi);
            delta += dot(gf[kk], load_frag(op + 16 * kk + 8 * hi));
        }
        if (sizeof(T) == 2 && a.rest) {
            const T *rp = (const T *)a.rest + (((int64_t)b * a.H + h) * a.Tq + qc) * D;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) delta += dot(gf[kk], load_frag(rp + 16 * kk + 8 * hi));
        }
        delta = half_sum(delta);
    }
    const int64_t row = ((int64_t)b * a.H + h) * a.Tq + qc;
    const float lse2 = live ? a.lse[row] * kLog2e : INFINITY;   // a row that sees nothing has no weights
    if (hi == 0 && qi < a.Tq) {
        a.stat[row] = lse2;
        a.stat[(int64_t)a.B * a.H * a.Tq + row] = live ? delta : 0.f;
    }
    f32x16 acc[ND];
#pragma unroll
    for (int c = 0; c < ND; ++c) acc[c] = f32x16{};

    const T *kb = (const T *)a.k + b * a.skv.sb + g * a.skv.sh, *vb = (const T *)a.v + b * a.skv.sb + g * a.skv.sh;
    const Chunks ch = wlo <= whi ? win_chunks<KC>(a, wlo, whi) : Chunks{0, 0, 0};
    const typename L::template Loads<kWinWaves> loads(a.skv.st, wave, lane);
    auto fetch_k = [&](int i) { loads.go(smem + (i & 1) * 2 * L::BYTES, kb, a.skv.st, ch.at(i) * KC, len, wave); };
    auto fetch_v = [&](int i) { loads.go(smem + (i & 1) * 2 * L::BYTES + L::BYTES, vb, a.skv.st, ch.at(i) * KC, len, wave); };
    uint32_t ka[NK], kc = L::col_base(smem, lane);
#pragma unroll
    for (int kk = 0; kk < NK; ++kk) ka[kk] = L::row_base(smem, n, hi) ^ L::row_step(kk);
    float sum = 0.f;                              // of the row's dS as the products took them
    if (ch.n > 0) fetch_k(0), fetch_v(0);
    for (int i = 0; i < ch.n; ++i) {
        tiles_ready();
        const int k0 = ch.at(i) * KC;
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
            const int kind = pa <= pb ? win_kind(a, k0 + 32 * j, 32, pa, pb) : 0;
            // the next tile's loads in two bursts, each behind a product's
            if (i + 1 < ch.n) {
                if (j == 0) fetch_k(i + 1);
                if (j == NJ - 1) fetch_v(i + 1);
            }
            if (kind == 0) continue;
            f32x16 s = f32x16{}, dp = f32x16{};
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
                mma(s, L::row_from(ka[kk] + 32 * j * L::ROWB, 0), qf[kk]);
                mma(dp, L::row_from(ka[kk] + L::BYTES + 32 * j * L::ROWB, 0), gf[kk]);
            }
            if constexpr (sizeof(T) == 2 && NK > 1) pace<1, 2 * NK, 4>();
            if (kind == 1) win_hide(s, win_keys(a, p, k0 + 32 * j), hi);
            float ds[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) ds[r] = __builtin_amdgcn_exp2f(fmaf(s[r], a.sl2, -lse2)) * (dp[r] - delta);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                Frag<T> f;
                pack(f, ds + 8 * t);
                sum = add_all(sum, f);
                if constexpr (sizeof(T) == 2 && ND == 1) {
                    // one product a block: dS goes in two parts, its rounding
                    // with it (relative error of dQ, its own rounding in it, 8
                    // x 32 heads of 16 and 2 x 32 of 32, 1,024 tokens, window
                    // 256: 2.48 and 2.43e-3 without, 1.74 and 1.72e-3 so; the
                    // backward's kernels 81 and 39 us, 90 and 40 so)
                    const Frag<T> k0c = L::col_from(kc, 32 * j + 16 * t, 0);
                    Frag<T> rest;
                    pack_rest(rest, ds + 8 * t, f);
                    sum = add_all(sum, rest);
                    mma(acc[0], k0c, f);
                    mma(acc[0], k0c, rest);
                } else {
#pragma unroll
                    for (int c = 0; c < ND; ++c) mma(acc[c], L::col_from(kc, 32 * j + 16 * t, c), f);
                }
            }
        }
        const int other = i & 1 ? -2 * L::BYTES : 2 * L::BYTES;          // the next tile's buffer
        kc += other;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) ka[kk] += other;
    }
    if (ch.n > 0) {
        // what is left of the sum goes, with its sign turned, to the first 32
        // keys of the last tile (rows past the length are zeros there)
        const int k0 = ch.at(ch.n - 1) * KC;
        const float each = -half_sum(sum) / (float)min(32, len - k0);
        const float w[8] = {each, each, each, each, each, each, each, each};
        const uint32_t last = L::col_base(smem + ((ch.n - 1) & 1) * 2 * L::BYTES, lane);
        Frag<T> f;
        pack(f, w);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int c = 0; c < ND; ++c) mma(acc[c], L::col_from(last, 16 * t, c), f);
    }
    if (qi >= a.Tq) return;
    T *dq = (T *)a.dq + (((int64_t)b * a.H + h) * a.Tq + qi) * D;
#pragma unroll
    for (int c = 0; c < ND; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int d = 32 * c + 8 * t + 4 * hi;
            if (D % 32 && d >= D) continue;
            const f32x4 v = f32x4{acc[c][4 * t], acc[c][4 * t + 1], acc[c][4 * t + 2], acc[c][4 * t + 3]} * a.scale;
            store4(dq + d, live ? v : f32x4{0.f, 0.f, 0.f, 0.f});
        }
}

// ---------------------------------------------------------------- backward: keys
// dK and dV of 32 keys per wavefront (a key block of 128 per workgroup) over
// the queries that see them, of every query head that shares them.  The
// (head, query tile) pairs of a block are cut into splits, each summed by a
// workgroup of its own: blocks with first tokens, which every later query
// sees, into ns, the others into nn.  A split block's parts go to `part` and
// are summed in a fixed order; an unsplit block is stored at once.  Keys stay
// in registers and queries pass by, so shared heads' gradients need no sum
// afterwards.  Four products, and registers for no more than one of the score
// tiles at a time: 273 to 311 us for the case above (loads in two bursts, as in the
// other kernels, took 12% more).  float32 at D = 64 runs two wavefronts per SIMD
// (332 us for 32 heads on 8, 2,048 tokens, causal; 368 with one).  The whole
// backward in float32 takes 2.0 ms for 2 x 32 heads of 64, 4,096 tokens, window
// 1,024, and 4.4 of 128: 74 and 68 TFLOP/s of the five products it cannot do
// without, 104 and 96 of the seven that the two kernels form.
template <typename T, int D> struct WinBwdCfg {
    static constexpr int KL = D == 128 && sizeof(T) == 2 ? 2 : 0;     // K operands kept in LDS
    static constexpr int QC = D == 128 && sizeof(T) == 4 ? 32 : 64;   // rows of a tile
};
// Tiles of QC queries (indexes from query 0) that see keys k0 .. k0 + 127.
template <int QC> __device__ __forceinline__ void win_q_tiles(const WinArgs &a, int k0, int len, int *first, int *count) {
    const int off = a.Tk - a.Tq;
    const int lo = max(k0, off);                                     // first position that has a query
    int end = min(len, a.Tk) - 1;
    if (a.W > 0 && k0 >= a.S) end = (int)min((int64_t)end, (int64_t)k0 + kWinQ - 1 + a.W - 1);
    *first = lo <= end ? (lo - off) / QC : 0;
    *count = lo <= end ? (end - off) / QC - *first + 1 : 0;
}

template <typename T, int D>
__global__ __launch_bounds__(64 * kWinWaves, sizeof(T) == 4 && D == 128 ? 1 : 2) void window_bwd_kv_kernel(WinArgs a) {
    constexpr int QC = WinBwdCfg<T, D>::QC, NK = WinCfg<T, D>::NK, ND = WinCfg<T, D>::ND, NJ = QC / 32;
    typedef Tile<T, D, QC> L;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ __align__(16) float stat[2][2][64];   // [buffer][lse * log2(e), Delta]
    // the last K operands of each lane wait in LDS where the registers of two
    // wavefronts per SIMD do not hold them all beside the accumulators
    constexpr int KL = WinBwdCfg<T, D>::KL, KR = NK - KL;
    __shared__ Frag<T> klast[KL ? KL : 1][KL ? 64 * kWinWaves : 1];
    const int per = a.nsb * a.ns + (a.nb - a.nsb) * a.nn;            // items per (sequence, kv head)
    const int id = xcd_item(per * a.G * a.B);
    if (id < 0) return;
    const int bg = uniform(id / per), it = id - bg * per, b = uniform(bg / a.G), g = bg - b * a.G;
    const bool sink = it < a.nsb * a.ns;
    const int nsplit = sink ? a.ns : a.nn, rel = sink ? it : it - a.nsb * a.ns, blk = uniform(rel / nsplit);
    const int kblk = sink ? blk : a.nsb + blk, split = rel - blk * nsplit;
    const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, n = lane & 31, hi = lane >> 5;
    const int len = win_len(a, b), off = a.Tk - a.Tq, R = uniform(a.H / a.G);
    const int k0 = kblk * kWinQ, kw = k0 + 32 * wave, key = kw + n;

    Frag<T> kf[KR], vf[NK];
    {
        const int64_t at = b * a.skv.sb + g * a.skv.sh + (int64_t)min(key, a.Tk - 1) * a.skv.st;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
            const Frag<T> f = load_frag((const T *)a.k + at + 16 * kk + 8 * hi);
            if (kk < KR) kf[kk] = f;
            else klast[kk - KR][threadIdx.x] = f;      // read by this lane only
            vf[kk] = load_frag((const T *)a.v + at + 16 * kk + 8 * hi);
        }
    }
    f32x16 ak[ND], av[ND];
#pragma unroll
    for (int c = 0; c < ND; ++c) ak[c] = av[c] = f32x16{};
    int t0, nt;
    win_q_tiles<QC>(a, k0, len, &t0, &nt);
    // this split's share of the R * nt (head, tile) pairs
    const int total = R * nt, i0 = uniform((int)((int64_t)total * split / nsplit));
    const int i1 = uniform((int)((int64_t)total * (split + 1) / nsplit));
    const int nq = max(0, min(a.Tq, len - off));                     // queries before the sequence's end
    auto fetch = [&](int i, int hr, int tile) {                      // pair i: head hr of the group, tile t0 + tile
        const int h = g * R + hr, q0 = (t0 + tile) * QC, lane = fresh(threadIdx.x & 63);
        unsigned char *dst = smem + (i & 1) * 2 * L::BYTES;
        L::template fetch<kWinWaves>(dst, (const T *)a.q + b * a.sq.sb + h * a.sq.sh, a.sq.st, q0, -off, nq, wave, lane);
        L::template fetch<kWinWaves>(dst + L::BYTES, (const T *)a.go + b * a.sgo.sb + h * a.sgo.sh, a.sgo.st, q0, -off,
                                     nq, wave, lane);
        // one wavefront the tile's lse, another its Delta; rows past the last
        // one are zeros, as their q and do are: weights of 1 times nothing
        const int w = __builtin_amdgcn_readfirstlane(wave);
        if (w < 2) {
            const float *sp = a.stat + ((int64_t)w * a.B * a.H + (int64_t)b * a.H + h) * a.Tq + q0;
            lds_load<4>(lds_load_rsrc(sp, (uint32_t)(4 * min(QC, nq - q0))), 4 * lane, lds_addr(&stat[i & 1][w][0]));
        }
    };
    int hr = nt ? uniform(i0 / nt) : 0, tile = i0 - hr * nt;
    if (i0 < i1) fetch(i0, hr, tile);
    for (int i = i0; i < i1; ++i) {
        tiles_ready();
        const int pq = (t0 + tile) * QC + off;                       // position of the tile's first query
        if (++tile == nt) tile = 0, ++hr;
        if (i + 1 < i1) fetch(i + 1, hr, tile);
        const unsigned char *ql = smem + (i & 1) * 2 * L::BYTES;   // then the tile of do
#pragma unroll 1
        for (int j = 0; j < NJ; ++j) {
            const int ln = fresh(lane), n = ln & 31, hi = ln >> 5;
            const int pa = pq + 32 * j, pb = pa + 31;
            const int kind = kw < len ? win_kind(a, kw, 32, pa, pb) : 0;
            if (kind == 0) continue;
            // scores, weights, dV; then do V^T, dS, dK: one after the other, so
            // that 32 results at a time are live beside the accumulators
            const uint32_t rows = L::row_base(ql + 32 * j * L::ROWB, n, hi), cols = L::col_base(ql + 32 * j * L::ROWB, ln);
            f32x16 s = f32x16{};
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
                mma(s, L::row_from(rows, kk), kk < KR ? kf[kk < KR ? kk : 0] : klast[kk < KR ? 0 : kk - KR][threadIdx.x]);
            if constexpr (sizeof(T) == 2 && NK > 3) pace<1, NK, 3>();
            if (kind == 1) win_hide(s, win_rows(a, pa, kw + n), hi);
            float w[16];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const f32x4 ls = *(const f32x4 *)&stat[i & 1][0][32 * j + 8 * t + 4 * hi];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[4 * t + e] = __builtin_amdgcn_exp2f(fmaf(s[4 * t + e], a.sl2, -ls[e]));
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                Frag<T> f;
                pack(f, w + 8 * t);
#pragma unroll
                for (int c = 0; c < ND; ++c) mma(av[c], L::col_from(cols + L::BYTES, 16 * t, c), f);
            }
            f32x16 dp = f32x16{};
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) mma(dp, L::row_from(rows + L::BYTES, kk), vf[kk]);
            if constexpr (sizeof(T) == 2 && NK > 3) pace<1, NK, 3>();
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const f32x4 de = *(const f32x4 *)&stat[i & 1][1][32 * j + 8 * t + 4 * hi];
#pragma unroll
                for (int e = 0; e < 4; ++e) w[4 * t + e] *= dp[4 * t + e] - de[e];
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                Frag<T> f;
                pack(f, w + 8 * t);
#pragma unroll
                for (int c = 0; c < ND; ++c) mma(ak[c], L::col_from(cols, 16 * t, c), f);
            }
        }
    }
    // keys past the length (whatever they hold) have no gradient
    if (key >= len) {
#pragma unroll
        for (int c = 0; c < ND; ++c) ak[c] = av[c] = f32x16{};
    }
    if (nsplit > 1) {
        // partial rows, float32: [b, g][block's slot][split][dK, dV][128][D]
        const int64_t slot = sink ? (int64_t)kblk * a.ns
                                  : (a.ns > 1 ? (int64_t)a.nsb * a.ns : 0) + (int64_t)(kblk - a.nsb) * a.nn;
        const int64_t slots = (a.ns > 1 ? (int64_t)a.nsb * a.ns : 0) + (a.nn > 1 ? (int64_t)(a.nb - a.nsb) * a.nn : 0);
        float *pk = a.part + (((int64_t)b * a.G + g) * slots + slot + split) * 2 * kWinQ * D + (32 * wave + n) * D;
#pragma unroll
        for (int c = 0; c < ND; ++c)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int d = 32 * c + 8 * t + 4 * hi;
                if (D % 32 && d >= D) continue;
                store4(pk + d, f32x4{ak[c][4 * t], ak[c][4 * t + 1], ak[c][4 * t + 2], ak[c][4 * t + 3]} * a.scale);
                store4(pk + kWinQ * D + d, f32x4{av[c][4 * t], av[c][4 * t + 1], av[c][4 * t + 2], av[c][4 * t + 3]});
            }
        return;
    }
    if (key >= a.Tk) return;
    const int64_t at = (((int64_t)b * a.G + g) * a.Tk + key) * D;
#pragma unroll
    for (int c = 0; c < ND; ++c)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int d = 32 * c + 8 * t + 4 * hi;
            if (D % 32 && d >= D) continue;
            store4((T *)a.dk + at + d,
                   f32x4{ak[c][4 * t], ak[c][4 * t + 1], ak[c][4 * t + 2], ak[c][4 * t + 3]} * a.scale);
            store4((T *)a.dv + at + d, f32x4{av[c][4 * t], av[c][4 * t + 1], av[c][4 * t + 2], av[c][4 * t + 3]});
        }
}

// dK and dV of the split key blocks: the splits' parts summed in order.  Bound
// by memory, a few us (4 for the case above, 18 for the largest splits timed).
template <typename T, int D> __global__ __launch_bounds__(256) void window_bwd_sum_kernel(WinArgs a) {
    const int blk0 = a.ns > 1 ? 0 : a.nsb, blk1 = a.nn > 1 ? a.nb : a.nsb;   // split blocks (host: at least one)
    const int kblk = blk0 + (int)blockIdx.x % (blk1 - blk0), bg = (int)blockIdx.x / (blk1 - blk0);
    const bool sink = kblk < a.nsb;
    const int nsplit = sink ? a.ns : a.nn;
    const int64_t slot = sink ? (int64_t)kblk * a.ns
                              : (a.ns > 1 ? (int64_t)a.nsb * a.ns : 0) + (int64_t)(kblk - a.nsb) * a.nn;
    const int64_t slots = (a.ns > 1 ? (int64_t)a.nsb * a.ns : 0) + (a.nn > 1 ? (int64_t)(a.nb - a.nsb) * a.nn : 0);
    const float *src = a.part + ((int64_t)bg * slots + slot) * 2 * kWinQ * D;
    const int rows = min(kWinQ, a.Tk - kblk * kWinQ);
    const int i = ((int)blockIdx.y * 256 + (int)threadIdx.x) * 4;            // element of [dK, dV][128][D]
    const int which = i / (kWinQ * D), at = i % (kWinQ * D);
    if (at / D >= rows) return;
    f32x4 s = load4(src + i);
    for (int k = 1; k < nsplit; ++k) s += load4(src + (int64_t)k * 2 * kWinQ * D + i);
    store4((T *)(which ? a.dv : a.dk) + ((int64_t)bg * a.Tk + kblk * kWinQ) * D + at, s);
}

// ---------------------------------------------------------------- host
// Splits of the key blocks' queries.  A split costs its partial sums, about
// five tiles' time written and read back, so blocks of a window, all of a
// length, are split only where they do not fill the chip (two workgroups per
// CU).  Without a window the first block is seen by every query and the last
// by few: a split then takes at most three quarters of an even part of the
// whole, or 24 tiles (32 heads on 8 of 64, 2 x 4,096 causal: dK, dV 665 us in
// one piece, 387 in three).  Blocks of first tokens, which every later tile
// sees, are split into parts as long as the others'.
static void win_splits(WinArgs &a, int QC) {
    a.nb = (int)ceil_div(a.Tk, kWinQ);
    a.nsb = a.W > 0 && a.W < a.Tk ? (int)ceil_div(a.S < a.Tk ? a.S : a.Tk, kWinQ) : 0;
    const int64_t R = a.H / a.G, full = R * (ceil_div(a.Tk, QC) + 1);
    int64_t near = a.W > 0 ? R * (ceil_div((int64_t)a.W + kWinQ, QC) + 1) : full;
    if (near > full) near = full;
    const int64_t blocks = (int64_t)a.B * a.G * a.nb, slots = 2 * (int64_t)device_info().cu_count;
    int64_t nn = blocks < slots ? ceil_div(slots, blocks) : 1;
    if (nn > ceil_div(near, 4)) nn = ceil_div(near, 4);   // four tiles at least
    if (a.W <= 0) {
        int64_t share = ceil_div(blocks * full / 2 * 3, slots * 4);
        if (share < 24) share = 24;
        if (nn < ceil_div(full, share)) nn = ceil_div(full, share);
    }
    if (nn > 64) nn = 64;
    const int64_t ns = ceil_div(full, ceil_div(near, nn));
    a.nn = (int)nn;
    a.ns = a.nsb ? (int)(ns > 256 ? 256 : ns) : 1;
}

static int64_t win_part_slots(const WinArgs &a) {
    return (a.ns > 1 ? (int64_t)a.nsb * a.ns : 0) + (a.nn > 1 ? (int64_t)(a.nb - a.nsb) * a.nn : 0);
}

static int win_check(const char *fn, const WinArgs &a, int64_t B, int64_t H, int64_t G, int64_t Tq, int64_t Tk,
                     int64_t D, int dtype) {
    if (B < 0 || H < 1 || G < 1 || H % G || Tq < 0 || Tk < 0 || Tq > (1 << 24) || Tk > (1 << 24))
        return set_error(WALSH_EINVAL, "%s: bad shape B=%lld H=%lld G=%lld Tq=%lld Tk=%lld", fn, (long long)B,
                         (long long)H, (long long)G, (long long)Tq, (long long)Tk);
    if (D != 16 && D != 32 && D != 64 && D != 128)
        return set_error(WALSH_ENOTSUP, "%s: head_dim %lld (16, 32, 64 or 128)", fn, (long long)D);
    if (dtype != WALSH_F32 && dtype != WALSH_BF16) return set_error(WALSH_ENOTSUP, "%s: dtype %d", fn, dtype);
    if (!(a.scale > 0.f) || a.scale > 1e6f)
        return set_error(WALSH_EINVAL, "%s: the scale must be positive and at most 1e6", fn);
    // work items of 128 positions, whose threads a launch counts in 32 bits
    if (B > (1 << 24) || H > (1 << 24) || B * H > ((1 << 24) - 8) / ceil_div(Tq > Tk ? Tq : Tk > 0 ? Tk : 1, kWinQ))
        return set_error(WALSH_ENOTSUP, "%s: B=%lld H=%lld T=%lld exceed the grid", fn, (long long)B, (long long)H,
                         (long long)(Tq > Tk ? Tq : Tk));
    return WALSH_OK;
}

// Rows are read in 16-byte pieces: strides multiples of 8 elements, rows that
// do not overlap, and 64 of them within 2 GiB.
static int win_check_tensor(const char *fn, const char *name, const void *p, const WinTensor &s, int64_t B, int64_t H,
                            int64_t T, int64_t D) {
    if (!p) return set_error(WALSH_EINVAL, "%s: null pointer (%s)", fn, name);
    if ((uintptr_t)p % 16 || s.sb % 8 || s.sh % 8 || s.st % 8)
        return set_error(WALSH_ENOTSUP, "%s: %s needs 16-byte alignment and strides that are multiples of 8", fn, name);
    if ((T > 1 && s.st < D) || s.st < 0 || s.sb < 0 || s.sh < 0 || s.st > (1 << 22))
        return set_error(WALSH_ENOTSUP, "%s: %s: row stride %lld (head_dim %lld to 2^22), no negative strides", fn, name,
                         (long long)s.st, (long long)D);
    return WALSH_OK;
}

}  // namespace walsh

using namespace walsh;

WALSH_EXPORT int walsh_window_attention_fwd(const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void *k,
                                            const void *v, int64_t kv_sb, int64_t kv_sh, int64_t kv_st, int64_t B,
                                            int64_t H, int64_t G, int64_t Tq, int64_t Tk, int64_t D, int64_t window,
                                            int64_t sinks, const int *lengths, float scale, void *o, int64_t o_sb,
                                            int64_t o_sh, int64_t o_st, float *lse, void *rest, int dtype,
                                            void *stream) {
    const char *fn = "walsh_window_attention_fwd";
    WinArgs a{};
    a.scale = scale;
    int rc = win_check(fn, a, B, H, G, Tq, Tk, D, dtype);
    if (rc) return rc;
    if (B == 0 || Tq == 0) return WALSH_OK;
    a.q = q, a.k = k, a.v = v, a.lengths = lengths, a.o = o, a.lse = lse, a.rest = dtype == WALSH_BF16 ? rest : nullptr;
    a.sq = {q_sb, q_sh, q_st}, a.skv = {kv_sb, kv_sh, kv_st}, a.so = {o_sb, o_sh, o_st};
    rc = win_check_tensor(fn, "q", q, a.sq, B, H, Tq, D);
    if (!rc && Tk) rc = win_check_tensor(fn, "k", k, a.skv, B, G, Tk, D);
    if (!rc && Tk) rc = win_check_tensor(fn, "v", v, a.skv, B, G, Tk, D);
    if (!rc) rc = win_check_tensor(fn, "o", o, a.so, B, H, Tq, D);
    if (!rc && (uintptr_t)rest % 16) rc = set_error(WALSH_ENOTSUP, "%s: rest must be 16-byte aligned", fn);
    if (rc) return rc;
    a.B = (int)B, a.H = (int)H, a.G = (int)G, a.Tq = (int)Tq, a.Tk = (int)Tk;
    a.W = window > 0 && window < Tk ? (int)window : 0;
    a.S = sinks < 0 ? 0 : (int)(sinks < Tk ? sinks : Tk);
    a.sl2 = scale * kLog2e;
    if (Tk == 1) a.skv.st = D;                    // (the tiles' loads count rows by it)
    const int64_t n = ceil_div(Tq, kWinQ) * H * B, n32 = ceil_div(Tq, 32) * H * B;
    const bool split = n < device_info().cu_count;   // a wavefront per SIMD and less: cut the keys, too
    attn_dispatch(dtype, D, [&](auto t, auto d) {
        typedef decltype(t) T;
        constexpr int DD = decltype(d)::value;
        if (split)
            launch(window_fwd_split_kernel<T, DD>, dim3((unsigned)(ceil_div(n32, 8) * 8)), dim3(64 * kWinWaves),
                   (uint32_t)(kWinWaves * WinSplitCfg<T, DD>::WAVE), (hipStream_t)stream, a);
        else
            launch(a.lse ? window_fwd_kernel<T, DD, true> : window_fwd_kernel<T, DD, false>,
                   dim3((unsigned)(ceil_div(n, 8) * 8)), dim3(64 * kWinWaves),
                   (uint32_t)(4 * Tile<T, DD, WinCfg<T, DD>::KC>::BYTES), (hipStream_t)stream, a);
    });
    return check_hip(hipGetLastError(), fn);
}

static int win_bwd_qc(int64_t D, int dtype) { return D == 128 && dtype == WALSH_F32 ? 32 : 64; }

static int64_t win_stat_bytes(const WinArgs &a) { return ceil_div((int64_t)a.B * a.H * a.Tq * 8, 16) * 16; }
static int64_t win_bwd_bytes(const WinArgs &a, int64_t D) {
    return win_stat_bytes(a) + (int64_t)a.B * a.G * win_part_slots(a) * 2 * kWinQ * D * 4;
}

WALSH_EXPORT int64_t walsh_window_attention_bwd_workspace_bytes(int64_t B, int64_t H, int64_t G, int64_t Tq, int64_t Tk,
                                                                int64_t D, int64_t window, int64_t sinks, int dtype) {
    if (B < 1 || H < 1 || G < 1 || H % G || Tq < 1 || Tk < 1 || D < 1 || Tq > (1 << 24) || Tk > (1 << 24)) return 0;
    WinArgs a{};
    a.B = (int)B, a.H = (int)H, a.G = (int)G, a.Tq = (int)Tq, a.Tk = (int)Tk;
    a.W = window > 0 && window < Tk ? (int)window : 0;
    a.S = sinks < 0 ? 0 : (int)(sinks < Tk ? sinks : Tk);
    win_splits(a, win_bwd_qc(D, dtype));
    return win_bwd_bytes(a, D);
}

WALSH_EXPORT int walsh_window_attention_bwd(const void *q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void *k,
                                            const void *v, int64_t kv_sb, int64_t kv_sh, int64_t kv_st, const void *o,
                                            int64_t o_sb, int64_t o_sh, int64_t o_st, const void *go, int64_t go_sb,
                                            int64_t go_sh, int64_t go_st, const float *lse, const void *rest, int64_t B,
                                            int64_t H, int64_t G, int64_t Tq, int64_t Tk, int64_t D, int64_t window, int64_t sinks,
                                            const int *lengths, float scale, void *dq, void *dk, void *dv, int dtype,
                                            void *work, int64_t work_bytes, void *stream) {
    const char *fn = "walsh_window_attention_bwd";
    WinArgs a{};
    a.scale = scale;
    int rc = win_check(fn, a, B, H, G, Tq, Tk, D, dtype);
    if (rc) return rc;
    if (B == 0) return WALSH_OK;
    if (Tq == 0 || Tk == 0) return set_error(WALSH_EINVAL, "%s: no queries or no keys: the gradients are zeros", fn);
    a.q = q, a.k = k, a.v = v, a.lengths = lengths, a.o = const_cast<void *>(o), a.lse = const_cast<float *>(lse);
    a.go = go, a.dq = dq, a.dk = dk, a.dv = dv, a.rest = dtype == WALSH_BF16 ? const_cast<void *>(rest) : nullptr;
    a.sq = {q_sb, q_sh, q_st}, a.skv = {kv_sb, kv_sh, kv_st}, a.so = {o_sb, o_sh, o_st}, a.sgo = {go_sb, go_sh, go_st};
    rc = win_check_tensor(fn, "q", q, a.sq, B, H, Tq, D);
    if (!rc) rc = win_check_tensor(fn, "k", k, a.skv, B, G, Tk, D);
    if (!rc) rc = win_check_tensor(fn, "v", v, a.skv, B, G, Tk, D);
    if (!rc) rc = win_check_tensor(fn, "o", o, a.so, B, H, Tq, D);
    if (!rc) rc = win_check_tensor(fn, "go", go, a.sgo, B, H, Tq, D);
    if (rc) return rc;
    if (!lse || !dq || !dk || !dv || !work) return set_error(WALSH_EINVAL, "%s: null pointer", fn);
    if ((uintptr_t)rest % 16 || (uintptr_t)dq % 16 || (uintptr_t)dk % 16 || (uintptr_t)dv % 16 || (uintptr_t)work % 16)
        return set_error(WALSH_ENOTSUP, "%s: rest, the gradients and the workspace must be 16-byte aligned", fn);
    a.B = (int)B, a.H = (int)H, a.G = (int)G, a.Tq = (int)Tq, a.Tk = (int)Tk;
    a.W = window > 0 && window < Tk ? (int)window : 0;
    a.S = sinks < 0 ? 0 : (int)(sinks < Tk ? sinks : Tk);
    a.sl2 = scale * kLog2e;
    if (Tk == 1) a.skv.st = D;                    // (the tiles' loads count rows by it)
    win_splits(a, win_bwd_qc(D, dtype));
    if (work_bytes < win_bwd_bytes(a, D))
        return set_error(WALSH_EINVAL, "%s: workspace of %lld bytes, needs %lld", fn, (long long)work_bytes,
                         (long long)win_bwd_bytes(a, D));
    a.stat = (float *)work;
    a.part = (float *)((char *)work + win_stat_bytes(a));
    hipStream_t s = (hipStream_t)stream;
    const int64_t nq = ceil_div(Tq, kWinQ) * H * B;
    const int64_t nk = ((int64_t)a.nsb * a.ns + (int64_t)(a.nb - a.nsb) * a.nn) * G * B;
    if (nk >= (1ll << 24) - 8) return set_error(WALSH_ENOTSUP, "%s: %lld work items", fn, (long long)nk);
    attn_dispatch(dtype, D, [&](auto t, auto d) {
        typedef decltype(t) T;
        constexpr int DD = decltype(d)::value;
        launch(window_bwd_q_kernel<T, DD>, dim3((unsigned)(ceil_div(nq, 8) * 8)), dim3(64 * kWinWaves),
               (uint32_t)(4 * Tile<T, DD, WinCfg<T, DD>::KC>::BYTES), s, a);
        launch(window_bwd_kv_kernel<T, DD>, dim3((unsigned)(ceil_div(nk, 8) * 8)), dim3(64 * kWinWaves),
               (uint32_t)(4 * Tile<T, DD, WinBwdCfg<T, DD>::QC>::BYTES), s, a);
        const int64_t blocks = (a.nn > 1 ? a.nb : a.nsb) - (a.ns > 1 ? 0 : a.nsb);
        if (blocks > 0)
            launch(window_bwd_sum_kernel<T, DD>, dim3((unsigned)(blocks * B * G), (unsigned)(2 * kWinQ * DD / 1024)),
                   dim3(256), 0, s, a);
    });
    return check_hip(hipGetLastError(), fn);
}
