// A key-value cache in pages: writing new tokens, and the attention of one new
// token per sequence over it.
//
// Token j of sequence b lies in row j % page of page table[b][j / page]; a
// page holds [G key heads][page][D] (any strides).  The query of a sequence is
// its last token, at position p = length - 1, and sees
//     j > p - W  or  j < S     (W the window, S the first tokens; W <= 0: all)
//     o = softmax(c q K^T) V
//
// Decode.  The visible keys t = 0 .. n - 1 (first tokens, then the window) are
// cut into chunks; a workgroup takes one chunk of one (sequence, key head) for
// all R = H / G query heads that share it, so the cache is read once.  Its
// four wavefronts take every fourth block of keys, each with its own running
// maximum, sum and accumulators, joined at the end in LDS, and chunks by a
// second kernel.  Scores are S^T = K Q^T on 32x32 matrix-core tiles (key rows
// come straight from memory in the operand's layout, 16 bytes a lane), so a
// lane holds 16 scores of one head; O^T = V^T P^T takes V from LDS, read
// transposed.  With R < 32 most of a tile is idle, which costs nothing in bf16:
// the matrix cores could feed ten times what memory delivers, and the vector
// units would be short at R >= 2.  Bound by memory: the next block's K
// (registers) and V (straight into LDS) are on the way while one is used; 64
// sequences of up to 4,096, 32 heads of 128: 370 us, 6.0 TB/s.  float32 takes
// the vector units up to R = 4 (paged_decode_rows_kernel), and reaches 2 to 3
// TB/s by products above.
//
// Scores, maxima, sums and accumulators are float32.  bf16 weights go into the
// product with V in two bf16 parts, so that the output's own rounding is the
// only one left (relative error 1.66e-3; 2.2e-3 with weights rounded to bf16,
// off by up to 2^-8 each): the matrix cores have the time for it (64 sequences
// of up to 4,096, 32 heads of 128: 390 us both ways, of 64, 32 sequences: 108
// and 109, of 32: 102 and 106).  Not so heads of 16, whose vector work is the
// bound (54 us with one part, 68 with two): they round the weights once, and
// their sum takes them as rounded, as in the whole-sequence kernel.
#include "tiles.h"

namespace walsh {

constexpr int kPgWaves = 4;
constexpr int kPgMaxChunk = 1024;                 // keys per workgroup
constexpr int kPgMinPage = 16;                    // rows of a page, where a sequence has several
constexpr int kPgEntries = kPgMaxChunk / kPgMinPage + 4;

struct PgArgs {
    const void *q;
    int64_t q_sb, q_sh;                           // q[b][h][d]
    const void *k, *v;
    int64_t sp, sg, sr;                           // page, head and row strides of both
    const int *table, *lengths;
    int64_t table_sb;
    int B, H, G, P, N, shift, W, S, chunk, ns;    // P pages in all, N per sequence of 2^shift rows; ns chunks
    int64_t cap;                                  // rows that a sequence's table covers
    float sl2;
    void *o;
    int64_t o_sb, o_sh;
    float *part;                                  // [B][H][ns][D] accumulators, then [B][H][ns] (max, sum)
};

// The visible keys of a sequence: n of them, the first s0 first tokens, key t
// >= s0 at row t + skip.  bad: a length that the table does not cover.
struct PgKeys {
    int n, s0, skip;
    bool bad;
};
__device__ __forceinline__ PgKeys pg_keys(const PgArgs &a, int b) {
    const int len = a.lengths[b];
    PgKeys r{max(len, 0), 0, 0, len > a.cap};
    if (a.W > 0 && r.n > a.W) {
        r.s0 = min(a.S, r.n - a.W);
        r.skip = r.n - a.W - r.s0;
        r.n = a.W + r.s0;
    }
    if (r.bad) r.n = 0;
    return r;
}

// Visible keys c0 .. c1 - 1 of a sequence and the entries of its page table
// that they need, read once into LDS.
struct PgChunk {
    PgKeys ks;
    int c0, c1;
    int ea, na, eb;      // first entry and number of the first tokens' entries; first of the window's, behind them
    __device__ __forceinline__ void open(const PgArgs &a, int b, int *pages, int *any_bad) {
        const int ta = min(c1, ks.s0);                // first tokens c0 .. ta - 1
        ea = c0 >> a.shift, na = c0 < ta ? ((ta - 1) >> a.shift) - ea + 1 : 0;
        const int tb = max(c0, ks.s0);
        eb = tb < c1 ? (tb + ks.skip) >> a.shift : 0;
        const int nb = tb < c1 ? ((c1 - 1 + ks.skip) >> a.shift) - eb + 1 : 0;
        if (threadIdx.x == 0) *any_bad = ks.bad;
        __syncthreads();
        for (int i = threadIdx.x; i < na + nb; i += 64 * kPgWaves) {
            const int e = a.table[b * a.table_sb + (i < na ? ea + i : eb + i - na)];
            const bool ok = (unsigned)e < (unsigned)a.P;
            pages[i] = ok ? e : 0;
            if (!ok) *any_bad = 1;
        }
        __syncthreads();
    }
    // element offset of visible key t (past the last one: the last, never counted)
    __device__ __forceinline__ int64_t at(const PgArgs &a, const int *pages, int t) const {
        t = min(t, c1 - 1);
        const int j = t < ks.s0 ? t : t + ks.skip, e = t < ks.s0 ? (j >> a.shift) - ea : na + (j >> a.shift) - eb;
        return pages[e] * a.sp + (j & ((1 << a.shift) - 1)) * a.sr;
    }
};

// The wavefronts' parts of `heads` query heads from h0 on, joined:
//     o = sum_w acc_w e^(m_w - m) / sum_w l_w e^(m_w - m)
// to the output, or where a sequence has several chunks to the workspace.
// stat(w, 0, r) and stat(w, 1, r): maximum and sum, acc(w, r): D accumulators.
template <typename T, int D, typename S, typename A>
__device__ __forceinline__ void pg_join(const PgArgs &a, int b, int h0, int heads, int s, bool some, bool bad, S stat, A acc) {
    for (int i = threadIdx.x; i < heads * (D / 4); i += 64 * kPgWaves) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        float mm = stat(0, 0, r);
#pragma unroll
        for (int w = 1; w < kPgWaves; ++w) mm = fmaxf(mm, stat(w, 0, r));
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        float ll = 0.f;
#pragma unroll
        for (int w = 0; w < kPgWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f((stat(w, 0, r) - mm) * a.sl2);
            v += load4(acc(w, r) + d) * f;
            ll += stat(w, 1, r) * f;
        }
        if (bad) ll = NAN;                        // a page or length outside the pool: not a number, never a stale value
        if (a.ns == 1) {
            store4((T *)a.o + b * a.o_sb + (h0 + r) * a.o_sh + d, some || bad ? v * (1.f / ll) : f32x4{0.f, 0.f, 0.f, 0.f});
        } else {
            const int64_t at = ((int64_t)b * a.H + h0 + r) * a.ns + s;
            store4(a.part + at * D + d, v);
            if (d == 0) ((float2 *)(a.part + (int64_t)a.B * a.H * a.ns * D))[at] = make_float2(mm, ll);
        }
    }
}

template <typename T, int D> struct PgCfg {
    // 32-key sub-blocks of a wavefront's step: 8 KB of K (bf16) whatever D
    static constexpr int NB = sizeof(T) == 2 ? (D == 128 ? 1 : D == 64 ? 2 : 4) : (D >= 64 ? 1 : D == 32 ? 2 : 4);
    static constexpr bool TWO = sizeof(T) == 2 && D >= 32;   // bf16 weights in two parts
    static constexpr int VBYTES = NB * Tile<T, D, 32>::BYTES;
    // two V buffers per wavefront; at the end 32 rows of D float32
    static constexpr int WAVE = 2 * VBYTES > 32 * D * 4 ? 2 * VBYTES : 32 * D * 4;
    static constexpr int LDS = kPgWaves * WAVE;
};

template <typename T, int D>
__global__ __launch_bounds__(64 * kPgWaves, sizeof(T) == 4 && D == 128 ? 1 : 2) void paged_decode_kernel(PgArgs a) {
    constexpr int NB = PgCfg<T, D>::NB, KB = 32 * NB, NK = D / 16, ND = (D + 31) / 32;
    constexpr bool TWO = PgCfg<T, D>::TWO;
    typedef Tile<T, D, 32> L;
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ int pages[kPgEntries];
    __shared__ float stat[kPgWaves][2][32];
    __shared__ int any_bad;
    const int R = uniform(a.H / a.G), nqt = (R + 31) / 32;
    // the heads of a chunk side by side: their rows share pages
    const int gy = a.G * nqt, s = uniform((int)blockIdx.x / gy), gq = (int)blockIdx.x - s * gy, b = blockIdx.y;
    const int g = uniform(gq / nqt), r0 = (gq - g * nqt) * 32;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n = lane & 31, hi = lane >> 5;
    const int heads = min(32, R - r0), h0 = g * R + r0;
    const PgKeys ks = pg_keys(a, b);
    const int c0 = s * a.chunk, c1 = min(c0 + a.chunk, ks.n);
    if (c0 >= c1 && s > 0) return;                // the combine looks at the chunks that exist

    PgChunk ck{ks, c0, c1};
    ck.open(a, b, pages, &any_bad);

    Frag<T> qf[NK];
    {
        const T *qp = (const T *)a.q + b * a.q_sb + (h0 + min(n, heads - 1)) * a.q_sh;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) qf[kk] = load_frag(qp + 16 * kk + 8 * hi);
    }
    const T *kb = (const T *)a.k + g * a.sg, *vb = (const T *)a.v + g * a.sg;
    unsigned char *vl = smem + wave * PgCfg<T, D>::WAVE;
    // K of the keys from t0 on into operands, V into a buffer; a V row's offset
    // comes from the lane that has that row of K
    auto fetch = [&](Frag<T> (&kf)[NB][NK], int buf, int t0) {
        const uint32_t dst = lds_addr(vl) + buf * PgCfg<T, D>::VBYTES;
#pragma unroll
        for (int u = 0; u < NB; ++u) {
            const int64_t at = ck.at(a, pages, t0 + 32 * u + n);
            const T *p = kb + at + 8 * hi;
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) kf[u][kk] = load_frag(p + 16 * kk);
#pragma unroll
            for (int i = 0; i < L::BYTES / 1024; ++i) {
                const int pos = i * 64 + lane, row = pos / L::NCH, c = (pos % L::NCH) ^ L::swz(row);
                const int64_t from = ((int64_t)__shfl((int)(at >> 32), row) << 32) | (uint32_t)__shfl((int)at, row);
                lds_gather(vb + from + c * (16 / (int)sizeof(T)), dst + u * L::BYTES + i * 1024);
            }
        }
    };

    f32x16 acc[ND];
#pragma unroll
    for (int c = 0; c < ND; ++c) acc[c] = f32x16{};
    float m = kNoScore, l = 0.f;
    const int stride = KB * kPgWaves;
    int t0 = c0 + wave * KB, buf = 0;
    Frag<T> kf[NB][NK];
    if (t0 < c1) fetch(kf, 0, t0);
    for (; t0 < c1; t0 += stride, buf ^= 1) {
        const int tn = t0 + stride;
        f32x16 sc[NB];
#pragma unroll
        for (int u = 0; u < NB; ++u) {
            sc[u] = f32x16{};
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) mma(sc[u], kf[u][kk], qf[kk]);
        }
        // this block's V has landed (it was requested after this block's K)
        wait_loads();
        if (tn < c1) fetch(kf, buf ^ 1, tn);
        if (t0 + KB > c1) {
#pragma unroll
            for (int u = 0; u < NB; ++u)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (t0 + 32 * u + 8 * (r >> 2) + 4 * hi + (r & 3) >= c1) sc[u][r] = -INFINITY;
        }
        float mx = sc[0][0];
#pragma unroll
        for (int u = 0; u < NB; ++u)
#pragma unroll
            for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[u][r]);
        mx = half_max(mx);
        if (__any((mx - m) * a.sl2 > 8.f)) {      // as in the whole-sequence kernel: move the maximum rarely
            const float mn = fmaxf(m, mx), al = __builtin_amdgcn_exp2f((m - mn) * a.sl2);
            m = mn;
            l *= al;
#pragma unroll
            for (int c = 0; c < ND; ++c) acc[c] *= al;
        }
        const float mo = -m * a.sl2;
        const unsigned char *vt = vl + buf * PgCfg<T, D>::VBYTES;
#pragma unroll
        for (int u = 0; u < NB; ++u) {
            float w[16];
#pragma unroll
            for (int r = 0; r < 16; ++r) w[r] = __builtin_amdgcn_exp2f(fmaf(sc[u][r], a.sl2, mo));
            if constexpr (sizeof(T) == 4 || TWO) {
#pragma unroll
                for (int r = 0; r < 16; ++r) l += w[r];
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                Frag<T> pf, rest;
                pack(pf, w + 8 * t);
                if constexpr (TWO) pack_rest(rest, w + 8 * t, pf);
                else if constexpr (sizeof(T) == 2) l = add_all(l, pf);
#pragma unroll
                for (int c = 0; c < ND; ++c) {
                    const Frag<T> vc = L::col(vt + u * L::BYTES, 16 * t, c, lane);
                    mma(acc[c], vc, pf);
                    if constexpr (TWO) mma(acc[c], vc, rest);
                }
            }
        }
    }
    l = half_sum(l);

    // the wavefronts' parts: o = sum_w acc_w e^(m_w - m) / sum_w l_w e^(m_w - m)
    wait_loads();
    float *av = (float *)vl;                      // [32 heads][D] of this wavefront (its V is used up)
    if (n < heads) {
#pragma unroll
        for (int c = 0; c < ND; ++c)
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const int d = 32 * c + 8 * t + 4 * hi;
                if (D % 32 && d >= D) continue;
                store4(av + n * D + d, f32x4{acc[c][4 * t], acc[c][4 * t + 1], acc[c][4 * t + 2], acc[c][4 * t + 3]});
            }
        if (hi == 0) {
            stat[wave][0][n] = m;
            stat[wave][1][n] = l;
        }
    }
    __syncthreads();
    pg_join<T, D>(a, b, h0, heads, s, ks.n > 0, any_bad != 0, [&](int w, int i, int r) { return stat[w][i][r]; },
                  [&](int w, int r) { return (const float *)(smem + w * PgCfg<T, D>::WAVE) + r * D; });
}

// Up to four heads on a key head in float32, where the matrix cores would be
// the bound (a 32x32 product costs 16 times a bf16 one, most of it for idle
// columns): the same chunks on the vector units.  D / 4 lanes hold one key's
// row, 16 bytes each, so a wavefront reads 1 KB of whole rows at a time, four
// of K and four of V on their way together, and with 60 to 122 registers four
// to eight wavefronts per SIMD are there to ask.  A dot product is summed over
// its row's lanes (a vector move per factor of two); every such group of lanes
// keeps a maximum, sum and accumulators of its own, joined at the end.
//   32 heads of 128, 16 sequences of up to 4,096:   312 us by products, 191 so (5.6 TB/s)
//   32 heads of 16, 64 sequences of up to 8,192:    349 us, 192 (5.6 TB/s)
//   32 heads of 128 on 8, 32 of up to 8,192:        370 us, 225 (4.8 TB/s)
// With eight heads the sums over lanes are the bound (158 us by products, 219 so
// for 32 heads of 64 on 4; 204 and 189 at 128; 88 and 113 at 32), and bf16,
// whose products are 16 times cheaper and values dearer to unpack, gains nothing
// with one head and loses with two (102 us by products, 130 so).
template <int CTRL> __device__ __forceinline__ float dpp(float v) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));
}
// v combined over N >= 4 neighbouring lanes (all hold the result).
template <int N, typename F> __device__ __forceinline__ float over_lanes(float v, F f) {
    v = f(v, dpp<0xB1>(v));                       // lane ^ 1
    v = f(v, dpp<0x4E>(v));                       // lane ^ 2
    if (N >= 8) v = f(v, dpp<0x141>(v));          // 7 - lane: the other four
    if (N >= 16) v = f(v, dpp<0x140>(v));         // 15 - lane: the other eight
    if (N >= 32) {
        const u32x2 u = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
        v = f(__uint_as_float(u.x), __uint_as_float(u.y));
    }
    return v;
}
// v combined over lanes N apart (N >= 4).
template <int N, typename F> __device__ __forceinline__ float over_groups(float v, F f) {
    if (N <= 4) v = f(v, dpp<0x124>(v));          // rotations of the row by 4 and 8
    if (N <= 8) v = f(v, dpp<0x128>(v));
    if (N <= 16) {
        const u32x2 u = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false));
        v = f(__uint_as_float(u.x), __uint_as_float(u.y));
    }
    const u32x2 u = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false));
    return f(__uint_as_float(u.x), __uint_as_float(u.y));
}

template <int D, int R> __global__ __launch_bounds__(64 * kPgWaves) void paged_decode_rows_kernel(PgArgs a) {
    constexpr int E = 4, LPR = D / E, KPL = 64 / LPR, U = 4, KB = U * KPL;
    __shared__ int pages[kPgEntries];
    __shared__ float stat[kPgWaves][2][R];
    __shared__ __align__(16) float part[kPgWaves][R][D];
    __shared__ int any_bad;
    const int s = uniform((int)blockIdx.x / a.G), g = (int)blockIdx.x - s * a.G, b = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), grp = lane / LPR, col = lane % LPR * E;
    const int heads = a.H / a.G, h0 = g * heads;  // at most R
    const PgKeys ks = pg_keys(a, b);
    const int c0 = s * a.chunk, c1 = min(c0 + a.chunk, ks.n);
    if (c0 >= c1 && s > 0) return;
    PgChunk ck{ks, c0, c1};
    ck.open(a, b, pages, &any_bad);

    f32x4 q[R], acc[R];
    float m[R], l[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        q[r] = load4((const float *)a.q + b * a.q_sb + (h0 + min(r, heads - 1)) * a.q_sh + col);
        acc[r] = f32x4{0.f, 0.f, 0.f, 0.f};
        m[r] = kNoScore, l[r] = 0.f;
    }
    const float *kb = (const float *)a.k + g * a.sg + col, *vb = (const float *)a.v + g * a.sg + col;
    auto larger = [](float x, float y) { return fmaxf(x, y); };
    auto sum = [](float x, float y) { return x + y; };
    for (int t0 = c0 + wave * KB; t0 < c1; t0 += KB * kPgWaves) {
        f32x4 k[U], v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t at = ck.at(a, pages, t0 + u * KPL + grp);
            k[u] = load4(kb + at);
            v[u] = load4(vb + at);
        }
        float w[U][R];
        bool up = false;                          // as above: move the maxima rarely
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float d = over_lanes<LPR>(q[r].x * k[u].x + q[r].y * k[u].y + q[r].z * k[u].z + q[r].w * k[u].w, sum);
                w[u][r] = t0 + u * KPL + grp < c1 ? d : -INFINITY;
                up |= (w[u][r] - m[r]) * a.sl2 > 8.f;
            }
        }
        if (__any(up)) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                float mn = m[r];
#pragma unroll
                for (int u = 0; u < U; ++u) mn = fmaxf(mn, w[u][r]);
                const float al = __builtin_amdgcn_exp2f((m[r] - mn) * a.sl2);
                m[r] = mn;
                l[r] *= al;
                acc[r] *= al;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float p = __builtin_amdgcn_exp2f(fmaf(w[u][r], a.sl2, -m[r] * a.sl2));
                l[r] += p;
                acc[r] += p * v[u];
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const float mm = over_groups<LPR>(m[r], larger), f = __builtin_amdgcn_exp2f((m[r] - mm) * a.sl2);
        const float ll = over_groups<LPR>(l[r] * f, sum);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[r][e] = over_groups<LPR>(acc[r][e] * f, sum);
        if (grp == 0) store4(&part[wave][r][col], acc[r]);
        if (lane == 0) stat[wave][0][r] = mm, stat[wave][1][r] = ll;
    }
    __syncthreads();
    pg_join<float, D>(a, b, h0, heads, s, ks.n > 0, any_bad != 0, [&](int w, int i, int r) { return stat[w][i][r]; },
                  [&](int w, int r) { return part[w][r]; });
}

// The chunks' parts of one (sequence, query head) joined: blockDim.x / D groups
// of D threads (whole wavefronts) take every so many parts each.  Latency of the launch and of
// two dependent loads: 3.8 us for 32 rows of 16 parts, 8 for 128 of 128.
template <typename T, int D> __global__ __launch_bounds__(1024) void paged_decode_join_kernel(PgArgs a) {
    __shared__ float num_l[1024], den_l[1024 / D], max_l[16];
    const int b = (int)blockIdx.x / a.H, h = (int)blockIdx.x % a.H, tid = threadIdx.x, d = tid % D, grp = tid / D;
    const int groups = (int)blockDim.x / D;
    const PgKeys ks = pg_keys(a, b);
    const int ns = max(1, (ks.n + a.chunk - 1) / a.chunk);
    const float *acc = a.part + (int64_t)blockIdx.x * a.ns * D + d;
    const float2 *st = (const float2 *)(a.part + (int64_t)a.B * a.H * a.ns * D) + (int64_t)blockIdx.x * a.ns;   // (max, sum)
    float mm = kNoScore;
    for (int s = tid; s < ns; s += (int)blockDim.x) mm = fmaxf(mm, st[s].x);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor(mm, o));
    if ((tid & 63) == 0) max_l[tid >> 6] = mm;
    __syncthreads();
    for (int w = 0; w < (int)blockDim.x / 64; ++w) mm = fmaxf(mm, max_l[w]);
    float num = 0.f, den = 0.f;
#pragma unroll 8
    for (int s = grp; s < ns; s += groups) {
        const float2 v = st[s];
        const float f = __builtin_amdgcn_exp2f((v.x - mm) * a.sl2);
        num += f * acc[(int64_t)s * D];
        den += f * v.y;
    }
    num_l[tid] = num;
    if (d == 0) den_l[grp] = den;
    __syncthreads();
    if (grp > 0) return;
    for (int g = 1; g < groups; ++g) num += num_l[g * D + d], den += den_l[g];
    Act<T>::store((T *)a.o + b * a.o_sb + h * a.o_sh + d, ks.n > 0 || ks.bad ? num / den : 0.f);
}

// ---------------------------------------------------------------- write
// New tokens' k and v [B][T][G][D] into the rows start[b] + t of their
// sequences, t < count[b]: 16 bytes of both per thread, neighbouring threads
// in one row.  Rows that no page holds are dropped.  Bound by memory: 24 us for
// 8 prompts of up to 1,024, 32 heads of 128 in bf16 (5.9 TB/s read and written).
struct PgWriteArgs {
    const void *k, *v;
    int64_t sb, st, sg;                           // new rows' strides (both)
    void *kp, *vp;
    int64_t pp, pg, pr;                           // page, head and row strides (both)
    const int *table, *start, *count;
    int64_t table_sb, total;                      // total: 16-byte pieces of k
    int T, G, P, N, shift, nch;                   // nch: pieces of a row
    int64_t cap;
};
template <typename T> __global__ __launch_bounds__(256) void paged_write_kernel(PgWriteArgs a) {
    constexpr int E = 16 / (int)sizeof(T);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.total; i += (int64_t)gridDim.x * 256) {
        const int c = (int)(i % a.nch);
        const int64_t r = i / a.nch, bt = r / a.G;
        const int g = (int)(r % a.G), t = (int)(bt % a.T), b = (int)(bt / a.T);
        if (a.count && t >= a.count[b]) continue;
        const int64_t j = (int64_t)a.start[b] + t;
        if (j < 0 || j >= a.cap) continue;
        const int e = a.table[b * a.table_sb + (j >> a.shift)];
        if ((unsigned)e >= (unsigned)a.P) continue;
        const int64_t src = b * a.sb + t * a.st + g * a.sg + c * E;
        const int64_t dst = e * a.pp + g * a.pg + (j & ((1ll << a.shift) - 1)) * a.pr + c * E;
        const uint4 kv = *(const uint4 *)((const T *)a.k + src), vv = *(const uint4 *)((const T *)a.v + src);
        *(uint4 *)((T *)a.kp + dst) = kv;
        *(uint4 *)((T *)a.vp + dst) = vv;
    }
}

// ---------------------------------------------------------------- host
// Rows of a page as a shift: powers of two from 16, or anything where one
// page holds a whole sequence.
static int pg_shift(int64_t N, int64_t page) {
    if (N == 1) return page >= 1 && page <= (1 << 30) ? 30 : -1;
    if (page < kPgMinPage || page > (1 << 20) || (page & (page - 1))) return -1;
    int s = 0;
    while ((1ll << s) < page) ++s;
    return s;
}

static int pg_check(const char *fn, int64_t B, int64_t G, int64_t D, int64_t P, int64_t N, int64_t page, int64_t sp,
                    int64_t sg, int64_t sr, const void *k, const void *v, const int *table, const int *lengths,
                    int64_t table_sb, int dtype) {
    if (B < 1 || B > 65535 || G < 1 || P < 1 || P > INT32_MAX || N < 1 || N > (1 << 24) || N * page > (1 << 30))
        return set_error(WALSH_EINVAL, "%s: bad shape B=%lld G=%lld pages=%lld x %lld, %lld per sequence", fn,
                         (long long)B, (long long)G, (long long)P, (long long)page, (long long)N);
    if (D != 16 && D != 32 && D != 64 && D != 128)
        return set_error(WALSH_ENOTSUP, "%s: head_dim %lld (16, 32, 64 or 128)", fn, (long long)D);
    if (dtype != WALSH_F32 && dtype != WALSH_BF16) return set_error(WALSH_ENOTSUP, "%s: dtype %d", fn, dtype);
    if (pg_shift(N, page) < 0)
        return set_error(WALSH_ENOTSUP, "%s: pages of %lld rows (a power of two from %d, or one page per sequence)", fn,
                         (long long)page, kPgMinPage);
    if (!k || !v || !table || !lengths) return set_error(WALSH_EINVAL, "%s: null pointer", fn);
    if ((uintptr_t)k % 16 || (uintptr_t)v % 16 || sp % 8 || sg % 8 || sr % 8 || sr < D || sp < 0 || sg < 0 || table_sb < 0)
        return set_error(WALSH_ENOTSUP, "%s: pages must be 16-byte aligned with strides multiples of 8", fn);
    return WALSH_OK;
}

// Keys per workgroup: 1,024, so that a batch of unequal lengths ends together
// (64 sequences of up to 4,096, 32 heads of 128 in bf16: 375 us with 1,024, 384
// with 2,048, 404 with 4,096); 512 where 1,024 would leave few workgroups to
// even out the lengths and a chunk's end costs little against its rows, with
// rows of 128 bytes and up to eight heads (32 of up to 8,192, 32 heads of 128
// on 4 in bf16: 59 us with 1,024, 51 with 512; but 4 of up to 131,072: 252 and
// 258, heads of 16: 98 and 113, and 16 heads of 64 on a key head: 31 and 33);
// fewer where that would not fill the chip (two workgroups per CU), down to a
// block per wavefront.
static void pg_split(int64_t pairs, int64_t keys, int64_t R, int64_t row_bytes, int KB, int64_t *chunk, int64_t *ns) {
    const int64_t slots = 2 * (int64_t)device_info().cu_count, step = KB * kPgWaves;
    const bool few = pairs * ceil_div(keys, kPgMaxChunk) < 8 * slots;
    const int64_t most = few && R <= 8 && row_bytes >= 128 ? kPgMaxChunk / 2 : kPgMaxChunk;
    int64_t c = ceil_div(ceil_div(pairs * keys, slots), step) * step;   // what one round of workgroups would take
    *chunk = c < step ? step : c > most ? most : c;
    *ns = ceil_div(keys, *chunk);
    if (*ns < 1) *ns = 1;
}
static void pg_plan(int64_t B, int64_t H, int64_t G, int64_t cap, int64_t D, int64_t W, int64_t S, int dtype,
                    int64_t *chunk, int64_t *ns) {
    const int64_t keys = W > 0 && W + S < cap ? W + S : cap;
    const int KB = 32 * (dtype == WALSH_BF16 ? (D == 128 ? 1 : D == 64 ? 2 : 4) : (D >= 64 ? 1 : D == 32 ? 2 : 4));
    pg_split(B * G * ceil_div(H / G, 32), keys, H / G, D * (dtype == WALSH_BF16 ? 2 : 4), KB, chunk, ns);
}

}  // namespace walsh

using namespace walsh;

WALSH_EXPORT int64_t walsh_paged_decode_workspace_bytes(int64_t B, int64_t H, int64_t G, int64_t pages_per_seq,
                                                        int64_t page, int64_t D, int64_t window, int64_t sinks,
                                                        int dtype) {
    if (B < 1 || H < 1 || G < 1 || H % G || pages_per_seq < 1 || page < 1 || D < 1) return 0;
    int64_t chunk, ns;
    pg_plan(B, H, G, pages_per_seq * page, D, window, sinks < 0 ? 0 : sinks, dtype, &chunk, &ns);
    return ns > 1 ? B * H * ns * (D + 2) * 4 : 0;
}

WALSH_EXPORT int walsh_paged_decode_attention(const void *q, int64_t q_sb, int64_t q_sh, const void *k_pages,
                                              const void *v_pages, int64_t sp, int64_t sg, int64_t sr, int64_t n_pages,
                                              int64_t page, const int *table, int64_t table_sb, int64_t pages_per_seq,
                                              const int *lengths, int64_t B, int64_t H, int64_t G, int64_t D,
                                              int64_t window, int64_t sinks, float scale, void *o, int64_t o_sb,
                                              int64_t o_sh, int dtype, void *work, int64_t work_bytes, void *stream) {
    const char *fn = "walsh_paged_decode_attention";
    if (B == 0) return WALSH_OK;
    int rc = pg_check(fn, B, G, D, n_pages, pages_per_seq, page, sp, sg, sr, k_pages, v_pages, table, lengths, table_sb,
                      dtype);
    if (rc) return rc;
    if (H < 1 || H % G || H > 65535) return set_error(WALSH_EINVAL, "%s: H=%lld for G=%lld", fn, (long long)H, (long long)G);
    if (!q || !o) return set_error(WALSH_EINVAL, "%s: null pointer", fn);
    if ((uintptr_t)q % 16 || (uintptr_t)o % 16 || q_sb % 8 || q_sh % 8 || o_sb % 8 || o_sh % 8)
        return set_error(WALSH_ENOTSUP, "%s: q and o must be 16-byte aligned with strides multiples of 8", fn);
    if (!(scale > 0.f) || scale > 1e6f)
        return set_error(WALSH_EINVAL, "%s: the scale must be positive and at most 1e6", fn);
    PgArgs a{};
    a.q = q, a.q_sb = q_sb, a.q_sh = q_sh, a.k = k_pages, a.v = v_pages, a.sp = sp, a.sg = sg, a.sr = sr;
    a.table = table, a.lengths = lengths, a.table_sb = table_sb;
    a.B = (int)B, a.H = (int)H, a.G = (int)G, a.P = (int)n_pages, a.N = (int)pages_per_seq;
    a.shift = pg_shift(pages_per_seq, page);
    a.cap = pages_per_seq * page;
    a.W = window > 0 && window < a.cap ? (int)window : 0;
    a.S = sinks < 0 ? 0 : (int)(sinks < a.cap ? sinks : a.cap);
    a.sl2 = scale * kLog2e;
    a.o = o, a.o_sb = o_sb, a.o_sh = o_sh, a.part = (float *)work;
    int64_t chunk, ns;
    pg_plan(B, H, G, a.cap, D, a.W, a.S, dtype, &chunk, &ns);
    a.chunk = (int)chunk, a.ns = (int)ns;
    if (ns > 1 && (!work || work_bytes < B * H * ns * (D + 2) * 4 || (uintptr_t)work % 16))
        return set_error(WALSH_EINVAL, "%s: workspace of %lld bytes, needs %lld (16-aligned)", fn, (long long)work_bytes,
                         (long long)(B * H * ns * (D + 2) * 4));
    const int64_t gy = G * ceil_div(H / G, 32);
    // (a launch counts its threads along an axis in 32 bits)
    if (B * H >= (1 << 22) || ns * gy >= (1 << 24)) return set_error(WALSH_ENOTSUP, "%s: H=%lld B=%lld", fn, (long long)H, (long long)B);
    hipStream_t s = (hipStream_t)stream;
    attn_dispatch(dtype, D, [&](auto t, auto d) {
        typedef decltype(t) T;
        constexpr int DD = decltype(d)::value;
        const dim3 grid((unsigned)(ns * gy), (unsigned)B), threads(64 * kPgWaves);
        const int64_t R = H / G;
        if constexpr (sizeof(T) == 4) {
            if (R == 1) launch(paged_decode_rows_kernel<DD, 1>, grid, threads, 0, s, a);
            else if (R == 2) launch(paged_decode_rows_kernel<DD, 2>, grid, threads, 0, s, a);
            else if (R <= 4) launch(paged_decode_rows_kernel<DD, 4>, grid, threads, 0, s, a);
        }
        if (sizeof(T) == 2 || R > 4)
            launch(paged_decode_kernel<T, DD>, grid, threads, (uint32_t)PgCfg<T, DD>::LDS, s, a);
        // about four parts per group of threads, whole wavefronts (the maximum goes over all 64 lanes)
        constexpr int64_t wave = DD < 64 ? 64 / DD : 1;
        int64_t groups = ceil_div(ceil_div(ns, 4), wave) * wave;
        if (groups > 1024 / DD) groups = 1024 / DD;
        if (ns > 1)
            launch(paged_decode_join_kernel<T, DD>, dim3((unsigned)(B * H)), dim3((unsigned)(groups * DD)), 0, s, a);
    });
    return check_hip(hipGetLastError(), fn);
}

WALSH_EXPORT int walsh_paged_kv_write(const void *k, const void *v, int64_t sb, int64_t st, int64_t sg, int64_t B,
                                      int64_t T, int64_t G, int64_t D, void *k_pages, void *v_pages, int64_t pp,
                                      int64_t pg, int64_t pr, int64_t n_pages, int64_t page, const int *table,
                                      int64_t table_sb, int64_t pages_per_seq, const int *start, const int *count,
                                      int dtype, void *stream) {
    const char *fn = "walsh_paged_kv_write";
    if (B == 0 || T == 0) return WALSH_OK;
    int rc = pg_check(fn, B, G, D, n_pages, pages_per_seq, page, pp, pg, pr, k_pages, v_pages, table, start, table_sb,
                      dtype);
    if (rc) return rc;
    if (!k || !v || T < 0 || T > (1 << 24)) return set_error(WALSH_EINVAL, "%s: null pointer or T=%lld", fn, (long long)T);
    if ((uintptr_t)k % 16 || (uintptr_t)v % 16 || sb % 8 || st % 8 || sg % 8)
        return set_error(WALSH_ENOTSUP, "%s: k and v must be 16-byte aligned with strides multiples of 8", fn);
    const int nch = (int)(D * (dtype == WALSH_BF16 ? 2 : 4) / 16);
    PgWriteArgs a{k, v, sb, st, sg, k_pages, v_pages, pp, pg, pr, table, start, count, table_sb, B * T * G * nch,
                  (int)T, (int)G, (int)n_pages, (int)pages_per_seq, pg_shift(pages_per_seq, page), nch,
                  pages_per_seq * page};
    const int64_t wgs = ceil_div(a.total, 256), most = 16 * (int64_t)device_info().cu_count;
    const dim3 grid((unsigned)(wgs < most ? wgs : most));
    if (dtype == WALSH_BF16) launch(paged_write_kernel<uint16_t>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else launch(paged_write_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, a);
    return check_hip(hipGetLastError(), fn);
}
