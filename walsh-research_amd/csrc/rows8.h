// Rows of activations in blocks of 8 columns, one block to a lane: their walk,
// loads and stores at any alignment, and the random bits of dropout.
#pragma once

#include "common.h"

namespace walsh {

// ---------------------------------------------------------------- 8 values
// Bytes that the memory side's cache holds.
constexpr int64_t kCacheBytes = 256 << 20;

// 16 bytes at any element alignment (the hardware takes them at any address).
// STREAM: past the caches, for what is touched once and is more than they hold.
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
template <bool STREAM> __device__ __forceinline__ u32x4 load16(const void *p) {
    if (STREAM) return __builtin_nontemporal_load((const u32x4_any *)p);
    return *(const u32x4_any *)p;
}
template <bool STREAM> __device__ __forceinline__ void store16(void *p, u32x4 v) {
    if (STREAM) __builtin_nontemporal_store(v, (u32x4_any *)p);
    else *(u32x4_any *)p = v;
}

// Values as they lie in memory.  Of float32 a lane's 32 bytes are two accesses,
// each half of what a line holds: streamed, lines go out in halves (a gradient
// of 50,257 x 512 takes 49 us instead of 32), so they never are.
template <typename T> struct Raw8;
template <> struct Raw8<uint16_t> {
    u32x4 a;
    template <bool STREAM> __device__ __forceinline__ void load(const uint16_t *p) { a = load16<STREAM>(p); }
    template <bool STREAM> __device__ __forceinline__ void store(uint16_t *p) const { store16<STREAM>(p, a); }
    __device__ __forceinline__ void unpack(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(a[i] << 16);
            v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
        }
    }
    __device__ __forceinline__ void pack(const float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
    }
};
template <> struct Raw8<float> {
    u32x4 a, b;
    template <bool> __device__ __forceinline__ void load(const float *p) { a = load16<false>(p), b = load16<false>(p + 4); }
    template <bool> __device__ __forceinline__ void store(float *p) const { store16<false>(p, a), store16<false>(p + 4, b); }
    __device__ __forceinline__ void unpack(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(a[i]), v[4 + i] = __uint_as_float(b[i]);
    }
    __device__ __forceinline__ void pack(const float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = __float_as_uint(v[i]), b[i] = __float_as_uint(v[4 + i]);
    }
};
// The first n of 8 values, 0 behind them; and back.
template <bool STREAM = false, typename T> __device__ __forceinline__ void load8(const T *p, int n, float (&v)[8]) {
    if (n >= 8) {
        Raw8<T> r;
        r.template load<STREAM>(p);
        r.unpack(v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i < n ? Act<T>::load(p + i) : 0.f;
    }
}
template <bool STREAM = false, typename T> __device__ __forceinline__ void store8(T *p, int n, const float (&v)[8]) {
    if (n >= 8) {
        Raw8<T> r;
        r.pack(v);
        r.template store<STREAM>(p);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (i < n) Act<T>::store(p + i, v[i]);
    }
}

// ---------------------------------------------------------------- the walk
// Blocks of 8 columns of rows of C, numbered row by row; a workgroup takes
// 256 * U in a row, lanes side by side, so that what a launch costs per lane
// does not depend on C.
struct Blocks {
    uint32_t rows, per_row, magic;     // magic: ceil(2^32 / per_row), where it is used
};
constexpr uint32_t kBlocksWide = 32768;
constexpr int64_t kMaxBlocks = 0x7fffffff - 65536;   // blocks of a launch, numbered in 32 bits

inline Blocks make_blocks(int64_t rows, int64_t C) {
    const uint32_t n = (uint32_t)ceil_div(C, 8);
    return Blocks{(uint32_t)rows, n, n > 1 ? (uint32_t)((0x100000000ull + n - 1) / n) : 0u};
}
struct BlockAt {
    uint32_t row, col;                 // the block's row and its number in it
};
// The block `step` further than the one numbered `first`, for step < 32768 -
// 1024 and `first` the same in all lanes.  One division by a uniform number,
// then a product: with per_row = d <= 32768 and n < d + 32768 the error of
// ceil(2^32 / d) stays below one, as n d < 2^32; wider rows are passed at most once.
__device__ __forceinline__ BlockAt block_at(const Blocks &g, uint32_t first, uint32_t step) {
    const uint32_t row0 = first / g.per_row, n = first - row0 * g.per_row + step;
    const uint32_t q = g.per_row == 1 ? n : g.per_row <= kBlocksWide ? __umulhi(n, g.magic) : n >= g.per_row ? 1u : 0u;
    return BlockAt{row0 + q, n - q * g.per_row};
}

// ---------------------------------------------------------------- random bits
// 16 bits for each of a block's 8 columns, of the counter-based generator of
// Salmon, Moraes, Dror and Shaw ("Parallel random numbers: as easy as 1, 2,
// 3", SC 2011), four words and ten rounds with the multipliers and key steps
// given there: key the 64 bits of the seed, counter (block in the row, row,
// stream).  Column c takes half c % 2 of word (c % 8) / 2.  16 bits an
// element are one call for 8: 20 products of 32 x 32 bits, and probabilities
// in steps of 2^-16, of which the kept values' factor takes account.
struct Drop {
    const uint64_t *seed;
    uint32_t stream, drop;             // dropped where the 16 bits are below `drop` (0: nothing is)
};
__device__ __forceinline__ uint32_t xor3(uint32_t a, uint32_t b, uint32_t c) {
    return __builtin_amdgcn_bitop3_b32(a, b, c, 0x96);             // (written out it is two instructions)
}
struct DropBits {
    uint32_t k0, k1, stream, drop;
    __device__ __forceinline__ explicit DropBits(const Drop &d) : k0(0), k1(0), stream(d.stream), drop(d.drop) {
        if (d.drop) {
            const uint64_t s = *d.seed;
            k0 = (uint32_t)s, k1 = (uint32_t)(s >> 32);
        }
    }
    __device__ __forceinline__ void apply(float (&v)[8], uint32_t row, uint32_t block) const {
        if (!drop) return;
        uint32_t c0 = block, c1 = row, c2 = 0, c3 = stream, a = k0, b = k1;
#pragma unroll
        for (int i = 0; i < 10; ++i) {
            const uint64_t p = (uint64_t)c0 * 0xD2511F53u, q = (uint64_t)c2 * 0xCD9E8D57u;
            c0 = xor3((uint32_t)(q >> 32), c1, a), c1 = (uint32_t)q;
            c2 = xor3((uint32_t)(p >> 32), c3, b), c3 = (uint32_t)p;
            a += 0x9E3779B9u, b += 0xBB67AE85u;
        }
        const uint32_t w[4] = {c0, c1, c2, c3};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = (w[i] & 0xffffu) < drop ? 0.f : v[2 * i];
            v[2 * i + 1] = (w[i] >> 16) < drop ? 0.f : v[2 * i + 1];
        }
    }
};
// The factor of what is kept.
inline double kept_factor(int drop) { return drop < 65536 ? 65536. / (65536 - drop) : 0.; }

}  // namespace walsh
