// Matrix-core tiles of the attention kernels (gfx950): operands of eight
// elements per lane for 32x32x16 products in bf16 and float32, and tiles of
// rows in LDS that are read both by rows and by columns.
#pragma once

#include <type_traits>

#include "common.h"

namespace walsh {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short i16x8 __attribute__((ext_vector_type(8)));

constexpr float kNoScore = -1e30f;  // running maximum of a row that has seen nothing: finite, so differences stay numbers
constexpr float kLog2e = 1.4426950408889634f;

// ---------------------------------------------------------------- operands
// Eight elements of one row or column: a product operand.
template <typename T> struct Frag;
template <> struct Frag<uint16_t> { i16x8 v; };
template <> struct Frag<float> { f32x8 v; };

__device__ __forceinline__ void mma(f32x16 &c, const Frag<uint16_t> &a, const Frag<uint16_t> &b) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a.v), __builtin_bit_cast(bf16x8, b.v), c, 0,
                                                0, 0);
}
__device__ __forceinline__ void mma(f32x16 &c, const Frag<float> &a, const Frag<float> &b) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[i], b.v[i], c, 0, 0, 0);
}
// Result rows 16 t + (4 hi + 0..3, 8 + 4 hi + 0..3) as an operand.
__device__ __forceinline__ void pack(Frag<uint16_t> &f, const float *p) {
    const u32x4 u = {pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]), pack_bf16x2(p[4], p[5]),
                     pack_bf16x2(p[6], p[7])};
    f.v = __builtin_bit_cast(i16x8, u);
}
__device__ __forceinline__ void pack(Frag<float> &f, const float *p) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f.v[i] = p[i];
}
// What pack rounded away, as an operand of its own.
__device__ __forceinline__ void pack_rest(Frag<uint16_t> &f, const float *p, const Frag<uint16_t> &packed) {
    const u32x4 u = __builtin_bit_cast(u32x4, packed.v);
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r[i] = pack_bf16x2(p[2 * i] - __uint_as_float(u[i] << 16), p[2 * i + 1] - __uint_as_float(u[i] & 0xffff0000u));
    f.v = __builtin_bit_cast(i16x8, r);
}
__device__ __forceinline__ Frag<uint16_t> load_frag(const uint16_t *p) { return {*(const i16x8 *)p}; }
__device__ __forceinline__ Frag<float> load_frag(const float *p) {
    const f32x4 a = *(const f32x4 *)p, b = *(const f32x4 *)(p + 4);
    return {f32x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
}
__device__ __forceinline__ float dot(const Frag<float> &a, const Frag<float> &b) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += a.v[i] * b.v[i];
    return s;
}
__device__ __forceinline__ float dot(const Frag<uint16_t> &a, const Frag<uint16_t> &b) {
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) s += bf16_to_f32((uint16_t)a.v[i]) * bf16_to_f32((uint16_t)b.v[i]);
    return s;
}

// c and the sum of an operand's elements (two to an instruction).
__device__ __forceinline__ float add_all(float c, const Frag<uint16_t> &f) {
    const u32x4 u = __builtin_bit_cast(u32x4, f.v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t pair = u[i];               // (of an element itself the cast takes the first)
        c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), __builtin_bit_cast(bf16x2, 0x3f803f80u), c, false);
    }
    return c;
}

__device__ __forceinline__ float add_all(float c, const Frag<float> &f) {
    return c + (((f.v[0] + f.v[1]) + (f.v[2] + f.v[3])) + ((f.v[4] + f.v[5]) + (f.v[6] + f.v[7])));
}

// A value that is the same in every lane, as a scalar: quotients and loads
// leave such values in vector registers, and their users with them.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// The value, newly computed as far as the compiler can see: what derives from
// it is worked out again where it is used and holds no registers across a loop.
__device__ __forceinline__ int fresh(int v) {
    asm volatile("" : "+v"(v));
    return v;
}

// Sum and maximum of a lane's value and that of lane ^ 32, by the exchange of
// the wavefront's halves (vector unit; no LDS round trip as a shuffle has).
__device__ __forceinline__ float half_sum(float v) {
    const u32x2 u = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v),
                                                                              false, false));
    return __uint_as_float(u.x) + __uint_as_float(u.y);
}
__device__ __forceinline__ float half_max(float v) {
    const u32x2 u = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v),
                                                                              false, false));
    return fmaxf(__uint_as_float(u.x), __uint_as_float(u.y));
}

// ---------------------------------------------------------------- loads into LDS
// 16 (4) bytes per lane from a buffer at byte offset off (past its size:
// zeros) to 64 consecutive slots at the LDS byte address lds; both scalar but
// off.  Written out, because the compiler makes every LDS read through the
// transposing load wait for all such loads of its own that are on their way,
// next tile's included.  Nothing comes back in registers; the caller waits
// (tiles_ready) before it reads.  (M0, the LDS address of such a load, has no
// other user in kernels that call this.)
__device__ __forceinline__ u32x4 lds_load_rsrc(const void *p, uint32_t bytes) {
    const uint64_t a = (uint64_t)p;
    return u32x4{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a),
                 (uint32_t)__builtin_amdgcn_readfirstlane((int)((uint32_t)(a >> 32) & 0xffffu)),
                 (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}
template <int BYTES> __device__ __forceinline__ void lds_load(u32x4 rsrc, uint32_t off, uint32_t lds) {
    static_assert(BYTES == 16 || BYTES == 4, "sizes in use");
    lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds);
    if (BYTES == 16)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                     ::"s"(lds), "v"(off), "s"(rsrc) : "memory");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
                     ::"s"(lds), "v"(off), "s"(rsrc) : "memory");
}
// 16 bytes per lane from each lane's own address, likewise.
__device__ __forceinline__ void lds_gather(const void *p, uint32_t lds) {
    lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory");
}
// The LDS byte address of a shared variable, as a scalar.
__device__ __forceinline__ uint32_t lds_addr(const void *p) {
    return (uint32_t)__builtin_amdgcn_readfirstlane(
        (int)(uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void *)p);
}

// ---------------------------------------------------------------- tiles in LDS
// ROWS rows of D elements, row-major in 16-byte chunks; chunk c of row r lies
// at position c ^ swz(r), so that the 16 rows of one chunk column fall on
// distinct banks (row operands) and so do the four rows of a transposing load.
template <typename T, int D, int ROWS> struct Tile {
    static constexpr int NCH = D * (int)sizeof(T) / 16;       // chunks per row: 2 .. 32
    static constexpr int ROWB = D * (int)sizeof(T);
    static constexpr int BYTES = ROWS * ROWB;
    static __device__ __forceinline__ int swz(int r) {
        if (sizeof(T) == 4) return NCH >= 16 ? r & 15 : NCH == 8 ? (r >> 1) & 7 : (r >> 2) & 3;
        if (NCH == 16) return ((r & 3) << 2) | ((r >> 2) & 3);
        if (NCH == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
        return NCH == 4 ? (r >> 2) & 3 : (r >> 3) & 1;
    }
    // Rows r0 .. r0 + ROWS - 1 of a matrix with row stride st into LDS, by
    // WAVES wavefronts (wave: a scalar), straight from memory (no registers);
    // rows before lo and at or past n are zeros and are not read.
    template <int WAVES>
    static __device__ __forceinline__ void fetch(unsigned char *lds, const T *base, int64_t st, int r0, int lo, int n, int wave,
                                                 int lane) {
        const int rows = min(n - r0, ROWS);
        const uint32_t span = rows > 0 ? (uint32_t)(((int64_t)(rows - 1) * st + D) * (int)sizeof(T)) : 0u;
        const u32x4 rs = lds_load_rsrc(base + (int64_t)r0 * st, span);
        const uint32_t dst = lds_addr(lds);
        constexpr int N = BYTES / 1024, STEP = 64 * WAVES / NCH;   // wavefront loads; rows that one of each cover
        static_assert(BYTES % 1024 == 0, "whole loads");
        const uint32_t rowb = (uint32_t)(st * (int)sizeof(T)), pos0 = (uint32_t)(wave * 64 + lane);
        const int row0 = (int)(pos0 / NCH);
        uint32_t c = (pos0 % NCH) ^ swz(row0);
#pragma unroll
        for (int i = 0; i < (N + WAVES - 1) / WAVES; ++i) {
            const int k = i * WAVES + wave, row = row0 + i * STEP;
            if (N % WAVES && k >= N) break;
            if (STEP % 16) c = (pos0 % NCH) ^ swz(row);            // (else the swizzle, of period 16, is the same)
            const uint32_t off = row < rows && row >= lo - r0 ? (uint32_t)row * rowb + 16 * c : kOOB;
            lds_load<16>(rs, off, dst + k * 1024);
        }
    }
    // The same of many tiles of one stride (st >= D), what depends on the lane
    // alone worked out once: rows past the last one lie past the buffer.
    template <int WAVES> struct Loads {
        static constexpr int N = BYTES / 1024, PER = (N + WAVES - 1) / WAVES;
        uint32_t off[PER];
        __device__ __forceinline__ Loads(int64_t st, int wave, int lane) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const uint32_t pos = (uint32_t)((i * WAVES + wave) * 64 + lane);
                const int row = (int)(pos / NCH);
                off[i] = (uint32_t)row * (uint32_t)(st * (int)sizeof(T)) + 16 * ((pos % NCH) ^ swz(row));
            }
        }
        __device__ __forceinline__ void go(unsigned char *lds, const T *base, int64_t st, int r0, int n, int wave) const {
            const int rows = min(n - r0, ROWS);
            const uint32_t span = rows > 0 ? (uint32_t)(((rows - 1) * (int)st + D) * (int)sizeof(T)) : 0u;
            const u32x4 rs = lds_load_rsrc(base + r0 * st, span);
            const uint32_t dst = lds_addr(lds) + wave * 1024;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (N % WAVES && i * WAVES + wave >= N) break;
                lds_load<16>(rs, off[i], dst + i * WAVES * 1024);
            }
        }
    };
    // Eight elements of row r from column 16 kk + 8 hi, and of column
    // 32 c + lane % 32 (modulo D) the rows r + 4 hi + 0..3 and r + 8 + 4 hi +
    // 0..3 (r a multiple of 16).  A swizzle's bits are bits of the row, so an
    // operand's address is that of the first one, worked out once, with an
    // exclusive or and an offset that the instruction holds (tiles lie at
    // multiples of 1,024 bytes).
    static __device__ __forceinline__ uint32_t row_base(const unsigned char *lds, int r, int hi) {
        return lds_addr(lds) + r * ROWB + ((((int)sizeof(T) / 2 * hi) ^ swz(r)) << 4);
    }
    static __device__ __forceinline__ uint32_t row_step(int kk) { return (uint32_t)kk * 16 * sizeof(T); }
    static __device__ __forceinline__ Frag<T> row_from(uint32_t base, int kk) {
        base ^= row_step(kk);
        if constexpr (sizeof(T) == 2) {
            return {*lds_at<i16x8>(base)};
        } else {
            const f32x4 a = *lds_at<f32x4>(base), b = *lds_at<f32x4>(base ^ 16);
            return {f32x8{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}};
        }
    }
    static __device__ __forceinline__ uint32_t col_base(const unsigned char *lds, int lane) {
        const int hi = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            const int l = lane & 15, half = D >= 32 ? (lane >> 4) & 1 : 0, r = 4 * hi + (l >> 2);
            return lds_addr(lds) + r * ROWB + (((2 * half + ((l & 3) >> 1)) ^ swz(r)) << 4) + 8 * (l & 1);
        } else {
            const int d = (lane & 31) % D;
            return lds_addr(lds) + 4 * hi * ROWB + (((d >> 2) ^ swz(4 * hi)) << 4) + 4 * (d & 3);
        }
    }
    static __device__ __forceinline__ Frag<T> col_from(uint32_t base, int r, int c) {
        if constexpr (sizeof(T) == 2) {
            typedef short i16x4v __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) i16x4v *P;
            const uint32_t a = base ^ (c << 6), b = a ^ (swz(8) << 4);
            const i16x4v u = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(uintptr_t)(a + r * ROWB));
            const i16x4v v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(uintptr_t)(b + (r + 8) * ROWB));
            return {__builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7)};
        } else {
            f32x8 v;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int k = (e & 3) + 8 * (e >> 2);
                v[e] = *lds_at<float>((base ^ (c << 7) ^ (swz(k) << 4)) + (r + k) * ROWB);
            }
            return {v};
        }
    }
    template <typename V> static __device__ __forceinline__ __attribute__((address_space(3))) const V *lds_at(uint32_t at) {
        return (__attribute__((address_space(3))) const V *)(uintptr_t)at;
    }
    static __device__ __forceinline__ Frag<T> col(const unsigned char *lds, int r, int c, int lane) {
        return col_from(col_base(lds, lane), r, c);
    }
};

// All loads of this wavefront have landed and its LDS reads are done: vmcnt(0)
// lgkmcnt(0), as the builtin that the compiler's own count of loads follows.
__device__ __forceinline__ void wait_loads() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);
    asm volatile("" ::: "memory");
}
// The same of all wavefronts: tiles requested before are there.
__device__ __forceinline__ void tiles_ready() {
    wait_loads();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Order of the LDS reads and products before this call, in its basic block: N
// products of READS reads each, the reads of DEPTH products ahead.  Left to
// itself the compiler, short of registers, puts each read right before its
// product, which then waits out the LDS latency, four times its own length.
template <int READS, int N, int DEPTH> __device__ __forceinline__ void pace() {
    __builtin_amdgcn_sched_group_barrier(0x100, READS * DEPTH, 0);
#pragma unroll
    for (int i = 0; i < N - DEPTH; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, DEPTH, 0);
}

// Calls go(T(), integral constant D) for the dtype and head_dim at hand.
template <typename F> static void attn_dispatch(int dtype, int64_t D, F go) {
    auto by_dim = [&](auto t) {
        if (D == 16) go(t, std::integral_constant<int, 16>());
        else if (D == 32) go(t, std::integral_constant<int, 32>());
        else if (D == 64) go(t, std::integral_constant<int, 64>());
        else go(t, std::integral_constant<int, 128>());
    };
    if (dtype == WALSH_BF16) by_dim(uint16_t(0));
    else by_dim(float(0));
}

}  // namespace walsh
