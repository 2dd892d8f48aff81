// Dropout whose mask is never stored:
//     y = x 65536 / (65536 - drop)  where the element's 16 random bits (rows8.h)
//     are at least `drop`, else 0;  + residual
// The gradient of x is the same function of the output's gradient without a
// residual, its bits computed again.  What is dropped is 0 whatever x holds.
//
// A lane takes two blocks of 8 columns, whose loads go out together.  Bound by
// memory: 8,192 x 4,096 bf16 with a residual (201 MB) 32 us, its gradient (134)
// 23 us; the bits are 19 multiply-adds of 64 bits for 8 elements, 13
// instructions' time an element where a bf16 copy leaves 31.
#include <type_traits>

#include "rows8.h"

namespace walsh {

struct DropoutArgs {
    const void *x, *residual;
    void *y;
    int64_t ldx, ldr, ldy;
    int C;
    Blocks g;
    Drop d;
    float f;
};

// TR void: no residual.  U: blocks of a lane, loaded before the first is used.
// SL: loads are streamed.  Stores of bf16 always are: the output displaces less
// of what its reader needs besides (forward and gradient of 8,192 x 4,096 one
// after the other 53 us instead of 69, of x 512 8.9 instead of 10, and as long
// with a reader behind each); from 256 MB a tensor on the loads too (32,768 x
// 4,096: 211 us, of 227 with streamed stores alone and 238 without).
template <typename TX, typename TR, typename TY, int U, bool SL>
__global__ __launch_bounds__(256) void dropout_kernel(DropoutArgs a) {
    const uint32_t first = blockIdx.x * (256u * U);
    const DropBits bits(a.d);
    BlockAt at[U];
    float v[U][8], r[U][8];
#pragma unroll
    for (int j = 0; j < U; ++j) {
        at[j] = block_at(a.g, first, 256u * j + threadIdx.x);
        if (at[j].row < a.g.rows) {
            const int64_t row = at[j].row;
            const int c = 8 * (int)at[j].col;
            load8<SL>((const TX *)a.x + row * a.ldx + c, a.C - c, v[j]);
            if constexpr (!__is_same(TR, void)) load8<SL>((const TR *)a.residual + row * a.ldr + c, a.C - c, r[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < U; ++j) {
        if (at[j].row < a.g.rows) {
            bits.apply(v[j], at[j].row, at[j].col);
            const int c = 8 * (int)at[j].col;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[j][i] *= a.f;
                if constexpr (!__is_same(TR, void)) v[j][i] += r[j][i];
            }
            store8<true>((TY *)a.y + at[j].row * a.ldy + c, a.C - c, v[j]);
        }
    }
}

}  // namespace walsh

using namespace walsh;

WALSH_EXPORT int walsh_dropout(const void *x, int64_t ldx, int xdtype, const void *residual, int64_t ldr, int rdtype,
                               int64_t M, int64_t C, int drop, const int64_t *seed, int64_t rng_stream, void *y,
                               int64_t ldy, int ydtype, void *stream) {
    const char *fn = "walsh_dropout";
    if (M < 0 || C < 0 || C > 0x7fffffff - 8 || M > 0x7fffffff || M * ceil_div(C, 8) > kMaxBlocks)
        return set_error(WALSH_ENOTSUP, "%s: M=%lld rows of C=%lld pass %lld blocks of 8", fn, (long long)M, (long long)C,
                         (long long)kMaxBlocks);
    if (drop < 0 || drop > 65536 || rng_stream < 0 || rng_stream > 0xffffffffll)
        return set_error(WALSH_EINVAL, "%s: drop %d (0 to 65536), stream %lld (32 bits)", fn, drop, (long long)rng_stream);
    for (int dt : {xdtype, ydtype, residual ? rdtype : ydtype})
        if (dt != WALSH_F32 && dt != WALSH_BF16) return set_error(WALSH_ENOTSUP, "%s: dtype %d", fn, dt);
    if (M == 0 || C == 0) return WALSH_OK;
    if (!x || !y || (drop && !seed)) return set_error(WALSH_EINVAL, "%s: null pointer", fn);
    if (M > 1 && (ldx < C || ldy < C || (residual && ldr < C)))
        return set_error(WALSH_EINVAL, "%s: rows of %lld overlap", fn, (long long)C);
    constexpr int U = 2;
    const DropoutArgs a{x, residual, y, ldx, ldr, ldy, (int)C, make_blocks(M, C),
                        Drop{(const uint64_t *)seed, (uint32_t)rng_stream, (uint32_t)drop}, (float)kept_factor(drop)};
    const dim3 G((unsigned)ceil_div(M * a.g.per_row, 256 * U)), N(256);
    const hipStream_t s = (hipStream_t)stream;
    const bool xb = xdtype == WALSH_BF16, rb = rdtype == WALSH_BF16, yb = ydtype == WALSH_BF16;
    if (residual ? yb != (xb && rb) : xb && !yb)
        return set_error(WALSH_ENOTSUP, "%s: the output has the wider type of x and the residual", fn);
    auto go = [&](auto x, auto r, auto y) {
        using TX = decltype(x);
        using TR = std::conditional_t<std::is_same_v<decltype(r), char>, void, decltype(r)>;
        using TY = decltype(y);
        if constexpr (sizeof(TX) == 2) {
            if (M * C * 2 >= kCacheBytes) return launch(dropout_kernel<TX, TR, TY, U, true>, G, N, 0, s, a);
        }
        launch(dropout_kernel<TX, TR, TY, U, false>, G, N, 0, s, a);
    };
    constexpr uint16_t b16 = 0;
    constexpr float f32 = 0;
    constexpr char none = 0;
    if (!residual) {
        if (xb) go(b16, none, b16);
        else if (yb) go(f32, none, b16);
        else go(f32, none, f32);
    } else {
        if (xb && rb) go(b16, b16, b16);
        else if (xb) go(b16, f32, f32);
        else if (rb) go(f32, b16, f32);
        else go(f32, f32, f32);
    }
    return check_hip(hipGetLastError(), fn);
}
