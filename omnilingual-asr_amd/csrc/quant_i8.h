// Row quantisation to 8-bit integers (device helpers shared by the quantiser, the LayerNorm kernels that write int8
// rows and the product kernel that quantises its few rows itself):
//   scale = max|x| / 127 (1 for an all-zero row),  q = rint(127 x / max|x|), ties to even, |q| <= 127.
#pragma once
#include "oasr_common.h"

namespace oasr {
namespace i8 {

// One row's factors, from the bit pattern of max|x|.  NaN patterns are the largest ones, so a row that holds a NaN or
// an infinity gets a scale that is one, and every output made from the row is NaN rather than a plausible number.
// `pre` (a power of two, so exact) keeps 127 x and 1 / max|x| inside float32's range for rows at its ends.
struct RowScale {
    float scale;   // max|x| / 127
    float gain;    // 127 * pre, pre = 1, 2^64 or 2^-64
    float top;     // max|x| * pre
    float inv;     // 1 / top
};

__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
    RowScale r;
    const float amax = __uint_as_float(amax_bits);
    r.scale = amax_bits ? amax / 127.0f : 1.0f;
    const float pre = amax_bits < 0x20000000u ? 0x1p64f : (amax_bits > 0x5f000000u ? 0x1p-64f : 1.0f);   // 2^-63, 2^63
    r.gain = 127.0f * pre;
    r.top = amax_bits ? amax * pre : 1.0f;
    r.inv = 1.0f / r.top;
    return r;
}

// rint of |v| <= 127 into the low byte (two's complement): adding 1.5 * 2^23 leaves the integer, rounded to nearest
// even, in the low bits of the sum.
__device__ __forceinline__ uint32_t code_bits(float v) { return __float_as_uint(v + 12582912.0f); }

// A bf16 value's code, decided exactly.  127 x has 15 significant bits; the quotient's residual t - r * top is exact
// (at most 10 bits above its last place), so one correction step returns the exact quotient wherever that has few
// bits.  Ties (x = max / 2 is 63.5) are therefore ties, and no other bf16 quotient comes within 2^-16 of one.
__device__ __forceinline__ uint32_t code_of_bf16(float x, const RowScale& s) {
    const float t = x * s.gain;
    const float r = t * s.inv;
    return code_bits(fmaf(fmaf(-r, s.top, t), s.inv, r));
}

// A float32 value's code, 127 x / max|x| in two rounded products (not in one with 127 / max|x|, which leaves float32's range
// for tiny rows).  A quotient within 2^-16 of a tie may go either way.
__device__ __forceinline__ uint32_t code_of_f32(float x, const RowScale& s) { return code_bits((x * s.gain) * s.inv); }

// The low bytes of four words.
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const uint32_t ab = __builtin_amdgcn_perm(b, a, 0x0c0c0400u);
    const uint32_t cd = __builtin_amdgcn_perm(d, c, 0x04000c0cu);
    return ab | cd;
}

__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t u = __shfl_xor(v, o, 64);
        v = v > u ? v : u;
    }
    return v;
}

// The largest over aligned groups of eight lanes, without LDS (the mirrored partner holds the other quad's).
__device__ __forceinline__ uint32_t eight_umax(uint32_t v) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xf, 0xf, true));    // quad_perm [1 0 3 2]
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xf, 0xf, true));    // quad_perm [2 3 0 1]
    return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xf, 0xf, true));  // row_half_mirror
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

}  // namespace i8
}  // namespace oasr
