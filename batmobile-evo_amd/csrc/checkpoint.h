// Activations kept in 8 bits for the backward pass.
//
// Eight channels of an atom's features [N, C, 16] (128 values; the last block of an atom may have fewer)
// share a power of two 2^E, the least with max |x| <= 448 * 2^E, E in [-110, 120], and hold x / 2^E as
// e4m3 (sign, 4 bits of exponent, 3 of mantissa, largest value 448), rounded to nearest even: a value of
// 2^-6 2^E or more is off by 2^-4 of itself at most, a smaller one by 2^-10 2^E.  The block's largest lies
// above 224 2^E (E > -110), so 2^-4 holds down to 2^-13.8 of it.  The power is exact in fp32 and bf16, and so is
// a decoded value, so the factors of the backward's products lose nothing more.  codes [N, C, 16]
// and exps [N, ceil(C / 8)] are bytes, an exponent kept as E + 127.  A value that is not finite is kept
// as NaN and has no part in the maximum.  At E = 120 the code 256 would be 2^128: values from 248 on take 240,
// which is within the same 2^-4.
#pragma once

#include "node_features.h"

namespace bmhip {

constexpr int kCkptChannels = 8;                 // channels of a block
__host__ __device__ inline int ckpt_blocks(int C) { return (C + kCkptChannels - 1) / kCkptChannels; }

// E + 127 of a block whose largest finite |x| is given: 448 = 1.75 * 2^8
__device__ __forceinline__ int ckpt_exponent(float largest) {
    const int bits = __float_as_int(largest), e = (bits >> 23) - 8 + ((bits & 0x7fffff) > 0x600000);
    return max(e, 127 - 110);
}
__device__ __forceinline__ float ckpt_up(int e) { return __int_as_float(e << 23); }           // 2^E
__device__ __forceinline__ float ckpt_down(int e) { return __int_as_float((254 - e) << 23); } // 2^-E
__device__ __forceinline__ float ckpt_finite(float v) {
    return fabsf(v) == __builtin_inff() ? __builtin_nanf("") : v;
}
// A value of a block of E = 120 as it goes to its code
__device__ __forceinline__ float ckpt_limit(float v) {
    return fabsf(v) >= 0x1.fp127f ? copysignf(0x1.ep127f, v) : v;
}
// Four values divided by 2^E as four codes
__device__ __forceinline__ unsigned ckpt_encode4(float a, float b, float c, float d, float down) {
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(a * down, b * down, 0, false);
    return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c * down, d * down, p, true);
}
__device__ __forceinline__ float4 ckpt_decode4(unsigned p, float up) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)p, false);
    const auto b = __builtin_amdgcn_cvt_pk_f32_fp8((int)p, true);
    return make_float4(a[0] * up, a[1] * up, b[0] * up, b[1] * up);
}

}  // namespace bmhip
