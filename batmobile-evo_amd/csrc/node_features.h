// Device helpers for features [N, C, 16] in fp32 or bf16: loads and stores of components, sums over
// neighbouring lanes, the sigmoid and its complement.
#pragma once

#include "common.h"

namespace bmhip {

// Four components as they lie in memory (bf16 takes half the registers until it is used)
template <typename T>
struct Raw4;
template <>
struct Raw4<float> {
    float4 v;
    __device__ __forceinline__ void load(const float* p) { v = *reinterpret_cast<const float4*>(p); }
    __device__ __forceinline__ void zero() { v = make_float4(0, 0, 0, 0); }
    __device__ __forceinline__ float4 get() const { return v; }
};
template <>
struct Raw4<uint16_t> {
    uint2 v;
    __device__ __forceinline__ void load(const uint16_t* p) {
        v = *reinterpret_cast<const uint2*>(p);
    }
    __device__ __forceinline__ void zero() { v = make_uint2(0, 0); }
    __device__ __forceinline__ float4 get() const {
        return make_float4(bf16_lo(v.x), bf16_hi(v.x), bf16_lo(v.y), bf16_hi(v.y));
    }
};
template <typename T>
__device__ __forceinline__ float4 norm_ld4(const T* p) {
    Raw4<T> r;
    r.load(p);
    return r.get();
}
__device__ __forceinline__ void norm_st4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void norm_st4(uint16_t* p, float4 v) {
    *reinterpret_cast<uint2*>(p) = make_uint2(bf16_pack(v.x, v.y), bf16_pack(v.z, v.w));
}
__device__ __forceinline__ float norm_ld(const float* p) { return *p; }
__device__ __forceinline__ float norm_ld(const uint16_t* p) {
    return __uint_as_float((uint32_t)*p << 16);
}
__device__ __forceinline__ void norm_st(float* p, float v) { *p = v; }
__device__ __forceinline__ void norm_st(uint16_t* p, float v) {
    *p = (uint16_t)(bf16_pack(v, 0.0f) & 0xffffu);
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <int S0, int S1, int S2, int S3>
__device__ __forceinline__ float quad(float v) {
    return dpp<S0 | (S1 << 2) | (S2 << 4) | (S3 << 6)>(v);
}

// sigmoid(g) and 1 - sigmoid(g), each to full relative precision at any g: the smaller one comes of the
// exponential of -|g|, the larger is 1 less that.  One register: the smaller, with a minus if it is
// 1 - sigmoid.
__device__ __forceinline__ float sigmoid_pair(float g) {
    const float a = fabsf(g) > 256.0f ? 128.0f : fabsf(g) * 0.5f; // (infinities end at 0, NaN stays)
    const float x = a * -1.44269504f;                             // log2 e, and what it leaves out
    float e = __builtin_amdgcn_exp2f(x);                          // exp(-|g| / 2), to the square
    e *= fmaf(fmaf(a, -1.44269504f, -x) - a * 1.92596299e-8f, 0.693147181f, 1.0f);
    e *= e;
    return copysignf(e * __builtin_amdgcn_rcpf(1.0f + e), -g);
}
__device__ __forceinline__ float sigmoid_on(float p) {
    return __float_as_int(p) < 0 ? 1.0f + p : p;
}
__device__ __forceinline__ float sigmoid_off(float p) {
    return __float_as_int(p) < 0 ? -p : 1.0f - p;
}

}  // namespace bmhip
