// Sums over lanes and over partial results, in a fixed order.
#pragma once

#include "node_features.h"

namespace bmhip {

// Sum (or maximum) over the groups of LANES lanes (2 to 64, a power of two) that follow each other, in
// every lane of the group.
template <int LANES, typename F>
__device__ __forceinline__ float lanes_reduce(float v, F&& f) {
    typedef unsigned v2u __attribute__((ext_vector_type(2)));
    if constexpr (LANES >= 2) v = f(v, quad<1, 0, 3, 2>(v));
    if constexpr (LANES >= 4) v = f(v, quad<2, 3, 0, 1>(v));
    if constexpr (LANES >= 8) v = f(v, dpp<0x141>(v));        // row_half_mirror
    if constexpr (LANES >= 16) v = f(v, dpp<0x140>(v));       // row_mirror
    if constexpr (LANES >= 32) {
        const v2u r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v),
                                                       false, false);
        v = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    if constexpr (LANES >= 64) {
        const v2u r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v),
                                                       false, false);
        v = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    }
    return v;
}
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
    return lanes_reduce<LANES>(v, [](float a, float b) { return a + b; });
}
template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
    return lanes_reduce<LANES>(v, [](float a, float b) { return fmaxf(a, b); });
}

// Sum of at(r), r = 0 .. rows - 1, over the 64 threads of column threadIdx.x % 16 of a workgroup of
// 1024 (at: of that column), in every thread.
template <typename F>
__device__ __forceinline__ float column_sum(int rows, F&& at) {
    __shared__ float sh[64][17];
    const int lane = threadIdx.x & 15, k = threadIdx.x >> 4;
    float s = 0.0f;
#pragma unroll 8
    for (int r = k; r < rows; r += 64) s += at(r);
    sh[k][lane] = s;
    __syncthreads();
    for (int o = 32; o > 0; o >>= 1) {
        if (k < o) sh[k][lane] += sh[k + o][lane];
        __syncthreads();
    }
    return sh[0][lane];
}

}  // namespace bmhip
