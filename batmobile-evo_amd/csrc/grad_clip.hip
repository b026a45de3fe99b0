// Global 2-norm of many gradient tensors and the gradients scaled to a maximum norm (no
// reference counterpart):
//
//   norm = (sum over all tensors of g^2)^1/2,  out = g min(1, max_norm / (norm + 1e-6))
//
// Two kernels: partial sums of squares per workgroup in 64 bits (no overflow, and the rounding
// of a sum of 10^8 terms stays out of the result), then every workgroup adds the partials in
// order and scales its share of the elements.  The tensors' addresses travel as kernel
// arguments, up to kClipTensors a launch, so that nothing is copied to the device first.
#include "common.h"
#include "batmobile_hip.h"

namespace bmhip {

constexpr int kClipTensors = 100;           // a launch's arguments stay under 4 KB
constexpr int kClipChunk = 8192;            // elements of a tensor a workgroup takes at a time
constexpr int kClipThreads = 256;
constexpr int kClipMaxBlocks = 1024;        // partial sums of a launch

struct ClipArgs {
    const void* in[kClipTensors];
    void* out[kClipTensors];
    int64_t numel[kClipTensors];
    int first[kClipTensors + 1];            // first chunk of each tensor
    uint8_t bf16[kClipTensors];
    int count;
};

__device__ __forceinline__ float4 clip_ld4(const void* p, int64_t i, bool bf) {
    if (!bf) return *reinterpret_cast<const float4*>((const float*)p + i);
    const uint2 u = *reinterpret_cast<const uint2*>((const uint16_t*)p + i);
    return make_float4(bf16_lo(u.x), bf16_hi(u.x), bf16_lo(u.y), bf16_hi(u.y));
}
__device__ __forceinline__ float clip_ld(const void* p, int64_t i, bool bf) {
    return bf ? __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16) : ((const float*)p)[i];
}
__device__ __forceinline__ void clip_st(void* p, int64_t i, bool bf, float v) {
    if (bf) ((uint16_t*)p)[i] = (uint16_t)(bf16_pack(v, 0.0f) & 0xffffu);
    else ((float*)p)[i] = v;
}

// f(tensor, first element, element count) for every chunk of this workgroup
template <typename F>
__device__ __forceinline__ void clip_chunks(const ClipArgs& a, F&& f) {
    const int total = a.first[a.count];
    for (int c = blockIdx.x; c < total; c += gridDim.x) {
        int lo = 0, hi = a.count - 1;
        while (lo < hi) {
            const int m = (lo + hi + 1) / 2;
            if (a.first[m] <= c) lo = m; else hi = m - 1;
        }
        const int64_t i0 = (int64_t)(c - a.first[lo]) * kClipChunk;
        f(lo, i0, (int)min((int64_t)kClipChunk, a.numel[lo] - i0));
    }
}

__device__ __forceinline__ double block_sum(double v) {
    __shared__ double sh[kClipThreads / 64];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
#pragma unroll
    for (int i = 0; i < kClipThreads / 64; ++i) v += sh[i];
    return v;
}

__global__ __launch_bounds__(kClipThreads) void clip_norm_kernel(ClipArgs a, double* part) {
    double s = 0.0;
    clip_chunks(a, [&](int k, int64_t i0, int n) {
        const bool bf = a.bf16[k];
        for (int i = threadIdx.x; i < n; i += kClipThreads) {
            const double v = clip_ld(a.in[k], i0 + i, bf);
            s = fma(v, v, s);
        }
    });
    s = block_sum(s);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__global__ __launch_bounds__(kClipThreads) void clip_scale_kernel(ClipArgs a, const double* part,
                                                                  int n_part, float max_norm,
                                                                  float* norm) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n_part; i += kClipThreads) s += part[i];
    const double total = sqrt(block_sum(s));
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
    // a norm that is not a number makes the factor, and every gradient, not a number
    const double r = (double)max_norm / (total + 1e-6);
    const float c = r < 1.0 ? (float)r : (r != r ? (float)r : 1.0f);
    clip_chunks(a, [&](int k, int64_t i0, int n) {
        const bool bf = a.bf16[k];
        for (int i = threadIdx.x; i < n; i += kClipThreads)
            clip_st(a.out[k], i0 + i, bf, clip_ld(a.in[k], i0 + i, bf) * c);
    });
}

}  // namespace bmhip

using namespace bmhip;

extern "C" size_t batteries_clip_grad_norm_workspace_bytes(int64_t n_tensors) {
    return (size_t)std::max<int64_t>(1, ceil_div(n_tensors, kClipTensors)) * kClipMaxBlocks *
           sizeof(double);
}

extern "C" int batteries_clip_grad_norm(const void* const* in, void* const* out,
                                        const int64_t* numel, const int* dtype, int64_t n_tensors,
                                        float max_norm, float* norm, void* workspace,
                                        size_t workspace_bytes, hipStream_t stream) {
    if (n_tensors < 0 || !norm || !(max_norm >= 0.0f)) return BM_ERR_ARG;
    for (int64_t i = 0; i < n_tensors; ++i)
        if (numel[i] < 0 || (dtype[i] != 0 && dtype[i] != 1) ||
            (numel[i] > 0 && (!in[i] || !out[i])) ||
            numel[i] > (int64_t)kClipChunk * (INT32_MAX / kClipTensors))
            return BM_ERR_ARG;
    if (!workspace || workspace_bytes < batteries_clip_grad_norm_workspace_bytes(n_tensors))
        return BM_ERR_WORKSPACE;
    double* part = (double*)workspace;
    int n_part = 0;
    for (int pass = 0; pass < 2; ++pass) {
        int64_t i = 0;
        do {
            ClipArgs a;
            a.count = 0;
            a.first[0] = 0;
            for (; i < n_tensors && a.count < kClipTensors; ++i) {
                if (numel[i] == 0) continue;
                a.in[a.count] = in[i];
                a.out[a.count] = out[i];
                a.numel[a.count] = numel[i];
                a.bf16[a.count] = dtype[i] == 1;
                a.first[a.count + 1] = a.first[a.count] + (int)ceil_div(numel[i], kClipChunk);
                ++a.count;
            }
            const int blocks = std::max(1, std::min(kClipMaxBlocks, a.first[a.count]));
            if (pass == 0) {
                clip_norm_kernel<<<blocks, kClipThreads, 0, stream>>>(a, part + n_part);
                n_part += blocks;
            } else {
                clip_scale_kernel<<<blocks, kClipThreads, 0, stream>>>(a, part, n_part, max_norm,
                                                                       norm);
            }
        } while (i < n_tensors);
    }
    return (int)hipGetLastError();
}
