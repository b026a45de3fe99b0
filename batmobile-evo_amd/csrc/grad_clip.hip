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

constexpr int kClipTensors = 160;           // a launch's arguments stay under 4 KB
constexpr int kClipThreads = 256;
constexpr int kClipLoads = 4;               // 16-byte loads a thread has under way
constexpr int kClipBytes = kClipThreads * kClipLoads * 16;  // a workgroup's share at a time
constexpr int kClipMaxBlocks = 1024;        // partial sums of a launch

struct ClipArgs {
    const void* in[kClipTensors];
    void* out[kClipTensors];
    uint32_t numel[kClipTensors];
    int first[kClipTensors + 1];            // first share of each tensor
    uint8_t bf16[kClipTensors];
    int count;
};
static_assert(sizeof(ClipArgs) + 64 <= 4096, "kernel arguments");

// 16 bytes at any address that an element may have (the hardware takes unaligned vectors)
struct __attribute__((packed, aligned(2))) Clip16 {
    uint32_t v[4];
};

__device__ __forceinline__ float clip_ld(const void* p, uint32_t i, bool bf) {
    return bf ? __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16) : ((const float*)p)[i];
}

// This workgroup's shares, the last first if `back`: f(tensor, first element, whole share?).
template <typename F>
__device__ __forceinline__ void clip_shares(const ClipArgs& a, bool back, F&& f) {
    const int total = a.first[a.count], b = blockIdx.x, g = gridDim.x;
    if (b >= total) return;
    const int n = (total - b - 1) / g;
    for (int i = 0; i <= n; ++i) {
        const int c = b + (back ? n - i : i) * g;
        int lo = 0, hi = a.count - 1;
        while (lo < hi) {
            const int m = (lo + hi + 1) / 2;
            if (a.first[m] <= c) lo = m; else hi = m - 1;
        }
        const uint32_t per = a.bf16[lo] ? kClipBytes / 2 : kClipBytes / 4;
        const uint32_t i0 = (uint32_t)(c - a.first[lo]) * per;
        f(lo, i0, a.numel[lo] - i0 >= per);
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

// Memory bound: 80 MB of gradients of mixed types and sizes take 20 us, 4.0 TB/s; 0.9 MB 5 us, a
// launch.
__global__ __launch_bounds__(kClipThreads) void clip_norm_kernel(ClipArgs a, double* part) {
    double s[2] = {0.0, 0.0};
    clip_shares(a, false, [&](int k, uint32_t i0, bool whole) {
        const bool bf = a.bf16[k];
        if (whole) {
            const Clip16* p = reinterpret_cast<const Clip16*>(
                (const char*)a.in[k] + (uint64_t)i0 * (bf ? 2 : 4)) + threadIdx.x;
            Clip16 x[kClipLoads];
#pragma unroll
            for (int j = 0; j < kClipLoads; ++j) x[j] = p[j * kClipThreads];
#pragma unroll
            for (int j = 0; j < kClipLoads; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    if (bf) {
                        const double u = bf16_lo(x[j].v[c]), w = bf16_hi(x[j].v[c]);
                        s[0] = fma(u, u, s[0]);
                        s[1] = fma(w, w, s[1]);
                    } else {
                        const double u = __uint_as_float(x[j].v[c]);
                        s[c & 1] = fma(u, u, s[c & 1]);
                    }
                }
            return;
        }
        for (uint32_t i = i0 + threadIdx.x; i < a.numel[k]; i += kClipThreads) {
            const double v = clip_ld(a.in[k], i, bf);
            s[0] = fma(v, v, s[0]);
        }
    });
    const double total = block_sum(s[0] + s[1]);
    if (threadIdx.x == 0) part[blockIdx.x] = total;
}

// The shares in the opposite order: the last ones read are still in the caches (30 us for the same
// 80 MB, 5.2 TB/s; in the first kernel's order both take 62.7 us instead of 60.4).
__global__ __launch_bounds__(kClipThreads) void clip_scale_kernel(ClipArgs a, const double* part,
                                                                  int n_part, float max_norm,
                                                                  float* norm) {
    double s = 0.0;
    for (int i = threadIdx.x; i < n_part; i += kClipThreads) s += part[i];
    const double total = sqrt(block_sum(s));
    if (blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
    // a norm that is not a number makes the factor, and every gradient, not a number
    const double r = (double)max_norm / (total + 1e-6);
    // a factor near fp32's smallest number would keep few of its bits: taken in two steps, both exact
    // in size (at 2^64 times its value it passes no element of 2^128 over fp32's range)
    const bool tiny = r < 0x1p-100;
    const float f = r < 1.0 ? (float)(tiny ? r * 0x1p64 : r) : (r != r ? (float)r : 1.0f);
    const float f2 = tiny ? 0x1p-64f : 1.0f;
    clip_shares(a, true, [&](int k, uint32_t i0, bool whole) {
        const bool bf = a.bf16[k];
        if (whole) {
            const uint64_t at = (uint64_t)i0 * (bf ? 2 : 4);
            const Clip16* p = reinterpret_cast<const Clip16*>((const char*)a.in[k] + at) + threadIdx.x;
            Clip16* q = reinterpret_cast<Clip16*>((char*)a.out[k] + at) + threadIdx.x;
            Clip16 x[kClipLoads];
#pragma unroll
            for (int j = 0; j < kClipLoads; ++j) x[j] = p[j * kClipThreads];
#pragma unroll
            for (int j = 0; j < kClipLoads; ++j) {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    x[j].v[c] = bf ? bf16_pack(bf16_lo(x[j].v[c]) * f * f2,
                                               bf16_hi(x[j].v[c]) * f * f2)
                                   : __float_as_uint(__uint_as_float(x[j].v[c]) * f * f2);
                q[j * kClipThreads] = x[j];
            }
            return;
        }
        for (uint32_t i = i0 + threadIdx.x; i < a.numel[k]; i += kClipThreads) {
            const float v = clip_ld(a.in[k], i, bf) * f * f2;
            if (bf) ((uint16_t*)a.out[k])[i] = (uint16_t)(bf16_pack(v, 0.0f) & 0xffffu);
            else ((float*)a.out[k])[i] = v;
        }
    });
}

}  // namespace bmhip

using namespace bmhip;

// Tensors of more than kClipMost elements travel as several entries.
constexpr int64_t kClipMost = (int64_t)1 << 31;

extern "C" size_t batteries_clip_grad_norm_workspace_bytes(int64_t n_tensors, int64_t n_elements) {
    const int64_t entries = n_tensors + n_elements / kClipMost;
    return (size_t)std::max<int64_t>(1, ceil_div(entries, kClipTensors)) * kClipMaxBlocks *
           sizeof(double);
}

extern "C" int batteries_clip_grad_norm(const void* const* in, void* const* out,
                                        const int64_t* numel, const int* dtype, int64_t n_tensors,
                                        float max_norm, float* norm, void* workspace,
                                        size_t workspace_bytes, hipStream_t stream) {
    if (n_tensors < 0 || !norm || !(max_norm >= 0.0f) ||
        (n_tensors > 0 && (!in || !out || !numel || !dtype)))
        return BM_ERR_ARG;
    int64_t elements = 0;
    for (int64_t i = 0; i < n_tensors; ++i) {
        if (numel[i] < 0 || numel[i] > (int64_t)1 << 40 || (dtype[i] != 0 && dtype[i] != 1) ||
            (numel[i] > 0 && (!in[i] || !out[i])))
            return BM_ERR_ARG;
        elements += numel[i];
    }
    if (!workspace || workspace_bytes < batteries_clip_grad_norm_workspace_bytes(n_tensors, elements))
        return BM_ERR_WORKSPACE;
    double* part = (double*)workspace;
    int n_part = 0;
    for (int pass = 0; pass < 2; ++pass) {
        int64_t i = 0, done = 0;            // tensor, and elements of it in earlier entries
        do {
            ClipArgs a;
            a.count = 0;
            a.first[0] = 0;
            while (i < n_tensors && a.count < kClipTensors) {
                const int64_t left = numel[i] - done, size = dtype[i] == 1 ? 2 : 4;
                if (left > 0) {
                    const int k = a.count++;
                    a.in[k] = (const char*)in[i] + done * size;
                    a.out[k] = (char*)out[i] + done * size;
                    a.numel[k] = (uint32_t)std::min(left, kClipMost);
                    a.bf16[k] = dtype[i] == 1;
                    a.first[k + 1] =
                        a.first[k] + (int)ceil_div((int64_t)a.numel[k] * size, kClipBytes);
                }
                if (left > kClipMost) done += kClipMost;
                else ++i, done = 0;
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
