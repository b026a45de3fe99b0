// Gated activation of features [N, C, 16], and the 8-bit form of features (no reference counterpart).
//
//   y[c, m] = sigmoid(x[c, 0]) x[c, m]             (silu of the invariant, the rest gated by it: the factor
//                                                   is the same for all components of a degree)
//   gx[c, m] = s g[c, m] + [m = 0] s (1 - s) sum_k g[c, k] x[c, k],   s = sigmoid(x[c, 0])
//
// Memory bound, one pass each way.  Forward, y and the 8-bit form of x come of the same registers; the
// backward takes x or its 8-bit form.  A block of 8 channels is 32 lanes of four components in fp32 and
// 16 lanes of eight in bf16, 16 bytes a lane: a channel is a quad or a pair of lanes.  Measured: 50,000 x 256
// in bf16 with the 8-bit form forward 174 us (5.9 TB/s), backward 194 us (5.3 TB/s); the 8-bit form alone
// of 50,000 x 128 57 us.
#include "checkpoint.h"
#include "sums.h"
#include "batmobile_hip.h"

namespace bmhip {

constexpr int kGateMaxC = 2048;

struct GateArgs {
    const void *x, *g;
    const uint8_t *codes_in, *exps_in;
    void *y;
    uint8_t *codes, *exps;
    uint32_t blocks;                       // of a launch: atoms * ckpt_blocks(C)
    int C;
};

template <typename T>
struct Chan;                               // a lane's components of a channel
template <>
struct Chan<float> {
    static constexpr int kN = 4, kLanes = 4;
    float v[4];
    __device__ __forceinline__ void load(const float* p) {
        const float4 t = *reinterpret_cast<const float4*>(p);
        v[0] = t.x, v[1] = t.y, v[2] = t.z, v[3] = t.w;
    }
    __device__ __forceinline__ void store(float* p) const {
        *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    }
    __device__ __forceinline__ float first() const { return quad<0, 0, 0, 0>(v[0]); }
};
template <>
struct Chan<uint16_t> {
    static constexpr int kN = 8, kLanes = 2;
    float v[8];
    __device__ __forceinline__ void load(const uint16_t* p) {
        const uint4 t = *reinterpret_cast<const uint4*>(p);
        v[0] = bf16_lo(t.x), v[1] = bf16_hi(t.x), v[2] = bf16_lo(t.y), v[3] = bf16_hi(t.y);
        v[4] = bf16_lo(t.z), v[5] = bf16_hi(t.z), v[6] = bf16_lo(t.w), v[7] = bf16_hi(t.w);
    }
    __device__ __forceinline__ void store(uint16_t* p) const {
        *reinterpret_cast<uint4*>(p) = make_uint4(bf16_pack(v[0], v[1]), bf16_pack(v[2], v[3]),
                                                  bf16_pack(v[4], v[5]), bf16_pack(v[6], v[7]));
    }
    __device__ __forceinline__ float first() const { return quad<0, 0, 2, 2>(v[0]); }
};

// Where a lane's components lie: block b of the features, this lane's share of it
struct Place {
    int64_t at;                            // element
    bool there;
};
template <typename T>
__device__ __forceinline__ Place place_of(uint32_t b, int lane, int C) {
    constexpr int kN = Chan<T>::kN;
    if (C % kCkptChannels == 0) return {(int64_t)b * 128 + lane * kN, true};
    const uint32_t per = ckpt_blocks(C), n = b / per, k = b - n * per;
    const int c = k * kCkptChannels + lane / Chan<T>::kLanes;
    return {((int64_t)n * C + c) * 16 + lane % Chan<T>::kLanes * kN, c < C};
}

constexpr int kGateAhead = 4;              // blocks of a lane under way

// y (ACT), codes and exps (KEEP)
template <typename T, bool ACT, bool KEEP>
__global__ __launch_bounds__(256) void gate_fwd_kernel(GateArgs a) {
    constexpr int kN = Chan<T>::kN, kLanes = 128 / kN, kPer = 256 / kLanes;
    const int lane = threadIdx.x % kLanes;
    const uint32_t b0 = (uint32_t)blockIdx.x * (kPer * kGateAhead) + threadIdx.x / kLanes;
    Chan<T> x[kGateAhead];
    Place p[kGateAhead];
#pragma unroll
    for (int i = 0; i < kGateAhead; ++i) {
        const uint32_t b = b0 + i * kPer;
        p[i] = place_of<T>(b, lane, a.C);
        p[i].there = p[i].there && b < a.blocks;
        if (p[i].there) x[i].load((const T*)a.x + p[i].at);
        else
#pragma unroll
            for (int j = 0; j < kN; ++j) x[i].v[j] = 0.0f;
    }
#pragma unroll
    for (int i = 0; i < kGateAhead; ++i) {
        if constexpr (KEEP) {
            float v[kN], m = 0.0f;
#pragma unroll
            for (int j = 0; j < kN; ++j) {
                v[j] = ckpt_finite(x[i].v[j]);
                m = fmaxf(m, fabsf(v[j]));             // (fmaxf drops a NaN)
            }
            const int e = ckpt_exponent(lanes_max<kLanes>(m));
            const float down = ckpt_down(e);
            if (e == 127 + 120) {
#pragma unroll
                for (int j = 0; j < kN; ++j) v[j] = ckpt_limit(v[j]);
            }
            if (p[i].there) {
                if constexpr (kN == 4)
                    *reinterpret_cast<unsigned*>(a.codes + p[i].at) =
                        ckpt_encode4(v[0], v[1], v[2], v[3], down);
                else
                    *reinterpret_cast<uint2*>(a.codes + p[i].at) =
                        make_uint2(ckpt_encode4(v[0], v[1], v[2], v[3], down),
                                   ckpt_encode4(v[4], v[5], v[6], v[7], down));
                if (lane == 0) a.exps[b0 + i * kPer] = (uint8_t)e;
            }
        }
        if constexpr (ACT) {
            const float s = sigmoid_on(sigmoid_pair(x[i].first()));
#pragma unroll
            for (int j = 0; j < kN; ++j) x[i].v[j] *= s;
            if (p[i].there) x[i].store((T*)a.y + p[i].at);
        }
    }
}

// gx from g and x or (KEPT) its codes; without GRAD the decoded features
template <typename T, bool KEPT, bool GRAD>
__global__ __launch_bounds__(256) void gate_bwd_kernel(GateArgs a) {
    constexpr int kN = Chan<T>::kN, kLanes = 128 / kN, kPer = 256 / kLanes;
    const int lane = threadIdx.x % kLanes;
    const uint32_t b0 = (uint32_t)blockIdx.x * (kPer * kGateAhead) + threadIdx.x / kLanes;
    Chan<T> x[kGateAhead], g[kGateAhead];
    Place p[kGateAhead];
    unsigned codes[kGateAhead][kN / 4];
    int exps[kGateAhead];
#pragma unroll
    for (int i = 0; i < kGateAhead; ++i) {
        const uint32_t b = b0 + i * kPer;
        p[i] = place_of<T>(b, lane, a.C);
        p[i].there = p[i].there && b < a.blocks;
        if (!p[i].there) p[i].at = 0;                  // some element that is there
        if constexpr (KEPT) {
            if constexpr (kN == 4) {
                codes[i][0] = *reinterpret_cast<const unsigned*>(a.codes_in + p[i].at);
            } else {
                const uint2 c = *reinterpret_cast<const uint2*>(a.codes_in + p[i].at);
                codes[i][0] = c.x, codes[i][1] = c.y;
            }
            exps[i] = a.exps_in[min(b, a.blocks - 1)];
        } else {
            x[i].load((const T*)a.x + p[i].at);
        }
        if constexpr (GRAD) g[i].load((const T*)a.g + p[i].at);
    }
#pragma unroll
    for (int i = 0; i < kGateAhead; ++i) {
        if constexpr (KEPT) {
            const float up = ckpt_up(exps[i]);
#pragma unroll
            for (int j = 0; j < kN / 4; ++j) {
                const float4 v = ckpt_decode4(codes[i][j], up);
                x[i].v[4 * j] = v.x, x[i].v[4 * j + 1] = v.y;
                x[i].v[4 * j + 2] = v.z, x[i].v[4 * j + 3] = v.w;
            }
        }
        if constexpr (GRAD) {
            float d = 0.0f;
#pragma unroll
            for (int j = 0; j < kN; ++j) d = fmaf(g[i].v[j], x[i].v[j], d);
            d = lanes_sum<Chan<T>::kLanes>(d);
            const float pair = sigmoid_pair(x[i].first());
            const float s = sigmoid_on(pair);
#pragma unroll
            for (int j = 0; j < kN; ++j) x[i].v[j] = s * g[i].v[j];
            if (lane % Chan<T>::kLanes == 0)
                x[i].v[0] = fmaf(s * sigmoid_off(pair), d, x[i].v[0]);
        }
        if (p[i].there) x[i].store((T*)a.y + p[i].at);
    }
}

// Blocks of a launch: 2^31 threads at most (8 threads a block and turn in fp32, 4 in bf16).  A grid of 2^32
// threads and more is not refused by the runtime: it leaves results unwritten.
constexpr int64_t kGateLaunch = (int64_t)1 << 28;

template <typename T>
static int gate_run(void (*kernel)(GateArgs), const GateArgs& all, int64_t N, hipStream_t s) {
    const int64_t per = ckpt_blocks(all.C), most = kGateLaunch / per;
    auto move = [](auto* p, int64_t n) { return p ? p + n : p; };
    for (int64_t n = 0; n < N; n += most) {
        GateArgs a = all;
        const int64_t at = n * a.C * 16;
        a.x = move((const T*)all.x, at);
        a.g = move((const T*)all.g, at);
        a.y = move((T*)all.y, at);
        a.codes_in = move(all.codes_in, at);
        a.exps_in = move(all.exps_in, n * per);
        a.codes = move(all.codes, at);
        a.exps = move(all.exps, n * per);
        a.blocks = (uint32_t)(std::min(N - n, most) * per);
        const int64_t grid = ceil_div(a.blocks, 256 / (128 / Chan<T>::kN) * kGateAhead);
        kernel<<<(unsigned)grid, 256, 0, s>>>(a);
    }
    return (int)hipGetLastError();
}
static bool gate_shape_ok(int64_t N, int C, int dtype) {
    return N >= 0 && C >= 1 && C <= kGateMaxC && (dtype == 0 || dtype == 1) &&
           N < ((int64_t)1 << 31) / ckpt_blocks(C);
}
}  // namespace bmhip

using namespace bmhip;

extern "C" int batteries_gate_activation(const void* x, void* y, uint8_t* codes, uint8_t* exps,
                                         int64_t N, int C, int dtype, hipStream_t stream) {
    if (!gate_shape_ok(N, C, dtype) || (N > 0 && (!x || !y)) || (codes && !exps)) return BM_ERR_ARG;
    if (!aligned_to({x, y}, 16) || !aligned_to({codes}, 8)) return BM_ERR_ARG;
    if (N == 0) return BM_OK;
    GateArgs a{};
    a.x = x; a.y = y; a.codes = codes; a.exps = exps; a.C = C;
    if (dtype == 0)
        return gate_run<float>(codes ? gate_fwd_kernel<float, true, true> : gate_fwd_kernel<float, true, false>,
                               a, N, stream);
    return gate_run<uint16_t>(
        codes ? gate_fwd_kernel<uint16_t, true, true> : gate_fwd_kernel<uint16_t, true, false>, a, N, stream);
}

extern "C" int batteries_gate_activation_backward(const void* x, const uint8_t* codes,
                                                  const uint8_t* exps, const void* g, void* gx,
                                                  int64_t N, int C, int dtype, hipStream_t stream) {
    if (!gate_shape_ok(N, C, dtype) || (N > 0 && (!g || !gx || (!x && (!codes || !exps)))))
        return BM_ERR_ARG;
    if (!aligned_to({x, g, gx}, 16) || !aligned_to({codes}, 8)) return BM_ERR_ARG;
    if (N == 0) return BM_OK;
    GateArgs a{};
    a.x = x; a.g = g; a.y = gx; a.codes_in = codes; a.exps_in = exps; a.C = C;
    if (dtype == 0)
        return gate_run<float>(x ? gate_bwd_kernel<float, false, true> : gate_bwd_kernel<float, true, true>, a,
                               N, stream);
    return gate_run<uint16_t>(
        x ? gate_bwd_kernel<uint16_t, false, true> : gate_bwd_kernel<uint16_t, true, true>, a, N, stream);
}

extern "C" int batteries_checkpoint_encode(const void* x, uint8_t* codes, uint8_t* exps, int64_t N,
                                           int C, int dtype, hipStream_t stream) {
    if (!gate_shape_ok(N, C, dtype) || (N > 0 && (!x || !codes || !exps))) return BM_ERR_ARG;
    if (!aligned_to({x}, 16) || !aligned_to({codes}, 8)) return BM_ERR_ARG;
    if (N == 0) return BM_OK;
    GateArgs a{};
    a.x = x; a.codes = codes; a.exps = exps; a.C = C;
    return dtype == 0 ? gate_run<float>(gate_fwd_kernel<float, false, true>, a, N, stream)
                      : gate_run<uint16_t>(gate_fwd_kernel<uint16_t, false, true>, a, N, stream);
}

extern "C" int batteries_checkpoint_decode(const uint8_t* codes, const uint8_t* exps, void* x, int64_t N,
                                           int C, int dtype, hipStream_t stream) {
    if (!gate_shape_ok(N, C, dtype) || (N > 0 && (!x || !codes || !exps))) return BM_ERR_ARG;
    if (!aligned_to({x}, 16) || !aligned_to({codes}, 8)) return BM_ERR_ARG;
    if (N == 0) return BM_OK;
    GateArgs a{};
    a.codes_in = codes; a.exps_in = exps; a.y = x; a.C = C;
    return dtype == 0 ? gate_run<float>(gate_bwd_kernel<float, true, false>, a, N, stream)
                      : gate_run<uint16_t>(gate_bwd_kernel<uint16_t, true, false>, a, N, stream);
}
