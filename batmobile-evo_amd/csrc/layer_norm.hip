// Layer norm of rows (no reference counterpart): x [rows, D], elements `step` apart,
//
//   m = mean x,  r = (mean (x - m)^2 + eps)^-1/2,  xh = (x - m) r,  y = xh w + b
//   gx = r (u - mean u - xh mean(u xh)),  u = g w;   gw = sum over rows of g xh,  gb = sum g
//
// Memory bound: a row is read once each way into the registers of its lanes; the variance is that of
// the differences from the mean, and the backward forms m and r again from the row, which costs
// lane sums but no memory.  Sums are fp32.  A row of few elements takes a part of a wave, a long one up
// to 16 waves.
//
// Measured, us (the bytes at 5 TB/s): 560,308 x 64 in bf16 forward 28 (29), backward 43 (43) and 4 for the
// weights; 50,000 x 1000 in fp32 78 (80) and 120 (120); 300,000 x 37 in fp32 17 (18) and 36 (27).  Invariants
// that lie 16 apart cost their lines: 20,011 x 100 in fp32 21 and 24, 6 TB/s of whole lines.
#include "sums.h"
#include "batmobile_hip.h"

namespace bmhip {

constexpr int kLnMaxD = 8192;

struct LnArgs {
    const void *x, *g;
    const float *w, *b;
    void *y, *gx;
    float* part;
    int64_t rows, row_stride, step;
    int D;
    float eps, inv;                        // inv: 1 / D
};

// 16 bytes at any address that an element may have (the hardware takes unaligned vectors)
struct __attribute__((packed, aligned(2))) Ln16 {
    uint32_t v[4];
};

// VEC elements in 16 bytes (or one element) as fp32
template <typename T, int VEC>
struct LnVec {
    float v[VEC];
    __device__ __forceinline__ void load(const T* p) {
        if constexpr (VEC == 1) {
            v[0] = norm_ld(p);
        } else {
            const Ln16 t = *reinterpret_cast<const Ln16*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (VEC == 4) v[i] = __uint_as_float(t.v[i]);
                else v[2 * i] = bf16_lo(t.v[i]), v[2 * i + 1] = bf16_hi(t.v[i]);
            }
        }
    }
    __device__ __forceinline__ void store(T* p) const {
        if constexpr (VEC == 1) {
            norm_st(p, v[0]);
        } else {
            Ln16 t;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (VEC == 4) t.v[i] = __float_as_uint(v[i]);
                else t.v[i] = bf16_pack(v[2 * i], v[2 * i + 1]);
            }
            *reinterpret_cast<Ln16*>(p) = t;
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = 0.0f;
    }
};

// Sum over a row: LPR lanes, or W whole waves (every thread of the workgroup takes part)
template <int LPR, int W>
__device__ __forceinline__ float ln_sum(float v, float* sh, int& turn) {
    v = lanes_sum<LPR>(v);
    if constexpr (W > 1) {
        float* s = sh + turn * 16;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) v += s[i];
    }
    return v;
}

// Where a lane's vector i of a row lies.  The last one of a row that is no whole number of vectors
// begins earlier (TAIL), so that it ends with the row: its first `skip` elements are another lane's, are worked
// out twice, and have no part in the sums.
template <int VEC, bool TAIL>
struct LnAt {
    int c, skip;
    bool there;
    __device__ __forceinline__ LnAt(int unit, int D) {
        const int first = unit * VEC;
        there = first < D;
        c = TAIL ? min(first, D - VEC) : first;
        skip = TAIL ? first - c : 0;
    }
    __device__ __forceinline__ bool counts(int j) const { return there && (!TAIL || j >= skip); }
};

// Takes the mean off a lane's part of a row and returns r.  The rounding of the mean, which is large next
// to the differences of a row far from 0, shows in the differences' own mean: that is taken off as well.
template <int LPR, int W, bool TAIL, typename T, int VEC, int NV>
__device__ __forceinline__ float ln_center(const LnArgs& a, int t, LnVec<T, VEC> (&x)[NV], float* sh,
                                           int& turn) {
    constexpr int kLanes = W == 1 ? LPR : 64 * W;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const LnAt<VEC, TAIL> at(i * kLanes + t, a.D);
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += !TAIL || at.counts(j) ? x[i].v[j] : 0.0f;
    }
    const float m = ln_sum<LPR, W>(s, sh, turn) * a.inv;
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const LnAt<VEC, TAIL> at(i * kLanes + t, a.D);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            x[i].v[j] -= m;
            const float d = at.counts(j) ? x[i].v[j] : 0.0f;
            s1 += d;
            s2 = fmaf(d, d, s2);
        }
    }
    s1 = ln_sum<LPR, W>(s1, sh, turn) * a.inv;
    s2 = ln_sum<LPR, W>(s2, sh, turn) * a.inv;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[i].v[j] -= s1;
    return 1.0f / sqrtf(fmaxf(fmaf(-s1, s1, s2), 0.0f) + a.eps);
}

template <int W>
constexpr int ln_threads() { return W == 1 ? 256 : 64 * W; }

// Workgroups take rows in turn, ROWS at a time for a group of lanes, whose loads are all asked for first;
// the weights stay in registers.
template <typename T, int VEC, int NV, int LPR, int W, int ROWS, bool TAIL>
__global__ __launch_bounds__(ln_threads<W>()) void ln_fwd_kernel(LnArgs a) {
    __shared__ float sh[2 * 16];
    int turn = 0;
    constexpr int kGroups = W == 1 ? 4 * (64 / LPR) : 1, kLanes = W == 1 ? LPR : 64 * W;
    const int t = W == 1 ? threadIdx.x % LPR : threadIdx.x;
    const int group = W == 1 ? threadIdx.x / LPR : 0;
    float w[NV][VEC], b[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const LnAt<VEC, TAIL> at(i * kLanes + t, a.D);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
            w[i][j] = at.there ? a.w[at.c + j] : 0.0f;
            b[i][j] = at.there && a.b ? a.b[at.c + j] : 0.0f;
        }
    }
    for (int64_t row0 = (int64_t)blockIdx.x * kGroups * ROWS + group; row0 - group < a.rows;
         row0 += (int64_t)gridDim.x * kGroups * ROWS) {
        LnVec<T, VEC> x[ROWS][NV];
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            const int64_t row = min(row0 + k * kGroups, a.rows - 1);
            const T* p = (const T*)a.x + row * a.row_stride;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const LnAt<VEC, TAIL> at(i * kLanes + t, a.D);
                x[k][i].zero();
                if (at.there) x[k][i].load(p + (VEC == 1 ? at.c * a.step : at.c));
            }
        }
#pragma unroll
        for (int k = 0; k < ROWS; ++k) {
            const int64_t row = row0 + k * kGroups;
            const float r = ln_center<LPR, W, TAIL>(a, t, x[k], sh, turn);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const LnAt<VEC, TAIL> at(i * kLanes + t, a.D);
#pragma unroll
                for (int j = 0; j < VEC; ++j) x[k][i].v[j] = fmaf(x[k][i].v[j] * r, w[i][j], b[i][j]);
                if (at.there && row < a.rows) x[k][i].store((T*)a.y + row * a.D + at.c);
            }
        }
    }
}

// Workgroups take rows in turn; a lane keeps its columns' sums of g xh and g in registers, which are
// joined over the workgroup's rows at the end: part [gridDim.x, 2, D].
template <typename T, int VEC, int NV, int LPR, int W, bool TAIL>
__global__ __launch_bounds__(ln_threads<W>()) void ln_bwd_kernel(LnArgs a) {
    __shared__ float sh[2 * 16];
    constexpr int kCols = NV * LPR * VEC;
    __shared__ float red[W == 1 ? 4 * kCols : 1];
    int turn = 0;
    constexpr int kGroups = W == 1 ? 4 * (64 / LPR) : 1, kLanes = W == 1 ? LPR : 64 * W;
    const int t = W == 1 ? threadIdx.x % LPR : threadIdx.x;
    const int group = W == 1 ? threadIdx.x / LPR : 0;
    float gw[NV][VEC], gb[NV][VEC];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VEC; ++j) gw[i][j] = gb[i][j] = 0.0f;
    for (int64_t row0 = (int64_t)blockIdx.x * kGroups; row0 < a.rows;
         row0 += (int64_t)gridDim.x * kGroups) {
        const bool there = row0 + group < a.rows;
        const int64_t row = there ? row0 + group : a.rows - 1;
        LnVec<T, VEC> x[NV], g[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const LnAt<VEC, TAIL> at(i * kLanes + t, a.D);
            x[i].zero();
            g[i].zero();
            if (at.there && there) {
                x[i].load((const T*)a.x + row * a.row_stride + (VEC == 1 ? at.c * a.step : at.c));
                g[i].load((const T*)a.g + row * a.D + at.c);
            }
        }
        const float r = ln_center<LPR, W, TAIL>(a, t, x, sh, turn);
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const LnAt<VEC, TAIL> at(i * kLanes + t, a.D);
            if (at.there && there) {                       // (without eps r of no row is infinite)
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float xh = x[i].v[j] * r;
                    gw[i][j] = fmaf(g[i].v[j], xh, gw[i][j]);
                    gb[i][j] += g[i].v[j];
                    x[i].v[j] = xh;
                    g[i].v[j] *= a.w[at.c + j];
                    const float u = at.counts(j) ? g[i].v[j] : 0.0f;
                    s1 += u;
                    s2 = fmaf(u, xh, s2);
                }
            }
        }
        s1 = ln_sum<LPR, W>(s1, sh, turn) * a.inv;
        s2 = ln_sum<LPR, W>(s2, sh, turn) * a.inv;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const LnAt<VEC, TAIL> at(i * kLanes + t, a.D);
            if (at.there && there) {
#pragma unroll
                for (int j = 0; j < VEC; ++j)
                    g[i].v[j] = r * (g[i].v[j] - s1 - x[i].v[j] * s2);
                g[i].store((T*)a.gx + row * a.D + at.c);
            }
        }
    }
    float* part = a.part + (int64_t)blockIdx.x * 2 * a.D;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        if constexpr (W == 1) __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const LnAt<VEC, TAIL> at(i * kLanes + t, a.D);
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
                float v = k ? gb[i][j] : gw[i][j];
                if constexpr (W == 1) {
#pragma unroll
                    for (int o = LPR; o < 64; o <<= 1) v += __shfl_xor(v, o);
                    if ((threadIdx.x & 63) < LPR && at.counts(j))
                        red[(threadIdx.x >> 6) * kCols + at.c + j] = v;
                } else if (at.counts(j)) {
                    part[k * a.D + at.c + j] = v;
                }
            }
        }
        if constexpr (W == 1) {
            __syncthreads();
            for (int c = threadIdx.x; c < a.D; c += 256)
                part[k * a.D + c] = (red[c] + red[kCols + c]) + (red[2 * kCols + c] + red[3 * kCols + c]);
        }
    }
}

__global__ __launch_bounds__(1024) void ln_weights_kernel(const float* part, int rows, int D,
                                                          float* gw, float* gb) {
    const int col = blockIdx.x * 16 + (threadIdx.x & 15);
    const bool there = col < (gb ? 2 * D : D);
    const float s =
        column_sum(there ? rows : 0, [&](int r) { return part[(int64_t)r * 2 * D + col]; });
    if (threadIdx.x < 16 && there) {
        if (col < D) gw[col] = s;
        else gb[col - D] = s;
    }
}

// Workgroups of the backward: enough to fill the card, and few enough that the partial sums stay a
// small part of the data
static int ln_parts(int64_t rows, int D) {
    const int64_t groups = D <= 64 ? 8 : D <= 256 ? 4 : 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(ceil_div(rows, 8 * groups), 1024));
}

template <typename T, int VEC, int NV, int LPR, int W, bool TAIL>
static void ln_launch(const LnArgs& a, bool bwd, hipStream_t s) {
    constexpr int kGroups = W == 1 ? 4 * (64 / LPR) : 1;
    constexpr int kRows = W > 1 ? 1 : NV * VEC <= 8 ? 4 : NV * VEC <= 16 ? 2 : 1;
    if (bwd) {
        ln_bwd_kernel<T, VEC, NV, LPR, W, TAIL><<<ln_parts(a.rows, a.D), ln_threads<W>(), 0, s>>>(a);
        return;
    }
    const int64_t most = W == 16 ? 512 : 2048;      // workgroups: what the card holds at once
    ln_fwd_kernel<T, VEC, NV, LPR, W, kRows, TAIL>
        <<<(unsigned)std::min(ceil_div(a.rows, kGroups * kRows), most), ln_threads<W>(), 0, s>>>(a);
}

template <typename T, int VEC, bool TAIL>
static void ln_pick(const LnArgs& a, bool bwd, hipStream_t s) {
    const int units = (a.D + VEC - 1) / VEC;
    if (units <= 8) ln_launch<T, VEC, 1, 8, 1, TAIL>(a, bwd, s);
    else if (units <= 16) ln_launch<T, VEC, 1, 16, 1, TAIL>(a, bwd, s);
    else if (units <= 32) ln_launch<T, VEC, 1, 32, 1, TAIL>(a, bwd, s);
    else if (units <= 64) ln_launch<T, VEC, 1, 64, 1, TAIL>(a, bwd, s);
    else if (units <= 128) ln_launch<T, VEC, 2, 64, 1, TAIL>(a, bwd, s);
    // 129 to 256 vectors: four waves a row in bf16 (20,000 x 2048 forward 37 us against 81 with four vectors a
    // lane and one wave, backward 57 and 65), one in fp32 (50,000 x 1000 forward 78 against 81, backward
    // 120 and 142)
    else if (units <= 256) ln_launch<T, VEC, VEC == 8 ? 1 : 4, 64, VEC == 8 ? 4 : 1, TAIL>(a, bwd, s);
    else if (units <= 512) ln_launch<T, VEC, 2, 64, 4, TAIL>(a, bwd, s);
    else if (units <= 1024) ln_launch<T, VEC, 4, 64, 4, TAIL>(a, bwd, s);
    else if constexpr (kLnMaxD / VEC > 1024) {
        if (units <= 2048) ln_launch<T, VEC, 2, 64, 16, TAIL>(a, bwd, s);
        else if constexpr (kLnMaxD / VEC > 2048) ln_launch<T, VEC, 8, 64, 16, TAIL>(a, bwd, s);
    }
}

// 16 bytes a lane where a row's elements follow each other, at any alignment; else one element
template <typename T>
static void ln_run(const LnArgs& a, bool bwd, hipStream_t s) {
    constexpr int VEC = 16 / sizeof(T);
    if (a.step != 1 || a.D < VEC) ln_pick<T, 1, false>(a, bwd, s);
    else if (a.D % VEC == 0) ln_pick<T, VEC, false>(a, bwd, s);
    else ln_pick<T, VEC, true>(a, bwd, s);
}

static bool ln_shape_ok(int64_t rows, int D, int dtype) {
    return rows >= 0 && rows < ((int64_t)1 << 38) && D >= 1 && D <= kLnMaxD &&
           (dtype == 0 || dtype == 1);
}
}  // namespace bmhip

using namespace bmhip;

extern "C" int batteries_layer_norm(const void* x, const float* weight, const float* bias, void* y,
                                    int64_t rows, int D, int64_t row_stride, int64_t step, float eps,
                                    int dtype, hipStream_t stream) {
    if (!ln_shape_ok(rows, D, dtype) || !weight || (rows > 0 && (!x || !y)) || !(eps >= 0.0f))
        return BM_ERR_ARG;
    if (!aligned_to({x, y}, dtype == 0 ? 4 : 2)) return BM_ERR_ARG;
    if (rows == 0) return BM_OK;
    LnArgs a{};
    a.x = x; a.w = weight; a.b = bias; a.y = y; a.rows = rows; a.row_stride = row_stride;
    a.step = step; a.D = D; a.eps = eps; a.inv = 1.0f / (float)D;
    if (dtype == 0) ln_run<float>(a, false, stream);
    else ln_run<uint16_t>(a, false, stream);
    return (int)hipGetLastError();
}

extern "C" size_t batteries_layer_norm_backward_workspace_bytes(int64_t rows, int D) {
    if (!ln_shape_ok(rows, D, 0)) return 0;
    return (size_t)ln_parts(rows, D) * 2 * D * sizeof(float);
}

extern "C" int batteries_layer_norm_backward(const void* x, const float* weight, const void* g,
                                             void* gx, float* gweight, float* gbias, int64_t rows,
                                             int D, int64_t row_stride, int64_t step, float eps,
                                             int dtype, void* workspace, size_t workspace_bytes,
                                             hipStream_t stream) {
    if (!ln_shape_ok(rows, D, dtype) || !weight || !gweight || (rows > 0 && (!x || !g || !gx)) ||
        !(eps >= 0.0f))
        return BM_ERR_ARG;
    if (!aligned_to({x, g, gx}, dtype == 0 ? 4 : 2)) return BM_ERR_ARG;
    if (workspace_bytes < batteries_layer_norm_backward_workspace_bytes(rows, D) || !workspace)
        return BM_ERR_WORKSPACE;
    LnArgs a{};
    a.x = x; a.w = weight; a.g = g; a.gx = gx; a.part = (float*)workspace; a.rows = rows;
    a.row_stride = row_stride; a.step = step; a.D = D; a.eps = eps; a.inv = 1.0f / (float)D;
    if (rows > 0) {
        if (dtype == 0) ln_run<float>(a, true, stream);
        else ln_run<uint16_t>(a, true, stream);
    }
    ln_weights_kernel<<<(unsigned)ceil_div(gbias ? 2 * D : D, 16), 1024, 0, stream>>>(
        a.part, rows > 0 ? ln_parts(rows, D) : 0, D, gweight, gbias);
    return (int)hipGetLastError();
}
