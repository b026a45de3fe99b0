// Normalisation of node features [N, C, 16] by degree, alone and fused with the end of a block
// (no reference counterpart).  Per row (atom) and degree l, components l^2 .. (l + 1)^2 - 1:
//
//   r_l(z) = (mean over channels and components of z^2 + eps)^-1/2
//   norm(z; w)[c, lm] = w[l, c] r_l(z) z[c, lm]
//   h = x + scale[c] sigmoid(gate[c, l]) norm(y; w_post)        (no gate: factor 1)
//   n = norm(h; w_pre)
//
// which commutes with rotations: the factors are the same for all components of a degree.
// Backward, with gh and gn the gradients of h and n, M_l = C (2 l + 1), f = scale sigmoid(gate),
// h formed again from x and y:
//
//   V[c, l] = sum_m gn h                     gw_pre[l, c] = sum over atoms of r_l(h) V
//   G = gh + r w_pre gn - h r^3 / M sum_c w_pre V          (gx = G)
//   Z[c, l] = sum_m G y                      gw_post[l, c] = sum over atoms of f r_l(y) Z
//   ggate = f (1 - sigmoid) w_post r_l(y) Z  gscale[c] = sum sigmoid w_post r_l(y) Z
//   gy = r f w_post G - y r^3 / M sum_c f w_post Z
//
// Memory bound: each array is read or written once (counted: 290 MB read forward, 546 MB backward
// at 20,011 x 100 in f32, the arrays' own size), a row lives in the registers of one wave (up to
// 64 channels; 2 to 16 waves share a wider row).  A quad of lanes holds a channel, a
// lane four of its components, so that every load and store is contiguous over the wave.  The
// first of the four and the other three are each of one degree, and lane q of a quad does the
// arithmetic per (channel, degree q): the quad's two partial sums per lane go to their degrees'
// lanes, and the factors back, by quad permutes.
#include "node_features.h"
#include "batmobile_hip.h"

namespace bmhip {

constexpr int kNormMaxC = 2048;

// Partial sums a (first component) and b (the other three) of the quad's lanes -> lane q: the
// sum over the components of degree q (0 | 1..3 | 4..8 | 9..15 of the 16).
__device__ __forceinline__ float to_degree(float a, float b, int q) {
    const float ab = a + b, fb = quad<0, 0, 2, 2>(b), fab = quad<0, 0, 1, 0>(ab);
    return q == 0 ? a : q == 1 ? fb : q == 2 ? fab + a : fb + ab;
}
// The factor of each lane's first and other components from the degrees' lanes.
__device__ __forceinline__ float first_of(float f) { return quad<0, 2, 2, 3>(f); }
__device__ __forceinline__ float others_of(float f) { return quad<1, 2, 3, 3>(f); }

__device__ __forceinline__ float dot4(float4 a, float4 b, int q) {
    return to_degree(a.x * b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, a.w * b.w)), q);
}

// Sum over the lanes of the same q, over the W waves of a row (every thread of the workgroup
// takes part); the result in every lane of that q.  sh: two buffers of 4 floats a wave, used in
// turn.
template <int W>
__device__ __forceinline__ float row_sum(float v, float* sh, int& turn) {
    v += dpp<0x124>(v);                        // row_ror:4 and :8 within 16 lanes
    v += dpp<0x128>(v);
    typedef unsigned v2u __attribute__((ext_vector_type(2)));
    v2u r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    if constexpr (W > 1) {
        float* s = sh + turn * 4 * 16;
        turn ^= 1;
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
        if (lane < 4) s[w * 4 + lane] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) v += s[(w / W * W + i) * 4 + (lane & 3)];
    }
    return v;
}

struct NormArgs {
    const void *x, *y, *gate, *gh, *gn;
    const float *scale, *w_post, *w_pre, *rs_in;
    void *out_h, *out_n, *gx, *gy, *ggate;
    float *rs, *part;                  // rs [N, 8]: 1/rms of y by degree, then of h
    int64_t n, row0;                   // rows; the launch's first
    int C;
    float eps;
};

// Rows per workgroup: 4 (W = 1) or 1.  BLOCK: h = x + f norm(y) first; else h = x.
//
// Measured: the block at 50,000 x 128 in bf16 164 us, 5.3 TB/s; at 20,011 x 100 in f32 with the
// rows' factors kept 100 us, 5.5 TB/s (a copy: 5.0 TB/s; part of the output stays in Infinity
// Cache); the norm alone at 1000 x 32 in f32 3.5 us, a launch.
template <typename T, int NV, int W, bool BLOCK, bool GATE, bool PRE>
__global__ __launch_bounds__(W == 1 ? 256 : 64 * W) void norm_fwd_kernel(NormArgs a) {
    __shared__ float sh[2 * 4 * 16];
    int turn = 0;
    const int64_t row =
        a.row0 + (W == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x);
    if (row >= a.n) return;
    const int t = W == 1 ? (threadIdx.x & 63) : threadIdx.x, q = t & 3;
    const int64_t at = row * (int64_t)a.C * 16;
    const float cnt = 1.0f / ((float)a.C * (float)(2 * q + 1));
    Raw4<T> x[NV], y[NV];
    float4 h[NV];
    float f[NV];
    // y, which the first sum waits for, before x
    if constexpr (BLOCK) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            y[i].zero();
            if (((i * 64 * W + t) >> 2) < a.C)
                y[i].load((const T*)a.y + at + (int64_t)(i * 64 * W + t) * 4);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int c = (i * 64 * W + t) >> 2;
        x[i].zero();
        f[i] = 0.0f;
        if (c < a.C) {
            x[i].load((const T*)a.x + at + (int64_t)(i * 64 * W + t) * 4);
            if constexpr (GATE)
                f[i] = norm_ld((const T*)a.gate + row * a.C * 4 + i * 64 * W + t);
        }
    }
    if constexpr (BLOCK) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) s += dot4(y[i].get(), y[i].get(), q);
        const float r = 1.0f / sqrtf(fmaf(row_sum<W>(s, sh, turn), cnt, a.eps));
        if (a.rs && t < 4) a.rs[row * 8 + t] = r;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = min((i * 64 * W + t) >> 2, a.C - 1);
            float w = a.scale[c] * a.w_post[q * a.C + c] * r;
            if constexpr (GATE) w *= sigmoid_on(sigmoid_pair(f[i]));
            const float fa = first_of(w), fb = others_of(w);
            const float4 yi = y[i].get(), xi = x[i].get();
            h[i] = make_float4(fmaf(fa, yi.x, xi.x), fmaf(fb, yi.y, xi.y), fmaf(fb, yi.z, xi.z),
                               fmaf(fb, yi.w, xi.w));
            if (((i * 64 * W + t) >> 2) < a.C)
                norm_st4((T*)a.out_h + at + (int64_t)(i * 64 * W + t) * 4, h[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) h[i] = x[i].get();
    }
    if constexpr (PRE) {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) s += dot4(h[i], h[i], q);
        const float r = 1.0f / sqrtf(fmaf(row_sum<W>(s, sh, turn), cnt, a.eps));
        if (a.rs && t < 4) a.rs[row * 8 + 4 + t] = r;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = (i * 64 * W + t) >> 2;
            const float w = a.w_pre[q * a.C + min(c, a.C - 1)] * r;
            const float fa = first_of(w), fb = others_of(w);
            if (c < a.C)
                norm_st4((T*)a.out_n + at + (int64_t)(i * 64 * W + t) * 4,
                         make_float4(fa * h[i].x, fb * h[i].y, fb * h[i].z, fb * h[i].w));
        }
    }
}

// Every workgroup takes rows in turn (4 / W at a time, W waves each) and keeps its share of the
// weights' gradients in registers: part [gridDim.x, 9 C] (pre [4][C], post [4][C], scale [C]),
// summed by norm_weights_kernel.
//
// Measured: 20,011 x 100 in f32 168 us, 5.0 TB/s; 50,000 x 128 in bf16 285 us; past 512 channels
// registers spill (6250 x 1024 in f32 809 us, 512 us for the same elements at 512 channels).
template <typename T, int NV, int W, bool BLOCK, bool GATE, bool PRE>
__global__ __launch_bounds__(W <= 4 ? 256 : 64 * W) void norm_bwd_kernel(NormArgs a) {
    constexpr int kRows = W <= 4 ? 4 / W : 1;
    __shared__ float sh[2 * 4 * 16];
    __shared__ float red[kRows > 1 ? 256 : 1];
    int turn = 0;
    const int group = threadIdx.x / (64 * W), t = threadIdx.x % (64 * W), q = t & 3;
    const float cnt = 1.0f / ((float)a.C * (float)(2 * q + 1));
    float aw_pre[NV], aw_post[NV], a_scale[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) aw_pre[i] = aw_post[i] = a_scale[i] = 0.0f;
    // the next row's loads are under way while this one's sums are formed; lanes past C read the
    // row's last channel and drop it
    struct Row {
        Raw4<T> gh[NV], x[NV], gn[NV], y[NV];
        float sg[NV], r_pre, r_post;
    };
    auto load = [&](Row& x, int64_t row0) {
        const int64_t row = min(row0 + group, a.n - 1);
        const int64_t at = row * (int64_t)a.C * 16;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int e = min(i * 64 * W + t, a.C * 4 - 4 + q);
            if constexpr (PRE) {
                x.x[i].load((const T*)a.x + at + e * 4);
                x.gn[i].load((const T*)a.gn + at + e * 4);
            }
            if (a.gh) x.gh[i].load((const T*)a.gh + at + e * 4);
            else x.gh[i].zero();
            if constexpr (BLOCK) {
                x.y[i].load((const T*)a.y + at + e * 4);
                if constexpr (GATE) x.sg[i] = norm_ld((const T*)a.gate + row * a.C * 4 + e);
            }
        }
        if constexpr (PRE) x.r_pre = a.rs_in[row * 8 + 4 + q];
        if constexpr (BLOCK) x.r_post = a.rs_in[row * 8 + q];
    };
    const int64_t step = (int64_t)gridDim.x * kRows;
    constexpr bool kAhead = W < 16;      // 16 waves have 128 registers each, too few for two rows
    Row next;
    if constexpr (kAhead) load(next, (int64_t)blockIdx.x * kRows);
    for (int64_t row0 = (int64_t)blockIdx.x * kRows; row0 < a.n; row0 += step) {
        const bool there = row0 + group < a.n;
        const int64_t row = there ? row0 + group : a.n - 1;
        const int64_t at = row * (int64_t)a.C * 16;
        if constexpr (!kAhead) load(next, row0);
        Row x = next;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (!(there && ((i * 64 * W + t) >> 2) < a.C)) {
                if constexpr (PRE) x.gn[i].zero();
                if constexpr (BLOCK) x.y[i].zero();
            }
        float sg[NV];                    // before the next row takes registers
        if constexpr (GATE) {
#pragma unroll
            for (int i = 0; i < NV; ++i) sg[i] = sigmoid_pair(x.sg[i]);
        }
        if (kAhead && row0 + step < a.n) load(next, row0 + step);
        float4 G[NV];
        float f[NV];
        if constexpr (BLOCK) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = min((i * 64 * W + t) >> 2, a.C - 1);
                f[i] = a.scale[c] * a.w_post[q * a.C + c];
                if constexpr (GATE) {
                    f[i] *= sigmoid_on(sg[i]);
                    asm volatile("" : "+v"(sg[i]));     // one register to the end, not two
                }
            }
        }
        if constexpr (PRE) {
            const float r = x.r_pre;
            float s = 0.0f, wp[NV];
            // h as the forward had it before rounding: gw_pre is fp32 whatever the features' type
            float4 h[NV];
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * 64 * W + t) >> 2;
                h[i] = x.x[i].get();
                if constexpr (BLOCK) {
                    const float fa = first_of(f[i] * x.r_post), fb = others_of(f[i] * x.r_post);
                    const float4 yi = x.y[i].get();
                    h[i] = make_float4(fmaf(fa, yi.x, h[i].x), fmaf(fb, yi.y, h[i].y),
                                       fmaf(fb, yi.z, h[i].z), fmaf(fb, yi.w, h[i].w));
                }
                wp[i] = a.w_pre[q * a.C + min(c, a.C - 1)];
                const float v = dot4(x.gn[i].get(), h[i], q);       // 0 past C
                aw_pre[i] = fmaf(r, v, aw_pre[i]);
                s = fmaf(wp[i], v, s);
            }
            const float k = -row_sum<W>(s, sh, turn) * cnt * r * r * r;
            const float ka = first_of(k), kb = others_of(k);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const float fa = first_of(wp[i] * r), fb = others_of(wp[i] * r);
                const float4 gni = x.gn[i].get(), ghi = x.gh[i].get();
                G[i] = make_float4(ghi.x + fmaf(fa, gni.x, ka * h[i].x),
                                   ghi.y + fmaf(fb, gni.y, kb * h[i].y),
                                   ghi.z + fmaf(fb, gni.z, kb * h[i].z),
                                   ghi.w + fmaf(fb, gni.w, kb * h[i].w));
            }
        } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) G[i] = x.gh[i].get();
        }
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (there && ((i * 64 * W + t) >> 2) < a.C)
                norm_st4((T*)a.gx + at + (int64_t)(i * 64 * W + t) * 4, G[i]);
        if constexpr (BLOCK) {
            const float r = x.r_post;
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const int c = (i * 64 * W + t) >> 2;
                const float sc = a.scale[min(c, a.C - 1)], w = a.w_post[q * a.C + min(c, a.C - 1)];
                const float z = dot4(G[i], x.y[i].get(), q), rz = r * z;    // 0 past C
                s = fmaf(f[i], z, s);
                const float on = GATE ? sigmoid_on(sg[i]) : 1.0f;
                aw_post[i] = fmaf(sc * on, rz, aw_post[i]);
                a_scale[i] = fmaf(on * w, rz, a_scale[i]);
                if constexpr (GATE)
                    if (there && c < a.C)
                        norm_st((T*)a.ggate + row * a.C * 4 + i * 64 * W + t,
                                f[i] * sigmoid_off(sg[i]) * rz);
            }
            const float k = -row_sum<W>(s, sh, turn) * cnt * r * r * r;
            const float ka = first_of(k), kb = others_of(k);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const float fa = first_of(f[i] * r), fb = others_of(f[i] * r);
                const float4 yi = x.y[i].get();
                if (there && ((i * 64 * W + t) >> 2) < a.C)
                    norm_st4((T*)a.gy + at + (int64_t)(i * 64 * W + t) * 4,
                             make_float4(fmaf(fa, G[i].x, ka * yi.x), fmaf(fb, G[i].y, kb * yi.y),
                                         fmaf(fb, G[i].z, kb * yi.z),
                                         fmaf(fb, G[i].w, kb * yi.w)));
            }
        }
    }
    float* part = a.part + (int64_t)blockIdx.x * 9 * a.C;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            float v = k == 0 ? aw_pre[i] : k == 1 ? aw_post[i] : a_scale[i];
            if (k == 0 && !PRE) continue;
            if (k > 0 && !BLOCK) continue;
            if (k == 2) v = v + quad<1, 0, 3, 2>(v), v = v + quad<2, 3, 0, 1>(v);
            if constexpr (kRows > 1) {
                __syncthreads();
                red[threadIdx.x] = v;
                __syncthreads();
                v = 0.0f;
#pragma unroll
                for (int r = 0; r < kRows; ++r) v += red[r * 64 * W + t];
                if (group != 0) continue;
            }
            const int c = (i * 64 * W + t) >> 2;
            if (c >= a.C) continue;
            if (k < 2) part[(k * 4 + q) * a.C + c] = v;
            else if (q == 0) part[8 * a.C + c] = v;
        }
    }
}

// Column sums of part [rows, 9 C] over the workgroups' rows: 16 columns a workgroup, 64 threads
// a column, thread k rows k, k + 64, ...; 5.4 us for 100 channels (3.7 MB of partial sums).
__global__ __launch_bounds__(1024) void norm_weights_kernel(const float* __restrict__ part,
                                                            int rows, int C, float* gw_pre,
                                                            float* gw_post, float* gscale) {
    __shared__ float sh[64][17];
    const int lane = threadIdx.x & 15, col = blockIdx.x * 16 + lane, k = threadIdx.x >> 4;
    const bool want = col < 9 * C && (col < 4 * C ? gw_pre != nullptr
                                                  : col < 8 * C ? gw_post != nullptr
                                                                : gscale != nullptr);
    float s = 0.0f;
    if (want) {
#pragma unroll 8
        for (int r = k; r < rows; r += 64) s += part[(int64_t)r * 9 * C + col];
    }
    sh[k][lane] = s;
    __syncthreads();
    for (int o = 32; o > 0; o >>= 1) {
        if (k < o) sh[k][lane] += sh[k + o][lane];
        __syncthreads();
    }
    if (k == 0 && want) {
        s = sh[0][lane];
        if (col < 4 * C) gw_pre[col] = s;
        else if (col < 8 * C) gw_post[col - 4 * C] = s;
        else gscale[col - 8 * C] = s;
    }
}

static int norm_bwd_blocks(int64_t n, int C) {
    const int rows = C <= 64 ? 4 : C <= 128 ? 2 : 1;
    return (int)std::min<int64_t>(ceil_div(n, rows), C <= 512 ? 1024 : 512);
}

template <typename T, int NV, int W, bool BLOCK, bool GATE, bool PRE>
static void norm_fwd_launch(const NormArgs& a, hipStream_t s) {
    constexpr int kRows = W == 1 ? 4 : 1, kThreads = W == 1 ? 256 : 64 * W;
    constexpr int64_t kMost = (int64_t)1 << 20;     // workgroups of a launch (threads < 2^32)
    NormArgs b = a;
    for (b.row0 = 0; b.row0 < a.n; b.row0 += kMost * kRows)
        norm_fwd_kernel<T, NV, W, BLOCK, GATE, PRE>
            <<<(unsigned)std::min(ceil_div(a.n - b.row0, kRows), kMost), kThreads, 0, s>>>(b);
}
template <typename T, int NV, int W, bool BLOCK, bool GATE, bool PRE>
static void norm_bwd_launch(const NormArgs& a, hipStream_t s) {
    norm_bwd_kernel<T, NV, W, BLOCK, GATE, PRE>
        <<<norm_bwd_blocks(a.n, a.C), W <= 4 ? 256 : 64 * W, 0, s>>>(a);
}

template <typename T, int NV, int W, bool BLOCK, bool GATE, bool PRE>
static void norm_launch(const NormArgs& a, bool bwd, hipStream_t s) {
    if (bwd) norm_bwd_launch<T, NV, W, BLOCK, GATE, PRE>(a, s);
    else norm_fwd_launch<T, NV, W, BLOCK, GATE, PRE>(a, s);
}

// Lanes of a row for its channels: four loads of each array a lane, and waves by the channels.
// Eight loads a lane with fewer waves, at 6.4 M channels in us (four loads): gated block forward
// bf16 128 channels 200 (162), 192: 284 (171), 512: 203 (169); f32 128 channels 327 (316); the
// gain is occupancy.  One and two loads with more waves: bf16 128 channels 188 and 162, 100
// channels (lanes idle) 233 and 193 (180); f32 within 6 %.  Past 1024 channels a workgroup has
// no more waves.
template <typename T, bool BLOCK, bool GATE, bool PRE>
static void norm_pick(const NormArgs& a, bool bwd, hipStream_t s) {
    if (a.C <= 16) norm_launch<T, 1, 1, BLOCK, GATE, PRE>(a, bwd, s);
    else if (a.C <= 32) norm_launch<T, 2, 1, BLOCK, GATE, PRE>(a, bwd, s);
    else if (a.C <= 64) norm_launch<T, 4, 1, BLOCK, GATE, PRE>(a, bwd, s);
    else if (a.C <= 128) norm_launch<T, 4, 2, BLOCK, GATE, PRE>(a, bwd, s);
    else if (a.C <= 256) norm_launch<T, 4, 4, BLOCK, GATE, PRE>(a, bwd, s);
    else if (a.C <= 512) norm_launch<T, 4, 8, BLOCK, GATE, PRE>(a, bwd, s);
    else if (a.C <= 1024) norm_launch<T, 4, 16, BLOCK, GATE, PRE>(a, bwd, s);
    else norm_launch<T, 8, 16, BLOCK, GATE, PRE>(a, bwd, s);
}

template <typename T>
static void norm_run(const NormArgs& a, bool block, bool pre, bool bwd, hipStream_t s) {
    if (!block) norm_pick<T, false, false, true>(a, bwd, s);
    else if (a.gate && pre) norm_pick<T, true, true, true>(a, bwd, s);
    else if (a.gate) norm_pick<T, true, true, false>(a, bwd, s);
    else if (pre) norm_pick<T, true, false, true>(a, bwd, s);
    else norm_pick<T, true, false, false>(a, bwd, s);
}

static bool norm_shape_ok(int64_t n, int C, int dtype) {
    return n >= 0 && C > 0 && C <= kNormMaxC && (dtype == 0 || dtype == 1) &&
           n < ((int64_t)1 << 31);
}
}  // namespace bmhip

using namespace bmhip;

extern "C" int batteries_gated_residual_norm(const void* x, const void* y, const void* gate,
                                             const float* scale, const float* w_post,
                                             const float* w_pre, void* h, void* n, float* rs,
                                             int64_t N, int C, float eps, int dtype,
                                             hipStream_t stream) {
    if (!norm_shape_ok(N, C, dtype) || (!y && !w_pre) || (y && (!scale || !w_post || !h)) ||
        (w_pre && !n) || (N > 0 && !x))
        return BM_ERR_ARG;
    if (!aligned_to({x, y, h, n}, dtype == 0 ? 16 : 8)) return BM_ERR_ARG;
    if (N == 0) return BM_OK;
    NormArgs a{};
    a.x = x; a.y = y; a.gate = gate; a.scale = scale; a.w_post = w_post; a.w_pre = w_pre;
    a.out_h = h; a.out_n = n; a.rs = rs; a.n = N; a.C = C; a.eps = eps;
    if (dtype == 0) norm_run<float>(a, y != nullptr, w_pre != nullptr, false, stream);
    else norm_run<uint16_t>(a, y != nullptr, w_pre != nullptr, false, stream);
    return (int)hipGetLastError();
}

extern "C" size_t batteries_gated_residual_norm_backward_workspace_bytes(int64_t N, int C) {
    if (!norm_shape_ok(N, C, 0)) return 0;
    return (size_t)norm_bwd_blocks(N, C) * 9 * (size_t)C * sizeof(float);
}

extern "C" int batteries_gated_residual_norm_backward(
    const void* gh, const void* gn, const void* x, const void* y, const void* gate,
    const float* scale, const float* w_post, const float* w_pre, const float* rs, void* gx,
    void* gy, void* ggate, float* gscale, float* gw_post, float* gw_pre, int64_t N, int C,
    int dtype, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    if (!norm_shape_ok(N, C, dtype) || (!y && !w_pre) || !gx ||
        (y && (!scale || !w_post || !gy || !gscale || !gw_post)) || (gate && !ggate) ||
        (w_pre && (!gn || !x || !gw_pre)) || (!w_pre && !gh) ||
        (N > 0 && !rs))
        return BM_ERR_ARG;
    if (!aligned_to({gh, gn, x, y, gx, gy}, dtype == 0 ? 16 : 8)) return BM_ERR_ARG;
    const size_t need = batteries_gated_residual_norm_backward_workspace_bytes(N, C);
    if (workspace_bytes < need || (need && !workspace)) return BM_ERR_WORKSPACE;
    NormArgs a{};
    a.gh = gh; a.gn = gn; a.x = x; a.y = y; a.gate = gate; a.scale = scale; a.w_post = w_post;
    a.w_pre = w_pre; a.rs_in = rs; a.gx = gx; a.gy = gy; a.ggate = ggate;
    a.part = (float*)workspace; a.n = N; a.C = C;
    if (N > 0) {
        if (dtype == 0) norm_run<float>(a, y != nullptr, w_pre != nullptr, true, stream);
        else norm_run<uint16_t>(a, y != nullptr, w_pre != nullptr, true, stream);
    }
    norm_weights_kernel<<<(unsigned)ceil_div(9 * (int64_t)C, 16), 1024, 0, stream>>>(
        a.part, N > 0 ? norm_bwd_blocks(N, C) : 0, C, w_pre ? gw_pre : nullptr,
        y ? gw_post : nullptr, y ? gscale : nullptr);
    return (int)hipGetLastError();
}
