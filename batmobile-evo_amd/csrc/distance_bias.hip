// A learned bias of attention by distance (no reference counterpart).  Edge e of length r, head h:
//
//   k(r) = number of boundaries <= r,   bias[e, h] = table[k(r_e), h] + log max(0, 1 - (r_e / c)^2)
//
// (the second term only with a cutoff c; an edge from the cutoff on has -inf, which attention leaves
// out).  Gradients, g that of the bias:
//
//   gtable[k, h] = sum over edges of bucket k of g[e, h]
//   glengths[e]  = -2 r / ((c - r) (c + r)) sum_h g[e, h]        (0 from the cutoff on)
//
// (c - r) (c + r) in place of c^2 - r^2: next to the cutoff the difference is exact.  A length that is
// not a number gives a bias that is none.
#include <type_traits>

#include "sums.h"
#include "batmobile_hip.h"

namespace bmhip {

constexpr int kBiasEdges = 256;             // edges of a workgroup at a time
constexpr int kBiasMaxBuckets = 4096, kBiasMaxHeads = 1024;
constexpr int kBiasTableLds = 8192;         // floats of the table that go to LDS
constexpr int kBiasRange = 64;              // buckets of a wave in the backward
constexpr int kBiasParts = 512;             // most partial tables
constexpr int64_t kBiasPartFloats = 1 << 22;

struct BiasArgs {
    const float *lengths, *boundaries, *table, *g;
    float *out, *glengths, *part;
    const uint16_t* bucket;
    uint16_t* out_bucket;
    int64_t edges;
    int H, B;
    float cutoff, inv;                      // inv: 1 / cutoff, 0 without one
};

// A workgroup finds the buckets of 256 edges by bisection in LDS, a lane an edge, then writes their
// 256 H values as one contiguous piece.  Bound by the writes: 1.4 M edges x 8 heads 14 us, 3.8 TB/s.
template <bool TABLE_LDS, bool VEC>
__global__ __launch_bounds__(256) void bias_fwd_kernel(BiasArgs a) {
    extern __shared__ __attribute__((aligned(16))) float sh[];
    float* bound = sh;                                  // [B - 1]
    float* table = bound + (a.B + 3) / 4 * 4;           // [B * H]
    __shared__ int sk[kBiasEdges];
    __shared__ float se[kBiasEdges];
    const int t = threadIdx.x, H = a.H;
    for (int i = t; i < a.B - 1; i += 256) bound[i] = a.boundaries[i];
    if constexpr (TABLE_LDS)
        for (int i = t; i < a.B * H; i += 256) table[i] = a.table[i];
    __syncthreads();
    const float* tab = TABLE_LDS ? table : a.table;
    for (int64_t e0 = (int64_t)blockIdx.x * kBiasEdges; e0 < a.edges;
         e0 += (int64_t)gridDim.x * kBiasEdges) {
        const int n = (int)min((int64_t)kBiasEdges, a.edges - e0);
        if (t < n) {
            const float r = a.lengths[e0 + t];
            int lo = 0, hi = a.B - 1;                   // bound[lo - 1] <= r < bound[hi]
            while (lo < hi) {
                const int m = (lo + hi) >> 1;
                if (bound[m] <= r) lo = m + 1; else hi = m;
            }
            if (a.out_bucket) a.out_bucket[e0 + t] = (uint16_t)lo;
            float env = r != r ? r : 0.0f;
            if (a.inv > 0.0f && r == r)
                env = logf(fmaxf(((a.cutoff - r) * a.inv) * ((a.cutoff + r) * a.inv), 0.0f));
            sk[t] = lo * H;
            se[t] = env;
        }
        __syncthreads();
        constexpr int V = VEC ? 4 : 1;
        const int per = H / V, total = n * per;
        int e = t / per, u = t - e * per;               // 256 units on: (de, du) further
        const int de = 256 / per, du = 256 - de * per;
        float* out = a.out + e0 * H;
        for (int i = t; i < total; i += 256) {
            const float env = se[e];
            const float* p = tab + sk[e] + u * V;
            if constexpr (VEC) {
                const float4 v = *reinterpret_cast<const float4*>(p);
                reinterpret_cast<float4*>(out)[i] =
                    make_float4(v.x + env, v.y + env, v.z + env, v.w + env);
            } else {
                out[i] = *p + env;
            }
            e += de;
            u += du;
            if (u >= per) u -= per, ++e;
        }
        __syncthreads();
    }
}

// Table gradient.  A wave holds 64 columns of sums in LDS for each of its (at most 64) buckets; lane
// (slot s, head h) adds the values of its edges to its own column alone, so no two lanes meet and the order
// is the edges'.  It reads, adds and writes: the LDS's own addition takes longer (1.4 M edges x 8
// heads in 64 buckets 66 us, so 18).  More than 64 buckets: the waves of a workgroup take ranges of 64 and
// read the same edges, of which each adds a part (256 buckets 40 us); more than 256: gridDim.y ranges of
// 256.  The columns' sums go to part [gridDim.x, B, H].  Heads past 64: gridDim.z.
template <bool RANGES>
__global__ __launch_bounds__(256) void bias_bwd_kernel(BiasArgs a, int range_waves) {
    extern __shared__ __attribute__((aligned(16))) float sh[];
    const int t = threadIdx.x, lane = t & 63, w = __builtin_amdgcn_readfirstlane(t >> 6);
    const int h0 = blockIdx.z * 64, H = min(64, a.H - h0), slots = 64 / H;
    const int range = w % range_waves, sub = w / range_waves, subs = 4 / range_waves;
    const int b0 = (blockIdx.y * range_waves + range) * kBiasRange, per = min(a.B, kBiasRange);
    float* mine = sh + w * per * 64;
    for (int i = lane; i < per * 64; i += 64) mine[i] = 0.0f;
    const int s = lane / H, h = lane - s * H;
    const int64_t share = (a.edges + gridDim.x - 1) / gridDim.x;
    const int64_t first = blockIdx.x * share, last = min(a.edges, first + share);
    const int step = slots * subs, from = sub * slots + s;
    // steps whose loads are under way, and steps that read, add and write together
    constexpr int kAhead = RANGES ? 16 : 8, kTogether = RANGES ? 2 : 1;
    auto batch = [&](int64_t e0, auto whole) {             // kAhead steps from edge e0 on
        const float* g = a.g + e0 * a.H + h0;
        const uint16_t* bucket = a.bucket + e0;
        const int left = (int)min(last - e0, (int64_t)1 << 20);
        float v[kAhead];
        int k[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            int e = from + i * step;
            if (!decltype(whole)::value) e = min(e, left - 1);
            k[i] = bucket[(uint32_t)e];
            v[i] = g[(uint32_t)(e * a.H + h)];
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            // an edge of another range, or past the last, adds 0 to some bucket
            bool there = true;
            if (RANGES) k[i] -= b0, there = (unsigned)k[i] < (unsigned)per;
            else k[i] = min(k[i], per - 1);                // (no array of buckets leads out of the LDS)
            if (!decltype(whole)::value) there = there && from + i * step < left;
            if (RANGES || !decltype(whole)::value) {
                k[i] = there ? k[i] : 0;
                v[i] = there ? v[i] : 0.0f;
            }
            k[i] = k[i] * 64 + lane;
        }
#pragma unroll
        for (int i0 = 0; i0 < kAhead; i0 += kTogether) {
            float sum[kTogether];
#pragma unroll
            for (int i = 0; i < kTogether; ++i) sum[i] = mine[k[i0 + i]];
#pragma unroll
            for (int i = 0; i < kTogether; ++i) {
                // a bucket that came before in the group goes on from there
#pragma unroll
                for (int j = 0; j < i; ++j) sum[i] = k[i0 + j] == k[i0 + i] ? sum[j] : sum[i];
                sum[i] += v[i0 + i];
            }
#pragma unroll
            for (int i = 0; i < kTogether; ++i) mine[k[i0 + i]] = sum[i];
        }
    };
    if (s < slots) {
        int64_t e = first;
        for (; e + kAhead * step <= last; e += kAhead * step) batch(e, std::true_type{});
        if (e < last) batch(e, std::false_type{});
    }
    __syncthreads();
    for (int i = t; i < range_waves * per * H; i += 256) {
        const int r = i / (per * H), j = i - r * per * H, b = j / H, hh = j - b * H;
        const int bucket = (blockIdx.y * range_waves + r) * kBiasRange + b;
        if (bucket >= a.B) continue;
        float sum = 0.0f;
        for (int u = 0; u < subs; ++u)
            for (int k = 0; k < slots; ++k)
                sum += sh[((u * range_waves + r) * per + b) * 64 + k * H + hh];
        a.part[((int64_t)blockIdx.x * a.B + bucket) * a.H + h0 + hh] = sum;
    }
}

__global__ __launch_bounds__(1024) void bias_table_kernel(const float* part, int rows, int64_t cols,
                                                          float* out) {
    const int64_t col = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15);
    const float s = column_sum(col < cols ? rows : 0, [&](int r) { return part[r * cols + col]; });
    if (threadIdx.x < 16 && col < cols) out[col] = s;
}

// LANES lanes an edge
template <bool VEC, int LANES>
__global__ __launch_bounds__(256) void bias_lengths_kernel(BiasArgs a) {
    const int64_t e = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
    if (e >= a.edges) return;
    const int lane = threadIdx.x % LANES;
    const float r = a.lengths[e];
    float s = 0.0f;
    if constexpr (VEC) {
        const float4* p = reinterpret_cast<const float4*>(a.g + e * a.H);
        for (int i = lane; i < a.H / 4; i += LANES) {
            const float4 v = p[i];
            s += (v.x + v.y) + (v.z + v.w);
        }
    } else {
        for (int i = lane; i < a.H; i += LANES) s += a.g[e * a.H + i];
    }
    if constexpr (LANES > 1) s = lanes_sum<LANES>(s);
    const bool in = fabsf(r) < a.cutoff;
    if (lane == 0)
        a.glengths[e] = in ? s * (-2.0f * r / (a.cutoff - r) / (a.cutoff + r)) : r != r ? r : 0.0f;
}

template <bool VEC, int LANES>
static void bias_lengths_launch(const BiasArgs& a, hipStream_t s) {
    constexpr int64_t kEdges = ((int64_t)1 << 22) * (256 / LANES);     // of a launch
    for (int64_t e = 0; e < a.edges; e += kEdges) {
        BiasArgs b = a;
        b.lengths = a.lengths + e;
        b.g = a.g + e * a.H;
        b.glengths = a.glengths + e;
        b.edges = std::min(a.edges - e, kEdges);
        bias_lengths_kernel<VEC, LANES><<<(unsigned)ceil_div(b.edges, 256 / LANES), 256, 0, s>>>(b);
    }
}
// One or two loads a lane (500,000 edges of 64 heads with a lane an edge: 97 us, with
// 16 lanes 22)
template <bool VEC>
static void bias_lengths_run(const BiasArgs& a, hipStream_t s) {
    const int loads = VEC ? a.H / 4 : a.H;
    if (loads <= 2) bias_lengths_launch<VEC, 1>(a, s);
    else if (loads <= 8) bias_lengths_launch<VEC, 4>(a, s);
    else bias_lengths_launch<VEC, 16>(a, s);
}

// A cutoff whose inverse, and whose products with a length, stay in fp32's range; 0: none
static bool bias_cutoff_ok(float c) { return c == 0.0f || (c >= 1e-30f && c <= 1e30f); }
static bool bias_shape_ok(int64_t E, int H, int B) {
    return E >= 0 && E < ((int64_t)1 << 38) && H >= 1 && H <= kBiasMaxHeads && B >= 1 &&
           B <= kBiasMaxBuckets;
}
static int bias_range_waves(int B) {
    const int r = (B + kBiasRange - 1) / kBiasRange;
    return r >= 3 ? 4 : r;
}
// Workgroups of the edges: 16 steps of a wave at least, 16 MB of partial tables at most
static int bias_parts(int64_t E, int H, int B) {
    const int slots = 64 / std::min(H, 64), subs = 4 / bias_range_waves(B);
    const int64_t most = std::min<int64_t>(
        kBiasParts, std::max<int64_t>(1, kBiasPartFloats / ((int64_t)B * H)));
    return (int)std::min(most, std::max<int64_t>(1, ceil_div(E, 16 * slots * subs)));
}
}  // namespace bmhip

using namespace bmhip;

extern "C" int batteries_distance_bias(const float* lengths, const float* boundaries,
                                       const float* table, float* bias, uint16_t* buckets,
                                       int64_t E, int H, int B, float cutoff, hipStream_t stream) {
    if (!bias_shape_ok(E, H, B) || !bias_cutoff_ok(cutoff) ||
        (B > 1 && !boundaries) || !table || (E > 0 && (!lengths || !bias)))
        return BM_ERR_ARG;
    if (E == 0) return BM_OK;
    BiasArgs a{};
    a.lengths = lengths; a.boundaries = boundaries; a.table = table; a.out = bias;
    a.out_bucket = buckets; a.edges = E; a.H = H; a.B = B;
    a.cutoff = cutoff; a.inv = cutoff > 0.0f ? 1.0f / cutoff : 0.0f;
    const bool lds = (int64_t)B * H <= kBiasTableLds;
    const bool vec = H % 4 == 0 && aligned_to({bias}, 16) && (lds || aligned_to({table}, 16));
    const size_t bytes = ((size_t)(B + 3) / 4 * 4 + (lds ? (size_t)B * H : 0)) * 4;
    const unsigned grid = (unsigned)std::min<int64_t>(ceil_div(E, kBiasEdges), 2048);
    if (lds && vec) bias_fwd_kernel<true, true><<<grid, 256, bytes, stream>>>(a);
    else if (lds) bias_fwd_kernel<true, false><<<grid, 256, bytes, stream>>>(a);
    else if (vec) bias_fwd_kernel<false, true><<<grid, 256, bytes, stream>>>(a);
    else bias_fwd_kernel<false, false><<<grid, 256, bytes, stream>>>(a);
    return (int)hipGetLastError();
}

extern "C" size_t batteries_distance_bias_backward_workspace_bytes(int64_t E, int H, int B) {
    if (!bias_shape_ok(E, H, B)) return 0;
    return (size_t)bias_parts(E, H, B) * B * H * sizeof(float);
}

extern "C" int batteries_distance_bias_backward(const float* lengths, const uint16_t* buckets,
                                                const float* g, float* gtable, float* glengths,
                                                int64_t E, int H, int B, float cutoff,
                                                void* workspace, size_t workspace_bytes,
                                                hipStream_t stream) {
    if (!bias_shape_ok(E, H, B) || !bias_cutoff_ok(cutoff) ||
        (E > 0 && (!g || (gtable && !buckets) || (glengths && !lengths))))
        return BM_ERR_ARG;
    BiasArgs a{};
    a.lengths = lengths; a.g = g; a.bucket = buckets; a.glengths = glengths;
    a.part = (float*)workspace; a.edges = E; a.H = H; a.B = B; a.cutoff = cutoff;
    if (gtable) {
        if (workspace_bytes < batteries_distance_bias_backward_workspace_bytes(E, H, B) || !workspace)
            return BM_ERR_WORKSPACE;
        const int rw = bias_range_waves(B), parts = E > 0 ? bias_parts(E, H, B) : 0;
        if (parts) {
            const dim3 grid((unsigned)parts, (unsigned)ceil_div(B, kBiasRange * rw),
                            (unsigned)ceil_div(H, 64));
            const size_t lds = 4 * std::min(B, kBiasRange) * 64 * sizeof(float);
            if (rw > 1) bias_bwd_kernel<true><<<grid, 256, lds, stream>>>(a, rw);
            else bias_bwd_kernel<false><<<grid, 256, lds, stream>>>(a, rw);
        }
        const int64_t cols = (int64_t)B * H;
        bias_table_kernel<<<(unsigned)ceil_div(cols, 16), 1024, 0, stream>>>(a.part, parts, cols,
                                                                            gtable);
    }
    if (glengths && E > 0) {
        if (H % 4 == 0 && aligned_to({g}, 16)) bias_lengths_run<true>(a, stream);
        else bias_lengths_run<false>(a, stream);
    }
    return (int)hipGetLastError();
}
