// Channels of features mixed degree by degree, the linear layer of equivariant features (no reference
// counterpart).  l(m) the degree of component m (0 | 1..3 | 4..8 | 9..15):
//
//   y[n, o, m]  = sum_c x[n, c, m] W[l(m), c, o]
//   gx[n, c, m] = sum_o g[n, o, m] W[l(m), c, o]                   (the same kernel, W transposed)
//   gW[l, c, o] = sum_n sum_{m of degree l} x[n, c, m] g[n, o, m]  (x as it was, or from its 8-bit form)
//
// All on the bf16 matrix cores with fp32 sums.  fp32 features and weights go in three parts and six
// products, as exact as fp32 products; the fp32 weight of bf16 features goes in two (off by 2^-15 of it
// at most), bf16 features in one, which is exact; an 8-bit form is exact in bf16, so against it only g is
// split.
//
// The features lie [N, C, 16], 16 components together, and a matrix operand wants 8 values along the sum
// for one component.  A lane therefore loads the same four components of 8 channels (or of 8 atoms,
// for gW), and the operand of each component is its values of the eight: in bf16 one v_perm for two of
// them.  The four waves of a workgroup take four components each of the same atoms and
// channels, so a cache line is read by all of them at about the same time, and a wave meets two
// degrees at most.  The order of the sum is free as long as both operands have the same one: value j of lane
// group q is channel (atom) 4 j + q, so that a load covers neighbours.
#include <type_traits>

#include "checkpoint.h"
#include "sums.h"
#include "batmobile_hip.h"

namespace bmhip {

constexpr int kMixMaxC = 2048;
constexpr int kMixFar = 0x7fffff00;        // a buffer offset past every buffer here: reads 0

// degrees of a wave's first component and of its other three
__device__ __forceinline__ int mix_degree0(int quarter) { return (0x3220 >> (4 * quarter)) & 15; }
__device__ __forceinline__ int mix_degree1(int quarter) { return (0x3321 >> (4 * quarter)) & 15; }

// Four components of eight rows, and from them the operand of each component, in PARTS parts
template <typename T>
struct Mix8;
template <>
struct Mix8<float> {
    static constexpr int kParts = 3, kBytes = 4;
    float4 r[8];
    __device__ __forceinline__ void load(int j, __amdgpu_buffer_rsrc_t b, int off) {
        r[j] = buffer_ld4(b, off, 0);
    }
    template <int I>
    __device__ __forceinline__ void operand(v4u* f) const {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = I == 0 ? r[j].x : I == 1 ? r[j].y : I == 2 ? r[j].z : r[j].w;
        const Bf3 s = bf16_split8(v);
        f[0] = s.h, f[1] = s.m, f[2] = s.l;
    }
};
template <>
struct Mix8<uint16_t> {
    static constexpr int kParts = 1, kBytes = 2;
    unsigned r[8][2];
    __device__ __forceinline__ void load(int j, __amdgpu_buffer_rsrc_t b, int off) {
        const auto v = __builtin_amdgcn_raw_buffer_load_b64(b, off, 0, 0);
        r[j][0] = v[0], r[j][1] = v[1];
    }
    template <int I>
    __device__ __forceinline__ void operand(v4u* f) const {
        constexpr unsigned kSel = I % 2 ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            f[0][j] = __builtin_amdgcn_perm(r[2 * j + 1][I / 2], r[2 * j][I / 2], kSel);
    }
};

// acc += A B in the products that PA and PB parts need, the small ones first
template <int PA, int PB>
__device__ __forceinline__ v4f mix_mfma(const v4u* a, const v4u* b, v4f acc) {
#pragma unroll
    for (int s = 2; s >= 0; --s)
#pragma unroll
        for (int i = PA - 1; i >= 0; --i) {
            const int j = s - i;
            if (j >= 0 && j < PB) acc = mfma_bf16(a[i], b[j], acc);
        }
    return acc;
}

// v in two parts of one sign, the leading bits (upper half of the result) and the rest (lower half, to
// nearest).  A feature's infinity then ends as one of the same sign in both products; so that it does where
// nothing is left over, the least number of that sign stands in for it.  An infinite v is all in the
// first part.
__device__ __forceinline__ unsigned mix_two_parts(float v) {
    const unsigned bits = __float_as_uint(v), h = bits & 0xffff0000u;
    if (v != v) return 0x7fc00000u;
    unsigned m = bf16_pack(v - __uint_as_float(h), 0.0f) & 0xffffu;
    if ((m & 0x7fffu) == 0 || (m & 0x7fffu) >= 0x7f80u) m = v == 0.0f ? 0u : (h >> 16 & 0x8000u) | 1u;
    return h | m;
}

// W (element W[l][k][m] at l K M + k sk + m sm) as the matrix operands of its parts: 16 bytes a lane,
// [step of 32 k][l][tile of 16 m][part][lane], zeros past K and M.
template <int PW>
__global__ __launch_bounds__(256) void mix_pack_kernel(const float* __restrict__ w, v4u* out, int K,
                                                       int M, int sk, int sm, int tiles, int total) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int lane = i & 63, tile = (i >> 6) % tiles, l = (i >> 6) / tiles & 3,
              step = (i >> 6) / tiles >> 2;
    const int m = tile * 16 + (lane & 15), q = lane >> 4;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int k = step * 32 + 4 * j + q;
        v[j] = k < K && m < M ? w[(int64_t)l * K * M + (int64_t)k * sk + (int64_t)m * sm] : 0.0f;
    }
    v4u* p = out + (int64_t)(i >> 6) * PW * 64 + lane;
    if constexpr (PW == 3) {
        const Bf3 s = bf16_split8(v);
        p[0] = s.h, p[64] = s.m, p[128] = s.l;
    } else {
        v4u h, m;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned a = mix_two_parts(v[2 * j]), b = mix_two_parts(v[2 * j + 1]);
            h[j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            m[j] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        }
        p[0] = h, p[64] = m;
    }
}

struct MixArgs {
    const void *x, *g;
    const uint8_t *codes, *exps;
    const v4u* w;
    void* y;
    float* part;
    int64_t n;
    int K, M;                              // channels in, out
    int tiles, chunks, groups;             // tiles of 16 outputs (padded), chunks of them; waves / 4
    int64_t units;                         // workgroups of atoms
    int splits, per_split;                 // gW: ranges of atoms, steps of 32 atoms in one
};

// Workgroup b of `units` times `per`: those of a unit follow each other on one XCD (b % 8), which
// then has in its L2 what they share.
__device__ __forceinline__ bool mix_place(int64_t units, int per, int64_t& unit, int& which) {
    const int xcd = blockIdx.x & 7;
    const unsigned i = blockIdx.x >> 3;
    unit = (int64_t)(i / per) * 8 + xcd;
    which = i % per;
    return unit < units;
}
static unsigned mix_grid(int64_t units, int per) { return (unsigned)(ceil_div(units, 8) * 8 * per); }

// y: 16 NT atoms, OT tiles of outputs for each group of four waves
template <typename T, int PW, int NT, int OT>
__global__ __launch_bounds__(512) void mix_kernel(MixArgs a) {
    constexpr int PX = Mix8<T>::kParts, kB = Mix8<T>::kBytes;
    constexpr int kPitch = 16 * 16 + 4;    // floats of an atom in LDS
    __shared__ __attribute__((aligned(16))) float sh[2][16 * kPitch];
    int64_t unit;
    int chunk;
    if (!mix_place(a.units, a.chunks, unit, chunk)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, quarter = wave & 3, group = wave >> 2;
    const int q = lane >> 4, at = lane & 15;
    const int64_t n0 = unit * 16 * NT;
    const int tile0 = (chunk * a.groups + group) * OT;
    const int rows = (int)min((int64_t)16 * NT, a.n - n0);
    const __amdgpu_buffer_rsrc_t xb =
        buffer_rsrc((const float*)((const char*)a.x + n0 * a.K * 16 * kB), rows * a.K * 16 * kB);
    const int d0 = mix_degree0(quarter), d1 = mix_degree1(quarter);
    v4f acc[4][NT][OT];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < NT; ++k)
#pragma unroll
            for (int o = 0; o < OT; ++o) acc[i][k][o] = v4f{0, 0, 0, 0};
    const int steps = (a.K + 31) / 32;
    for (int s = 0; s < steps; ++s) {
        v4u f[4][NT][PX];
#pragma unroll
        for (int k = 0; k < NT; ++k) {
            Mix8<T> x;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int c = s * 32 + 4 * j + q;
                x.load(j, xb, c < a.K ? (((k * 16 + at) * a.K + c) * 16 + quarter * 4) * kB : kMixFar);
            }
            x.template operand<0>(f[0][k]);
            x.template operand<1>(f[1][k]);
            x.template operand<2>(f[2][k]);
            x.template operand<3>(f[3][k]);
        }
        const v4u* w = a.w + (int64_t)(s * 4 * a.tiles + tile0) * PW * 64 + lane;
#pragma unroll
        for (int o = 0; o < OT; ++o) {
            v4u w0[PW], w1[PW];
#pragma unroll
            for (int p = 0; p < PW; ++p) {
                w0[p] = w[((int64_t)d0 * a.tiles + o) * PW * 64 + p * 64];
                w1[p] = w[((int64_t)d1 * a.tiles + o) * PW * 64 + p * 64];
            }
#pragma unroll
            for (int k = 0; k < NT; ++k) {
                acc[0][k][o] = mix_mfma<PW, PX>(w0, f[0][k], acc[0][k][o]);
#pragma unroll
                for (int i = 1; i < 4; ++i)
                    acc[i][k][o] = mix_mfma<PW, PX>(w1, f[i][k], acc[i][k][o]);
            }
        }
    }
    // the four waves' components of 16 atoms x 16 outputs together, and out as whole lines
    const int t = threadIdx.x & 255;
#pragma unroll
    for (int k = 0; k < NT; ++k)
#pragma unroll
        for (int o = 0; o < OT; ++o) {
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *reinterpret_cast<float4*>(&sh[group][at * kPitch + (4 * q + r) * 16 + quarter * 4]) =
                    make_float4(acc[0][k][o][r], acc[1][k][o][r], acc[2][k][o][r], acc[3][k][o][r]);
            __syncthreads();
            const int m0 = (tile0 + o) * 16;
            constexpr int kUnit = 16 / kB, kPer = 256 / kUnit;     // 16-byte pieces of an atom
#pragma unroll
            for (int i = 0; i < 16 * kPer / 256; ++i) {
                const int p = i * 256 + t, node = p / kPer, e = p % kPer * kUnit;
                if (k * 16 + node >= rows || m0 + e / 16 >= a.M) continue;
                const float4 u = *reinterpret_cast<const float4*>(&sh[group][node * kPitch + e]);
                const int64_t to = ((n0 + k * 16 + node) * a.M + m0) * 16 + e;
                if constexpr (kB == 4) {
                    *reinterpret_cast<float4*>((float*)a.y + to) = u;
                } else {
                    const float4 v = *reinterpret_cast<const float4*>(&sh[group][node * kPitch + e + 4]);
                    *reinterpret_cast<uint4*>((uint16_t*)a.y + to) =
                        make_uint4(bf16_pack(u.x, u.y), bf16_pack(u.z, u.w), bf16_pack(v.x, v.y),
                                   bf16_pack(v.z, v.w));
                }
            }
        }
}

// The 8-bit form of eight atoms: the code's value is exact in bf16
struct MixKept {
    static constexpr int kParts = 1, kBytes = 1;
};
__device__ __forceinline__ void mix_decode(unsigned code, int e, unsigned* r) {
    const float4 v = ckpt_decode4(code, ckpt_up(e));
    r[0] = bf16_pack(v.x, v.y);
    r[1] = bf16_pack(v.z, v.w);
}

// gW: a workgroup takes CT x OT tiles of (c, o) over a range of atoms.  part [splits, 6, K, M]: the
// sums of the quarters' degrees 0 1 | 2 | 2 3 | 3.
template <typename X, typename G, int CT, int OT>
__global__ __launch_bounds__(256) void mix_weight_kernel(MixArgs a) {
    constexpr bool kKept = X::kBytes == 1;
    constexpr int PX = X::kParts, PG = G::kParts;
    int64_t split;
    int which;
    if (!mix_place(a.splits, a.tiles * a.chunks, split, which)) return;
    const int lane = threadIdx.x & 63, quarter = threadIdx.x >> 6;
    const int q = lane >> 4, at = lane & 15;
    const int c0 = which % a.tiles * CT * 16, o0 = which / a.tiles * OT * 16;
    v4f acc[2][CT][OT];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < CT; ++k)
#pragma unroll
            for (int o = 0; o < OT; ++o) acc[i][k][o] = v4f{0, 0, 0, 0};
    const int exps = ckpt_blocks(a.K);
    const int64_t last = min(a.n, (split + 1) * a.per_split * 32);
    for (int64_t n0 = split * a.per_split * 32; n0 < last; n0 += 32) {
        const int rows = (int)min((int64_t)32, a.n - n0);
        const __amdgpu_buffer_rsrc_t gb = buffer_rsrc(
            (const float*)((const char*)a.g + n0 * a.M * 16 * G::kBytes), rows * a.M * 16 * G::kBytes);
        const void* xs = kKept ? (const void*)(a.codes + n0 * a.K * 16)
                               : (const void*)((const char*)a.x + n0 * a.K * 16 * X::kBytes);
        const __amdgpu_buffer_rsrc_t xb = buffer_rsrc((const float*)xs, rows * a.K * 16 * X::kBytes);
        typename std::conditional<kKept, Mix8<uint16_t>, X>::type x[CT];
        G g[OT];
        if constexpr (kKept) {
            const __amdgpu_buffer_rsrc_t eb =
                buffer_rsrc((const float*)(a.exps + n0 * exps), rows * exps);
            unsigned code[CT][8];
            int e[CT][8];
#pragma unroll
            for (int k = 0; k < CT; ++k)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int c = c0 + k * 16 + at, n = 4 * j + q;
                    code[k][j] = __builtin_amdgcn_raw_buffer_load_b32(
                        xb, c < a.K ? (n * a.K + c) * 16 + quarter * 4 : kMixFar, 0, 0);
                    e[k][j] = __builtin_amdgcn_raw_buffer_load_b8(
                        eb, c < a.K ? n * exps + c / kCkptChannels : kMixFar, 0, 0);
                }
#pragma unroll
            for (int k = 0; k < CT; ++k)
#pragma unroll
                for (int j = 0; j < 8; ++j) mix_decode(code[k][j], e[k][j], x[k].r[j]);
        } else {
#pragma unroll
            for (int k = 0; k < CT; ++k)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int c = c0 + k * 16 + at;
                    x[k].load(j, xb, c < a.K ? (((4 * j + q) * a.K + c) * 16 + quarter * 4) * X::kBytes
                                             : kMixFar);
                }
        }
#pragma unroll
        for (int k = 0; k < OT; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int o = o0 + k * 16 + at;
                g[k].load(j, gb, o < a.M ? (((4 * j + q) * a.M + o) * 16 + quarter * 4) * G::kBytes
                                         : kMixFar);
            }
        static_for<4>([&](auto ii) {
            constexpr int I = decltype(ii)::value;
            v4u fx[CT][PX], fg[OT][PG];
#pragma unroll
            for (int k = 0; k < CT; ++k) x[k].template operand<I>(fx[k]);
#pragma unroll
            for (int k = 0; k < OT; ++k) g[k].template operand<I>(fg[k]);
#pragma unroll
            for (int k = 0; k < CT; ++k)
#pragma unroll
                for (int o = 0; o < OT; ++o)
                    acc[I > 0][k][o] = mix_mfma<PX, PG>(fx[k], fg[o], acc[I > 0][k][o]);
        });
    }
    const int slab = quarter + (quarter + 1) / 2;          // 0 2 3 5
    const bool one = quarter & 1;                          // one degree: the two sums together
    float* part = a.part + ((int64_t)split * 6 + slab) * a.K * a.M;
#pragma unroll
    for (int k = 0; k < CT; ++k)
#pragma unroll
        for (int o = 0; o < OT; ++o)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int c = c0 + k * 16 + 4 * q + r, m = o0 + o * 16 + at;
                if (c >= a.K || m >= a.M) continue;
                const float u = acc[0][k][o][r], v = acc[1][k][o][r];
                part[(int64_t)c * a.M + m] = one ? u + v : u;
                if (!one) part[((int64_t)a.K + c) * a.M + m] = v;
            }
}

__global__ __launch_bounds__(1024) void mix_weight_sum_kernel(const float* __restrict__ part, int splits,
                                                              int64_t cells, float* out) {
    const int64_t col = (int64_t)blockIdx.x * 16 + (threadIdx.x & 15);
    const bool there = col < 4 * cells;
    const int l = there ? (int)(col / cells) : 0;
    const float* p = part + (l < 2 ? l : 2 * l - 2) * cells + (col - l * cells);
    const float s = column_sum(there ? splits : 0, [&](int r) {
        const float* v = p + r * 6 * cells;
        return l < 2 ? v[0] : v[0] + v[cells];
    });
    if (threadIdx.x < 16 && there) out[col] = s;
}

static bool mix_shape_ok(int64_t N, int C, int O, int dtype) {
    return N >= 0 && N < ((int64_t)1 << 31) && C >= 1 && C <= kMixMaxC && O >= 1 && O <= kMixMaxC &&
           (dtype == 0 || dtype == 1);
}

// Tiles of outputs of a wave, and groups of four waves
template <typename T>
struct MixShape {
    static constexpr int kNT = 2, kOT = sizeof(T) == 4 ? 2 : 4, kPW = sizeof(T) == 4 ? 3 : 2;
};
template <typename T>
static void mix_tiles(int M, MixArgs& a) {
    constexpr int kOT = MixShape<T>::kOT;
    a.groups = M <= kOT * 16 ? 1 : 2;
    a.chunks = (M + kOT * a.groups * 16 - 1) / (kOT * a.groups * 16);
    a.tiles = a.chunks * a.groups * kOT;
}
template <typename T>
static size_t mix_bytes(int K, int M) {
    MixArgs a{};
    mix_tiles<T>(M, a);
    return (size_t)((K + 31) / 32) * 4 * a.tiles * MixShape<T>::kPW * 64 * 16;
}

template <typename T>
static void mix_run(MixArgs a, const float* w, int sk, int sm, void* ws, hipStream_t s) {
    using S = MixShape<T>;
    mix_tiles<T>(a.M, a);
    const int total = (a.K + 31) / 32 * 4 * a.tiles * 64;
    mix_pack_kernel<S::kPW><<<(total + 255) / 256, 256, 0, s>>>(w, (v4u*)ws, a.K, a.M, sk, sm, a.tiles,
                                                               total);
    a.w = (const v4u*)ws;
    constexpr int64_t kAtoms = (int64_t)1 << 24;     // of a launch
    const int64_t n = a.n;
    const char *x = (const char*)a.x;
    char* y = (char*)a.y;
    for (int64_t n0 = 0; n0 < n; n0 += kAtoms) {
        a.x = x + n0 * a.K * 16 * (int64_t)sizeof(T);
        a.y = y + n0 * a.M * 16 * (int64_t)sizeof(T);
        a.n = std::min(n - n0, kAtoms);
        a.units = ceil_div(a.n, 16 * S::kNT);
        mix_kernel<T, S::kPW, S::kNT, S::kOT>
            <<<mix_grid(a.units, a.chunks), 256 * a.groups, 0, s>>>(a);
    }
}

// Ranges of atoms of gW: about 1024 workgroups of at least four steps, 64 MB of partial sums at most
static int mix_splits(int64_t N, int C, int O) {
    const int64_t tiles = ceil_div(C, 64) * ceil_div(O, 32);
    const int64_t most = std::max<int64_t>(1, ((int64_t)1 << 24) / ((int64_t)6 * C * O));
    return (int)std::max<int64_t>(
        1, std::min({ceil_div(1024, tiles), ceil_div(N, 128), most}));
}

template <typename X, typename G, int CT, int OT>
static void mix_weight_run(MixArgs a, hipStream_t s) {
    a.tiles = (a.K + 16 * CT - 1) / (16 * CT);
    a.chunks = (a.M + 16 * OT - 1) / (16 * OT);
    a.per_split = (int)ceil_div(ceil_div(a.n, 32), a.splits);
    mix_weight_kernel<X, G, CT, OT>
        <<<mix_grid(a.splits, a.tiles * a.chunks), 256, 0, s>>>(a);
}
}  // namespace bmhip

using namespace bmhip;

extern "C" size_t batteries_channel_mixing_workspace_bytes(int C, int O, int transposed, int dtype) {
    if (!mix_shape_ok(0, C, O, dtype)) return 0;
    if (transposed) std::swap(C, O);
    return dtype == 0 ? mix_bytes<float>(C, O) : mix_bytes<uint16_t>(C, O);
}

extern "C" int batteries_channel_mixing(const void* x, const float* weight, void* y, int64_t N, int C,
                                        int O, int transposed, int dtype, void* workspace,
                                        size_t workspace_bytes, hipStream_t stream) {
    if (!mix_shape_ok(N, C, O, dtype) || (N > 0 && (!x || !weight || !y))) return BM_ERR_ARG;
    if (!aligned_to({x, y, workspace}, 16) || !aligned_to({weight}, 4)) return BM_ERR_ARG;
    if (N == 0) return BM_OK;
    if (workspace_bytes < batteries_channel_mixing_workspace_bytes(C, O, transposed, dtype) || !workspace)
        return BM_ERR_WORKSPACE;
    MixArgs a{};
    a.x = x; a.y = y; a.n = N; a.K = transposed ? O : C; a.M = transposed ? C : O;
    const int sk = transposed ? 1 : O, sm = transposed ? O : 1;
    if (dtype == 0) mix_run<float>(a, weight, sk, sm, workspace, stream);
    else mix_run<uint16_t>(a, weight, sk, sm, workspace, stream);
    return (int)hipGetLastError();
}

extern "C" size_t batteries_channel_mixing_weight_grad_workspace_bytes(int64_t N, int C, int O) {
    if (!mix_shape_ok(N, C, O, 0)) return 0;
    return (size_t)mix_splits(N, C, O) * 6 * C * O * sizeof(float);
}

extern "C" int batteries_channel_mixing_weight_grad(const void* x, const uint8_t* codes,
                                                    const uint8_t* exps, const void* g, float* gweight,
                                                    int64_t N, int C, int O, int dtype, void* workspace,
                                                    size_t workspace_bytes, hipStream_t stream) {
    if (!mix_shape_ok(N, C, O, dtype) || !gweight || (N > 0 && (!g || (!x && (!codes || !exps)))))
        return BM_ERR_ARG;
    if (!aligned_to({x, g}, 16) || !aligned_to({codes}, 4)) return BM_ERR_ARG;
    if (workspace_bytes < batteries_channel_mixing_weight_grad_workspace_bytes(N, C, O) || !workspace)
        return BM_ERR_WORKSPACE;
    MixArgs a{};
    a.x = x; a.codes = codes; a.exps = exps; a.g = g; a.part = (float*)workspace; a.n = N; a.K = C;
    a.M = O; a.splits = mix_splits(N, C, O);
    if (N > 0) {
        using F = Mix8<float>;
        using B = Mix8<uint16_t>;
        if (dtype == 0) {
            if (x) mix_weight_run<F, F, 2, 2>(a, stream);
            else mix_weight_run<MixKept, F, 4, 2>(a, stream);
        } else {
            if (x) mix_weight_run<B, B, 4, 2>(a, stream);
            else mix_weight_run<MixKept, B, 4, 2>(a, stream);
        }
    }
    const int64_t cells = (int64_t)C * O;
    mix_weight_sum_kernel<<<(unsigned)ceil_div(4 * cells, 16), 1024, 0, stream>>>(
        a.part, N > 0 ? a.splits : 0, cells, gweight);
    return (int)hipGetLastError();
}
