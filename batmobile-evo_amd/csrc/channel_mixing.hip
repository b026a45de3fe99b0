// Channels of features mixed degree by degree, the linear layer of equivariant features (no reference
// counterpart).  l(m) the degree of component m (0 | 1..3 | 4..8 | 9..15):
//
//   y[n, o, m]  = sum_c x[n, c, m] W[l(m), c, o]
//   gx[n, c, m] = sum_o g[n, o, m] W[l(m), c, o]                   (the same kernel, W transposed)
//   gW[l, c, o] = sum_n sum_{m of degree l} x[n, c, m] g[n, o, m]  (x as it was, or from its 8-bit form)
//
// Sums are fp32. bf16 features go to the bf16 matrix cores as they are; their weight, which is fp32, goes
// in two parts (off by 2^-15 of it at most): a third would make a wave's 128 registers of weight 192, for
// results that are rounded to 8 bits. At 128 to 128 channels 0.45 % of them round the other way than with
// all 24 bits, and the error against 64 bits is the same, 1.659e-3. fp32 features run on the fp32 matrix
// cores (up to 64 channels in, and for gW) or, three parts each, in six products on the bf16 ones, as exact
// as fp32 products. An 8-bit form is exact in bf16, so against it only g is split.
//
// The features lie [N, C, 16], 16 components together, and a matrix operand wants 8 values along the sum
// for one component.  Whole lines come to LDS by direct loads; from there a lane takes the same components
// of 8 channels (for gW of 4 atoms), and the operand of each component is its values of the eight: in bf16
// one v_perm for two of them.  A wave takes 4 or 8 of the components, which have two degrees at most.  The
// order of the sum is free as long as both operands have the same one: value j of lane group q is channel
// (atom) 4 j + q.
//
// Measured, us (what the bytes take at a copy's 5 TB/s): 50,000 atoms 128 to 128 in bf16 104 to 112 (82), its gW
// 122 to 136, from the 8-bit form 94 (62); 256 to 128 200 (123); 64 to 64 in bf16 38 (41), in fp32 101 (82); 20,011
// atoms 100 to 200 in fp32 184 (77), 200 to 100 141, gW 234, from the 8-bit form 146.  bf16 is bound by memory and
// by waits for all of it at barriers (stay_wait), above 128 channels by features read again for each 32 outputs;
// fp32 by the matrix cores and the splitting.
#include <atomic>
#include <type_traits>

#include "checkpoint.h"
#include "batmobile_hip.h"

namespace bmhip {

constexpr int kMixMaxC = 2048;
// Channels up to which the weight stays in registers.  Against the general kernel, us: fp32 50,000 atoms 64
// to 64 101 and 114, 33 to 100 162 and 158; bf16 50,000 64 to 64 38 and 52, 128 to 128 104 to 112 and 151, 128 to
// 256 188 and 266, 256 to 128 200 and 222; 20,011 160 to 160 72 and 72, 200 to 256 162 and 159, 256 to 64 47 and 62.
// fp32 above 64 in registers took 250 at 20,011 100 to 200 (184 as it is); above 256 in bf16 a degree's weight does
// not fit.
template <typename T>
constexpr int kStayMost = sizeof(T) == 4 ? 64 : 256;
constexpr int kMixFar = 0x7fffff00;        // a buffer offset past every buffer here: reads 0

// degrees of a wave's first component and of its other three
__device__ __forceinline__ int mix_degree0(int quarter) { return (0x3220 >> (4 * quarter)) & 15; }
__device__ __forceinline__ int mix_degree1(int quarter) { return (0x3321 >> (4 * quarter)) & 15; }

// Four components of eight channels, and from them the operand of each component, in its parts
template <typename T>
struct Mix8;
template <>
struct Mix8<float> {
    static constexpr int kParts = 3, kBytes = 4;
    float4 r[8];
    __device__ __forceinline__ void load(int j, const char* p) { r[j] = *reinterpret_cast<const float4*>(p); }
    __device__ __forceinline__ void zero(int j) { r[j] = make_float4(0, 0, 0, 0); }
    template <int I>
    __device__ __forceinline__ void operand(v4u* f) const {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = I == 0 ? r[j].x : I == 1 ? r[j].y : I == 2 ? r[j].z : r[j].w;
        // the leading bits, of the rest the leading ones to nearest, and what is left, at most 8 bits.  Of a
        // product second part times third is dropped twice, 2^-23 of it at most and of either sign.  An
        // infinity ends as NaN: mix_again.
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned a = __float_as_uint(v[2 * j]), b = __float_as_uint(v[2 * j + 1]);
            const float ra = v[2 * j] - __uint_as_float(a & 0xffff0000u);
            const float rb = v[2 * j + 1] - __uint_as_float(b & 0xffff0000u);
            const unsigned m = bf16_pack(ra, rb);
            f[0][j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            f[1][j] = m;
            f[2][j] = __builtin_amdgcn_perm(__float_as_uint(rb - bf16_hi(m)),
                                            __float_as_uint(ra - bf16_lo(m)), 0x07060302u);
        }
    }
};
template <>
struct Mix8<uint16_t> {
    static constexpr int kParts = 1, kBytes = 2;
    unsigned r[8][2];
    __device__ __forceinline__ void load(int j, const char* p) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        r[j][0] = v.x, r[j][1] = v.y;
    }
    __device__ __forceinline__ void zero(int j) { r[j][0] = r[j][1] = 0; }
    template <int I>
    __device__ __forceinline__ void operand(v4u* f) const {
        constexpr unsigned kSel = I % 2 ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            f[0][j] = __builtin_amdgcn_perm(r[2 * j + 1][I / 2], r[2 * j][I / 2], kSel);
    }
};

// v in two parts of one sign, the leading bits (upper half of the result) and the rest (lower half, to
// nearest).  A feature's infinity then ends as one of the same sign in both products; so that it does where
// nothing is left over, the least number of that sign stands in for it.  An infinite v is all in the
// first part.
__device__ __forceinline__ unsigned mix_two_parts(float v) {
    const unsigned h = __float_as_uint(v) & 0xffff0000u;
    const unsigned m = bf16_pack(v - __uint_as_float(h), 0.0f) & 0xffffu;
    const unsigned least = v == 0.0f ? 0u : (h >> 16 & 0x8000u) | 1u;
    // (nothing left over, or an infinite v)
    const unsigned rest = (m & 0x7fffu) - 1u >= 0x7f7fu ? least : m;
    return v != v ? 0x7fc00000u : h | rest;
}

// Eight fp32 values as the operands of their parts
template <int PW>
__device__ __forceinline__ void mix_split(const float* v, v4u* p) {
    if constexpr (PW == 3) {
        const Bf3 s = bf16_split8(v);
        p[0] = s.h, p[1] = s.m, p[2] = s.l;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const unsigned a = mix_two_parts(v[2 * j]), b = mix_two_parts(v[2 * j + 1]);
            p[0][j] = __builtin_amdgcn_perm(b, a, 0x07060302u);
            p[1][j] = __builtin_amdgcn_perm(b, a, 0x05040100u);
        }
    }
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
    v4u f[PW];
    mix_split<PW>(v, f);
#pragma unroll
    for (int p = 0; p < PW; ++p) out[((int64_t)(i >> 6) * PW + p) * 64 + lane] = f[p];
}

struct MixArgs {
    const void *x, *g;
    const uint8_t *codes, *exps;
    const v4u* w;                          // in parts (mix_pack_kernel)
    const float* weight;                   // as given: element l K M + k sk + m sm
    int sk, sm;
    void* y;
    float* part;
    int64_t n;
    int K, M;                              // channels in, out
    int tiles, chunks;                     // tiles of 16 outputs (padded), chunks of them
    int64_t units;                         // workgroups of atoms
    int splits, per_split;                 // gW: ranges of atoms, steps in one
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

// Four components, from `comp` on, of one fp32 result: those that are not finite again in plain fp32
__device__ __forceinline__ float4 mix_again(const MixArgs& a, int64_t n, int m, int comp, float4 u) {
    const float* x = (const float*)a.x + n * a.K * 16 + comp;
    const float* w0 = a.weight + (int64_t)mix_degree0(comp / 4) * a.K * a.M + (int64_t)m * a.sm;
    const float* w1 = a.weight + (int64_t)mix_degree1(comp / 4) * a.K * a.M + (int64_t)m * a.sm;
    float4 s = make_float4(0, 0, 0, 0);
#pragma unroll 1
    for (int k = 0; k < a.K; ++k) {
        const float4 v = *reinterpret_cast<const float4*>(x + k * 16);
        const float f = w0[(int64_t)k * a.sk], g = w1[(int64_t)k * a.sk];
        s.x = fmaf(v.x, f, s.x);
        s.y = fmaf(v.y, g, s.y);
        s.z = fmaf(v.z, g, s.z);
        s.w = fmaf(v.w, g, s.w);
    }
    const float inf = __builtin_inff();
    return make_float4(fabsf(u.x) < inf ? u.x : s.x, fabsf(u.y) < inf ? u.y : s.y,
                       fabsf(u.z) < inf ? u.z : s.z, fabsf(u.w) < inf ? u.w : s.w);
}

// y of 16 NG atoms and OT tiles of outputs: NG groups of four waves take 16 atoms each, a wave four
// components.
//
// A step is 32 channels.  Its weights (4 degrees x OT tiles x PW parts, 1 KB each) and its features come to LDS
// by direct loads while the step before is worked on, the weights into two buffers, the features into one: a
// wave takes its share to registers first.  Loaded to registers from memory, 16 bytes of every 64 a lane, each
// wave had its lines to itself: 64 KB of a step do not stay in L1 until the other three waves ask for them
// (20,011 x 100 to 200 in f32 207 us, so 196).
template <typename T>
struct MixTile {
    static constexpr int kB = sizeof(T), kPW = kB == 4 ? 3 : 2, kOT = 4, kNG = 2;
    static constexpr int kAtom = 512 * kB;                         // bytes of an atom's 32 channels
    static constexpr int kW = 4 * kOT * kPW * 1024, kX = 16 * kNG * kAtom;
    static constexpr int kBytes = 2 * kW + kX;
    static constexpr int kPitch = 16 * 16 + 4;                     // floats of an atom on the way out
    static_assert(kNG * 16 * kPitch * 4 <= kBytes, "the results take the buffers' place");
};

template <typename T>
__device__ __forceinline__ void mix_general(const MixArgs& a, char* sh) {      // sh: weights, weights, features
    using S = MixTile<T>;
    constexpr int PW = S::kPW, PX = Mix8<T>::kParts, OT = S::kOT, kB = S::kB, kWaves = 4 * S::kNG;
    constexpr int kPitch = S::kPitch, kPieces = S::kAtom / 16;
    int64_t unit;
    int chunk;
    if (!mix_place(a.units, a.chunks, unit, chunk)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int quarter = wave & 3, group = wave >> 2, q = lane >> 4, at = lane & 15;
    const int64_t n0 = unit * S::kNG * 16;
    const int tile0 = chunk * OT;
    const int rows = (int)min((int64_t)16 * S::kNG, a.n - n0);
    const __amdgpu_buffer_rsrc_t xb =
        buffer_rsrc((const float*)((const char*)a.x + n0 * a.K * 16 * kB), rows * a.K * 16 * kB);
    const int d0 = mix_degree0(quarter), d1 = mix_degree1(quarter);
    const int steps = (a.K + 31) / 32;
    // weights of a step: [l][tile][part][lane], OT tiles of a.tiles
    const __amdgpu_buffer_rsrc_t wb = buffer_rsrc(
        (const float*)(a.w + (int64_t)tile0 * PW * 64), (uint32_t)((steps * 4 * a.tiles - tile0) * PW * 1024));
    // lanes past the last atom or, after the last step of K, past the last channel bring what lies there
    // (past the buffer nothing): no result that is stored takes them
    auto ask = [&](int s, char* lds) {
        char* to = lds + (s & 1) * S::kW;
#pragma unroll
        for (int i = 0; i < S::kW / 1024 / kWaves; ++i) {
            const int f = i * kWaves + wave;               // 1 KB: degree f / (OT PW)
            const int from = ((s * 4 + f / (OT * PW)) * a.tiles * PW + f % (OT * PW)) * 1024;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                wb, (__attribute__((address_space(3))) void*)(to + f * 1024), 16, lane * 16 + from, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < S::kX / 1024 / kWaves; ++i) {
            const int load = i * kWaves + wave, node = load * 64 / kPieces;
            const int p = (load * 64 % kPieces + lane) ^ (node & 15);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                xb, (__attribute__((address_space(3))) void*)(lds + 2 * S::kW + load * 1024), 16,
                node * a.K * 16 * kB + s * S::kAtom + p * 16, 0, 0, 0);
        }
        asm volatile("" ::: "memory");
    };
    // this lane's pieces: (4 j + q) kB + quarter kB / 4, permuted by the atom's number
    const char* mine = sh + 2 * S::kW + (group * 16 + at) * S::kAtom;
    const int piece = q * kB + quarter * kB / 4;
    v4f acc[4][OT];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int o = 0; o < OT; ++o) acc[i][o] = v4f{0, 0, 0, 0};
    ask(0, sh);
    for (int s = 0; s < steps; ++s) {
        // this step's loads are in, those of every wave; the step before is worked off
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __syncthreads();
        Mix8<T> x;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            x.load(j, mine + ((piece + 4 * j * kB) ^ at) * 16 + (kB == 2 ? quarter % 2 * 8 : 0));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __syncthreads();                                   // the features' buffer is free
        if (s + 1 < steps) ask(s + 1, sh);
        if ((a.K & 31) && s == steps - 1) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (s * 32 + 4 * j + q >= a.K) x.zero(j);
        }
        v4u f[4][PX];
        x.template operand<0>(f[0]);
        x.template operand<1>(f[1]);
        x.template operand<2>(f[2]);
        x.template operand<3>(f[3]);
        const v4u* w = reinterpret_cast<const v4u*>(sh + (s & 1) * S::kW) + lane;
#pragma unroll
        for (int o = 0; o < OT; ++o) {
            v4u w0[PW], w1[PW];
#pragma unroll
            for (int p = 0; p < PW; ++p) w0[p] = w[((d0 * OT + o) * PW + p) * 64];
#pragma unroll
            for (int p = 0; p < PW; ++p) w1[p] = w[((d1 * OT + o) * PW + p) * 64];
            // the small products first, successive ones to different sums
#pragma unroll
            for (int sum = 2; sum >= 0; --sum)
#pragma unroll
                for (int p = PW - 1; p >= 0; --p) {
                    const int r = sum - p;
                    if (r < 0 || r >= PX) continue;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        acc[i][o] = mfma_bf16(i ? w1[p] : w0[p], f[i][r], acc[i][o]);
                }
        }
    }
    // the four waves' components of 16 atoms x 16 outputs together, and out as whole lines
    const int t = threadIdx.x & 255;
    float* out = reinterpret_cast<float*>(sh) + group * 16 * kPitch;
#pragma unroll
    for (int o = 0; o < OT; ++o) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int r = 0; r < 4; ++r)
            *reinterpret_cast<float4*>(&out[at * kPitch + (4 * q + r) * 16 + quarter * 4]) =
                make_float4(acc[0][o][r], acc[1][o][r], acc[2][o][r], acc[3][o][r]);
        __syncthreads();
        const int m0 = (tile0 + o) * 16;
        constexpr int kUnit = 16 / kB, kPer = 256 / kUnit;     // 16-byte pieces of an atom
#pragma unroll
        for (int i = 0; i < 16 * kPer / 256; ++i) {
            const int p = i * 256 + t, node = p / kPer, e = p % kPer * kUnit;
            if (group * 16 + node >= rows || m0 + e / 16 >= a.M) continue;
            float4 u = *reinterpret_cast<const float4*>(&out[node * kPitch + e]);
            const int64_t n = n0 + group * 16 + node, to = (n * a.M + m0) * 16 + e;
            if constexpr (kB == 4) {
                if (!(fabsf((u.x + u.y) + (u.z + u.w)) < __builtin_inff()))
                    u = mix_again(a, n, m0 + e / 16, e % 16, u);
                *reinterpret_cast<float4*>((float*)a.y + to) = u;
            } else {
                const float4 v = *reinterpret_cast<const float4*>(&out[node * kPitch + e + 4]);
                *reinterpret_cast<uint4*>((uint16_t*)a.y + to) =
                    make_uint4(bf16_pack(u.x, u.y), bf16_pack(u.z, u.w), bf16_pack(v.x, v.y),
                               bf16_pack(v.z, v.w));
            }
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256 * MixTile<T>::kNG) void mix_kernel(MixArgs a) {
    extern __shared__ __attribute__((aligned(16))) char sh[];
    mix_general<T>(a, sh);
}

// ---------------------------------------------------------------------------
// The same with the weight in registers, for up to 32 KS channels: a workgroup stays, takes tiles of 16
// atoms in turn and reads nothing but features.
//
// A step's features (32 channels of 16 atoms) come to LDS by direct loads of 16 bytes a lane, whole lines,
// asked for kAhead steps ahead (1 in fp32, 2 in bf16; but see stay_wait); straight to registers a wave would
// ask for 8 or 16 bytes of every 32 or 64, whose rate is the address units' (3.6 TB/s with every line in L1). A
// wave takes 8 of the 16 components, those of degrees 1 and 2 (1..8) or of 3 and 0 (9..15, 0), so two degrees
// of the weight, for OT tiles of outputs: 2 KS OT PW registers x 4, 128 at most. With 65 to 128 channels that
// and the sums do not quite fit: to more than 32 outputs 12 bytes a lane lie in scratch memory, to 32 and fewer
// 84, read back in a tile's last step. In LDS the 16-byte pieces of an atom are permuted by its number, so that
// 16 atoms' reads meet no bank twice.
// The two kinds of wave run code of their own, barrier for barrier alike.
// ---------------------------------------------------------------------------
template <typename T>
struct StayRead;
// Of 8 channels components 1..7 of one half of the 16 and the first of the other half, a part at a time
// (all at once they would not fit beside the weight)
template <>
struct StayRead<uint16_t> {
    static constexpr int kPieces = 64;     // 16-byte pieces of an atom's 32 channels
    static constexpr int kParts = 2, kFrom[3] = {0, 7, 8};     // the parts' first components
    v4u m[8];
    __device__ __forceinline__ static int first(int at, int q, int half) {
        return at * 1024 + ((2 * q + half) ^ at) * 16;
    }
    template <int PART>
    __device__ __forceinline__ void load(const char* x, int main, int other) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (PART == 0)
                m[j] = *reinterpret_cast<const v4u*>(x + (main ^ (j & 1) * 128) + (j >> 1) * 256);
            else
                m[j][0] = *reinterpret_cast<const unsigned*>(x + (other ^ (j & 1) * 128) + (j >> 1) * 256);
        }
    }
    __device__ __forceinline__ void cut(int j) { m[j] = v4u{0, 0, 0, 0}; }
    template <int I>                       // component I + 1 of the half; 7: the other's first
    __device__ __forceinline__ void operand(v4u* o) const {
        constexpr int kAt = I < 7 ? I + 1 : 0;
        constexpr unsigned kSel = kAt % 2 ? 0x07060302u : 0x05040100u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            o[0][j] = __builtin_amdgcn_perm(m[2 * j + 1][kAt / 2], m[2 * j][kAt / 2], kSel);
    }
};
template <>
struct StayRead<float> {
    static constexpr int kPieces = 128;
    static constexpr int kParts = 3, kFrom[4] = {0, 3, 7, 8};
    float4 m[8];
    __device__ __forceinline__ static int first(int at, int q, int half) {
        return at * 2048 + ((4 * q + 2 * half) ^ at) * 16;
    }
    template <int PART>
    __device__ __forceinline__ void load(const char* x, int main, int other) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if constexpr (PART < 2)
                m[j] = *reinterpret_cast<const float4*>(x + (main ^ PART * 16) + j * 256);
            else
                m[j].x = *reinterpret_cast<const float*>(x + other + j * 256);
        }
    }
    __device__ __forceinline__ void cut(int j) { m[j] = make_float4(0, 0, 0, 0); }
    template <int I>
    __device__ __forceinline__ float value(int j) const {
        constexpr int kAt = I < 7 ? (I + 1) % 4 : 0;
        return kAt == 0 ? m[j].x : kAt == 1 ? m[j].y : kAt == 2 ? m[j].z : m[j].w;
    }
};

// The weight of 32 channels and 16 outputs, and acc[i][o] += its products with a part of the components
template <typename T>
struct StayWeight;
template <>
struct StayWeight<uint16_t> {
    v4u p[2];
    __device__ __forceinline__ void set(const float* v) { mix_split<2>(v, p); }
};
template <>
struct StayWeight<float> {
    float v[8];
    __device__ __forceinline__ void set(const float* t) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = t[j];
    }
};
// Successive products go to different sums: one that waits for the last result waits for all its cycles
template <int FROM, int TO, int SECOND, int OT>
__device__ __forceinline__ void stay_products(const StayRead<uint16_t>& x,
                                              const StayWeight<uint16_t>* const (&w)[2], v4f (&acc)[8][OT]) {
    constexpr int kAtOnce = OT == 1 ? 2 : 1;
    static_for<(TO - FROM + kAtOnce - 1) / kAtOnce>([&](auto kk) {
        constexpr int I0 = FROM + decltype(kk)::value * kAtOnce, kN = std::min(kAtOnce, TO - I0);
        v4u f[kN];
        static_for<kN>([&](auto ii) {
            x.template operand<I0 + decltype(ii)::value>(&f[decltype(ii)::value]);
        });
#pragma unroll
        for (int p = 1; p >= 0; --p)
#pragma unroll
            for (int i = 0; i < kN; ++i)
#pragma unroll
                for (int o = 0; o < OT; ++o)
                    acc[I0 + i][o] = mfma_bf16(w[I0 + i >= SECOND][o].p[p], f[i], acc[I0 + i][o]);
    });
}
template <int FROM, int TO, int SECOND, int OT>
__device__ __forceinline__ void stay_products(const StayRead<float>& x,
                                              const StayWeight<float>* const (&w)[2], v4f (&acc)[8][OT]) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
        static_for<TO - FROM>([&](auto ii) {
            constexpr int I = FROM + decltype(ii)::value;
#pragma unroll
            for (int o = 0; o < OT; ++o)
                acc[I][o] = mfma1(w[I >= SECOND][o].v[j], x.template value<I>(j), acc[I][o]);
        });
}

template <typename T>
struct StayShape {
    static constexpr int kRing = sizeof(T) == 4 ? 2 : 3, kAhead = kRing - 1;
    static constexpr int kStep = StayRead<T>::kPieces * 16 * 16;       // bytes of a step
    static constexpr int kOut = 16 * 8 * 16 * 4;       // of a group's 16 atoms x 8 outputs on the way out
    static constexpr int bytes(int groups) { return kRing * kStep + groups * kOut; }
};

// Until at most LATER loads and `tiles` tiles' stores are under way: what was asked for before them is
// there (the counter goes down in the order of issue, loads and stores alike).  The wave's own loads, that is: the
// __syncthreads() behind it orders them for the other waves, and for that the compiler has it wait for all vector
// memory, at every step of a tile but the first and at the first barrier of the way out.  So only the first step's
// count lets anything go on: in effect loads have one step, and a tile's stores end within the next one's first.
template <int LATER, int STORES, int MOST>
__device__ __forceinline__ void stay_wait(int tiles) {
    static_for<MOST + 1>([&](auto ii) {
        constexpr int I = decltype(ii)::value;
        static_assert(LATER + I * STORES < 64, "the counter's range");
        if (tiles == I)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LATER + I * STORES) : "memory");
    });
}

template <typename T, int KS, int OT, int OG, int HALF>
__device__ __forceinline__ void mix_stay(const MixArgs& a, char* sh) {
    using S = StayShape<T>;
    constexpr int kB = sizeof(T), kWaves = 2 * OG;
    constexpr int kPieces = StayRead<T>::kPieces, kLoads = kPieces / 4 / kWaves;   // of a wave and step
    constexpr int kStores = OT * 4 * kB / 2;                                       // of a wave and tile
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = wave >> 1, q = lane >> 4, at = lane & 15;
    const int slot = blockIdx.x >> 3, chunk = slot % a.chunks;
    const int64_t tiles = ceil_div(a.n, 16), streams = gridDim.x / a.chunks;
    const int64_t first = (int64_t)(slot / a.chunks) * 8 + (blockIdx.x & 7);
    if (first >= tiles) return;
    const int steps = (a.K + 31) / 32;
    const int m0 = (chunk * OG + group) * OT * 16;

    // steps of this workgroup one after the other; past the last tile the last one again, so that
    // the number of loads under way is always the same.  Lanes past the tile's last atom or (after the last
    // step of K) its last channel read the next one's or, past the buffer's bounds, nothing: no result
    // takes them.
    int offset[kLoads];                    // of a load's lane in its tile
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int load = i * kWaves + wave;                // 64 pieces of one atom
        const int node = load * 64 / kPieces, p = (load * 64 % kPieces + lane) ^ node;
        offset[i] = node * a.K * 16 * kB + p * 16;
    }
    int64_t ask_tile = first;
    int ask_step = 0, ask_place = 0;
    auto ask = [&]() {
        const int64_t n0 = min(ask_tile, tiles - 1) * 16;
        const int rows = (int)min((int64_t)16, a.n - n0);
        const __amdgpu_buffer_rsrc_t xb =
            buffer_rsrc((const float*)((const char*)a.x + n0 * a.K * 16 * kB), rows * a.K * 16 * kB);
        char* to = sh + ask_place * S::kStep + wave * 1024;
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                xb, (__attribute__((address_space(3))) void*)(to + i * kWaves * 1024), 16,
                offset[i] + ask_step * 512 * kB, 0, 0, 0);
        asm volatile("" ::: "memory");
        ask_place = ask_place + 1 == S::kRing ? 0 : ask_place + 1;
        if (++ask_step == steps) ask_step = 0, ask_tile += streams;
    };
#pragma unroll
    for (int i = 0; i < S::kAhead; ++i) ask();

    // degrees of this wave: 1 2 (half 0) or 3 0
    StayWeight<T> w[2][KS][OT];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const __amdgpu_buffer_rsrc_t wb = buffer_rsrc(
            a.weight + (int64_t)(HALF ? 3 - 3 * u : 1 + u) * a.K * a.M, (uint32_t)(a.K * a.M * 4));
        float v[KS][OT][8];
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int o = 0; o < OT; ++o)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int k = s * 32 + 4 * j + q, m = m0 + o * 16 + at;
                    v[s][o][j] = buffer_ld(wb, k < a.K && m < a.M ? (k * a.sk + m * a.sm) * 4 : kMixFar, 0);
                }
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int o = 0; o < OT; ++o) w[u][s][o].set(v[s][o]);
        asm volatile("" ::: "memory");                     // one degree at a time: registers
    }
    const int main = StayRead<T>::first(at, q, HALF), other = StayRead<T>::first(at, q, 1 - HALF);
    char* out = sh + S::kRing * S::kStep + group * S::kOut;
    int place = 0;
    unsigned ends = 0;                     // bit i: a tile ended i steps ago
    for (int64_t tile = first; tile < tiles; tile += streams) {
        v4f acc[8][OT];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int o = 0; o < OT; ++o) acc[i][o] = v4f{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            if (s >= steps) break;
            // this step's loads are in, those of every wave; the step before is read
            constexpr int kMost = std::min(S::kAhead, (63 - (S::kAhead - 1) * kLoads) / kStores);
            stay_wait<(S::kAhead - 1) * kLoads, kStores, kMost>(
                min(__builtin_popcount(ends & ((1u << S::kAhead) - 1)), kMost));
            ends <<= 1;
            __syncthreads();
            ask();
            const char* from = sh + place * S::kStep;
            place = place + 1 == S::kRing ? 0 : place + 1;
            const bool cut = s == steps - 1 && (a.K & 31);
            StayRead<T> x;
            const StayWeight<T>* const ws[2] = {w[0][s], w[1][s]};
            static_for<StayRead<T>::kParts>([&](auto ii) {
                constexpr int P = decltype(ii)::value;
                if constexpr (P > 0) asm volatile("" ::: "memory");
                x.template load<P>(from, main, other);
                if (cut) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (s * 32 + 4 * j + q >= a.K) x.cut(j);
                }
                constexpr int kFrom = StayRead<T>::kFrom[P], kTo = StayRead<T>::kFrom[P + 1];
                stay_products<kFrom, kTo, (HALF ? 7 : 3)>(x, ws, acc);
            });
        }
        ends |= 1;
        // the two waves' components of 16 atoms x 8 outputs together, and out as whole lines
        const int64_t n0 = tile * 16;
        const int rows = (int)min((int64_t)16, a.n - n0);
        const __amdgpu_buffer_rsrc_t yb =
            buffer_rsrc((const float*)((const char*)a.y + n0 * a.M * 16 * kB), rows * a.M * 16 * kB);
#pragma unroll
        for (int o = 0; o < OT; ++o)
#pragma unroll
            for (int rp = 0; rp < 2; ++rp) {
                int mine = (at * 32 + (q * 8 ^ at)) * 16;
                asm volatile("" : "+v"(mine));             // the places are formed again, not kept
                __syncthreads();
#pragma unroll
                for (int rr = 0; rr < 2; ++rr) {
                    // pieces of four components, permuted by the atom's number
                    auto to = [&](int piece) {
                        return reinterpret_cast<float*>(out + (mine ^ (rr * 4 + piece) * 16));
                    };
                    const int r = rp * 2 + rr;
                    to(HALF * 2)[1] = acc[0][o][r];
                    *reinterpret_cast<float2*>(to(HALF * 2) + 2) = make_float2(acc[1][o][r], acc[2][o][r]);
                    *reinterpret_cast<float4*>(to(HALF * 2 + 1)) =
                        make_float4(acc[3][o][r], acc[4][o][r], acc[5][o][r], acc[6][o][r]);
                    to(2 - HALF * 2)[0] = acc[7][o][r];
                }
                __syncthreads();
                constexpr int kUnit = 16 / kB, kPer = 128 / kUnit;     // 16-byte pieces of an atom
#pragma unroll
                for (int i = 0; i < 16 * kPer / 128; ++i) {
                    const int p = i * 128 + (threadIdx.x & 127), node = p / kPer, e = p % kPer * kUnit;
                    const int row = e / 16, m = m0 + o * 16 + (row >> 1) * 4 + rp * 2 + (row & 1);
                    // (every store is issued, those past the end dropped by the buffer's bounds: the
                    // waits count them)
                    const int to = m < a.M ? ((node * a.M + m) * 16 + e % 16) * kB : kMixFar;
                    const float4 u =
                        *reinterpret_cast<const float4*>(out + (node * 32 + (e / 4 ^ node)) * 16);
                    v4u piece;
                    if constexpr (kB == 4) {
                        piece = __builtin_bit_cast(v4u, u);
                    } else {
                        const float4 v = *reinterpret_cast<const float4*>(
                            out + (node * 32 + ((e / 4 + 1) ^ node)) * 16);
                        piece = v4u{bf16_pack(u.x, u.y), bf16_pack(u.z, u.w), bf16_pack(v.x, v.y),
                                    bf16_pack(v.z, v.w)};
                    }
                    __builtin_amdgcn_raw_buffer_store_b128(piece, yb, to, 0, 0);
                }
            }
    }
    // the loads past the last tile, before the LDS that they write goes to another workgroup
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <typename T, int KS, int OT, int OG>
__global__ __launch_bounds__(128 * OG, 2) void mix_stay_kernel(MixArgs a) {
    extern __shared__ __attribute__((aligned(16))) char sh[];
    if (__builtin_amdgcn_readfirstlane(threadIdx.x >> 6) & 1) mix_stay<T, KS, OT, OG, 1>(a, sh);
    else mix_stay<T, KS, OT, OG, 0>(a, sh);
}

// ---------------------------------------------------------------------------
// gW: a workgroup takes 32 CT channels in and 64 out over a range of atoms.  A step is 16 atoms in bf16 (8
// in fp32, whose products run on the fp32 matrix cores, 4 atoms each), features and gradients brought to
// LDS by direct loads while the step before is worked on.  A wave takes four components (two degrees at
// most) and half of the channels in: lane l holds channel l % 16 and atoms l / 16 + 4 j.  part [splits,
// 4, K, M].
// ---------------------------------------------------------------------------
typedef short v4s __attribute__((ext_vector_type(4)));

template <typename T, bool KEPT, int CT>
struct GradShape {
    static constexpr int kB = sizeof(T), kAtoms = kB == 2 || KEPT ? 16 : 8;
    static constexpr int kIn = 32 * CT, kOut = 64;                 // channels
    static constexpr int kXB = KEPT ? 1 : kB;                      // bytes of a value of x
    static constexpr int kX = kAtoms * kIn * 16 * kXB, kG = kAtoms * kOut * 16 * kB;
    static constexpr int kStep = kX + kG, kBytes = 2 * kStep;
    static constexpr int kExps = KEPT ? kAtoms * 2 * CT / 64 + (kAtoms * 2 * CT % 64 != 0) : 0;
};

// Where piece p (16 bytes) of an atom lies in LDS: 16 neighbouring channels' pieces of the same
// components in different banks (its own inverse)
template <int BYTES>
__device__ __forceinline__ int grad_place(int p) {
    return BYTES == 4 ? p ^ (p >> 4 & 3) : BYTES == 2 ? p ^ (p >> 4 & 1) : p;
}

// Four components of a channel and atom
template <typename T>
struct Four;
template <>
struct Four<float> {
    float4 v;
    __device__ __forceinline__ void load(const char* p) { v = *reinterpret_cast<const float4*>(p); }
    __device__ __forceinline__ void zero() { v = make_float4(0, 0, 0, 0); }
    template <int I>
    __device__ __forceinline__ float get() const {
        return I == 0 ? v.x : I == 1 ? v.y : I == 2 ? v.z : v.w;
    }
};
template <>
struct Four<uint16_t> {
    unsigned v[2];
    __device__ __forceinline__ void load(const char* p) {
        const uint2 t = *reinterpret_cast<const uint2*>(p);
        v[0] = t.x, v[1] = t.y;
    }
    __device__ __forceinline__ void decode(unsigned code, float up) {
        const float4 t = ckpt_decode4(code, up);               // exact in bf16
        v[0] = bf16_pack(t.x, t.y), v[1] = bf16_pack(t.z, t.w);
    }
    __device__ __forceinline__ void zero() { v[0] = v[1] = 0; }
};
// acc[k][o] += sum over the step's atoms of component I
template <int I, int CT>
__device__ __forceinline__ void grad_products(const Four<uint16_t> (&x)[CT][4], const Four<uint16_t> (&g)[4][4],
                                              v4f (&acc)[CT][4]) {
    constexpr unsigned kSel = I % 2 ? 0x07060302u : 0x05040100u;
    auto operand = [&](const Four<uint16_t>(&r)[4]) {
        return __builtin_bit_cast(v4s, uint2{__builtin_amdgcn_perm(r[1].v[I / 2], r[0].v[I / 2], kSel),
                                             __builtin_amdgcn_perm(r[3].v[I / 2], r[2].v[I / 2], kSel)});
    };
    v4s f[4];
#pragma unroll
    for (int o = 0; o < 4; ++o) f[o] = operand(g[o]);
#pragma unroll
    for (int k = 0; k < CT; ++k) {
        const v4s e = operand(x[k]);
#pragma unroll
        for (int o = 0; o < 4; ++o)
            acc[k][o] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(e, f[o], acc[k][o], 0, 0, 0);
    }
}
template <int I, int CT>
__device__ __forceinline__ void grad_products(const Four<uint16_t> (&x)[CT][4], const Four<float> (&g)[4][4],
                                              v4f (&acc)[CT][4]) {
    constexpr unsigned kSel = I % 2 ? 0x07060302u : 0x05040100u, kHigh = 0x07060302u;
    v4s e[CT];
#pragma unroll
    for (int k = 0; k < CT; ++k)
        e[k] = __builtin_bit_cast(v4s, uint2{__builtin_amdgcn_perm(x[k][1].v[I / 2], x[k][0].v[I / 2], kSel),
                                             __builtin_amdgcn_perm(x[k][3].v[I / 2], x[k][2].v[I / 2], kSel)});
#pragma unroll
    for (int o = 0; o < 4; ++o) {
        uint2 f[3];
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = g[o][j].template get<I>();
#pragma unroll
        for (int p = 0; p < 3; ++p) {                      // the leading bits, and what is left
            f[p].x = __builtin_amdgcn_perm(__float_as_uint(v[1]), __float_as_uint(v[0]), kHigh);
            f[p].y = __builtin_amdgcn_perm(__float_as_uint(v[3]), __float_as_uint(v[2]), kHigh);
            if (p < 2) {
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] -= __uint_as_float(__float_as_uint(v[j]) & 0xffff0000u);
            }
        }
#pragma unroll
        for (int p = 2; p >= 0; --p)
#pragma unroll
            for (int k = 0; k < CT; ++k)
                acc[k][o] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(
                    e[k], __builtin_bit_cast(v4s, f[p]), acc[k][o], 0, 0, 0);
    }
}
template <int I, int CT>
__device__ __forceinline__ void grad_products(const Four<float> (&x)[CT][2], const Four<float> (&g)[4][2],
                                              v4f (&acc)[CT][4]) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int k = 0; k < CT; ++k)
#pragma unroll
            for (int o = 0; o < 4; ++o)
                acc[k][o] = mfma1(x[k][j].template get<I>(), g[o][j].template get<I>(), acc[k][o]);
}

template <typename T, bool KEPT, int CT>
__global__ __launch_bounds__(512, 2) void mix_weight_kernel(MixArgs a) {
    using S = GradShape<T, KEPT, CT>;
    constexpr int kJ = S::kAtoms / 4, kXPieces = S::kIn * S::kXB, kGPieces = S::kOut * S::kB;   // of an atom
    extern __shared__ __attribute__((aligned(16))) char sh[];
    int64_t split;
    int which;
    if (!mix_place(a.splits, a.tiles * a.chunks, split, which)) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int quarter = wave & 3, side = wave >> 2, q = lane >> 4, at = lane & 15;
    const int c0 = which % a.tiles * S::kIn, o0 = which / a.tiles * S::kOut;
    const int exps = ckpt_blocks(a.K);
    const int64_t begin = split * a.per_split * S::kAtoms;
    const int64_t end = min(a.n, begin + (int64_t)a.per_split * S::kAtoms);

    // channels past K or M read what lies there (the next atom's, past the buffer nothing): no result
    // that is stored takes them
    int code[S::kExps ? S::kExps : 1];
    auto ask = [&](int64_t n0, char* to) {
        const int rows = (int)min((int64_t)S::kAtoms, a.n - n0);
        const void* xs = KEPT ? (const void*)(a.codes + n0 * a.K * 16)
                              : (const void*)((const char*)a.x + n0 * a.K * 16 * S::kB);
        const __amdgpu_buffer_rsrc_t xb = buffer_rsrc((const float*)xs, rows * a.K * 16 * S::kXB);
        const __amdgpu_buffer_rsrc_t gb = buffer_rsrc(
            (const float*)((const char*)a.g + n0 * a.M * 16 * S::kB), rows * a.M * 16 * S::kB);
#pragma unroll
        for (int i = 0; i < S::kX / 8192; ++i) {
            const int at0 = (i * 8 + wave) * 64 + lane;            // place in the step
            const int off = (at0 / kXPieces * a.K + c0) * 16 * S::kXB +
                            grad_place<S::kXB>(at0 % kXPieces) * 16;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                xb, (__attribute__((address_space(3))) void*)(to + (i * 8 + wave) * 1024), 16, off, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < S::kG / 8192; ++i) {
            const int at0 = (i * 8 + wave) * 64 + lane;
            const int off = (at0 / kGPieces * a.M + o0) * 16 * S::kB +
                            grad_place<S::kB>(at0 % kGPieces) * 16;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                gb, (__attribute__((address_space(3))) void*)(to + S::kX + (i * 8 + wave) * 1024), 16, off,
                0, 0, 0);
        }
        if constexpr (KEPT) {
            // exponent e of the wave's 2 CT blocks of atom n in lane (n 2 CT + e) % 64 of a register
            const __amdgpu_buffer_rsrc_t eb = buffer_rsrc((const float*)(a.exps + n0 * exps), rows * exps);
#pragma unroll
            for (int i = 0; i < S::kExps; ++i) {
                const int e = i * 64 + lane;
                code[i] = __builtin_amdgcn_raw_buffer_load_b8(
                    eb, e / (2 * CT) * exps + (c0 + side * CT * 16) / 8 + e % (2 * CT), 0, 0);
            }
        }
        asm volatile("" ::: "memory");
    };

    v4f acc[2][CT][4];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < CT; ++k)
#pragma unroll
            for (int o = 0; o < 4; ++o) acc[i][k][o] = v4f{0, 0, 0, 0};
    if (begin < end) ask(begin, sh);
    int turn = 0;
    for (int64_t n0 = begin; n0 < end; n0 += S::kAtoms, turn ^= 1) {
        // this step's loads are in, those of every wave; the step before is read
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        int now[S::kExps ? S::kExps : 1];
        if constexpr (KEPT) {
#pragma unroll
            for (int i = 0; i < S::kExps; ++i) now[i] = code[i];
        }
        __syncthreads();
        if (n0 + S::kAtoms < end) ask(n0 + S::kAtoms, sh + (turn ^ 1) * S::kStep);
        const char* from = sh + turn * S::kStep;
        Four<typename std::conditional<KEPT, uint16_t, T>::type> x[CT][kJ];
        Four<T> g[4][kJ];
#pragma unroll
        for (int k = 0; k < CT; ++k)
#pragma unroll
            for (int j = 0; j < kJ; ++j) {
                const int c = (side * CT + k) * 16 + at, n = 4 * j + q;
                if constexpr (KEPT) {
                    const int e = (4 * j * 2 * CT) % 64 + q * 2 * CT + 2 * k + (at >> 3);
                    const int exponent = __builtin_amdgcn_ds_bpermute(e * 4, now[4 * j * 2 * CT / 64]);
                    x[k][j].decode(*reinterpret_cast<const unsigned*>(from + (n * S::kIn + c) * 16 + quarter * 4),
                                   ckpt_up(exponent));
                } else {
                    const int p = c * S::kB + quarter * S::kB / 4;
                    x[k][j].load(from + (n * kXPieces + grad_place<S::kB>(p)) * 16 +
                                 (S::kB == 2 ? quarter % 2 * 8 : 0));
                }
            }
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int j = 0; j < kJ; ++j) {
                const int p = (k * 16 + at) * S::kB + quarter * S::kB / 4;
                g[k][j].load(from + S::kX + ((4 * j + q) * kGPieces + grad_place<S::kB>(p)) * 16 +
                             (S::kB == 2 ? quarter % 2 * 8 : 0));
            }
        if (n0 + S::kAtoms > a.n) {                        // atoms past the last add nothing
#pragma unroll
            for (int j = 0; j < kJ; ++j)
                if (n0 + 4 * j + q >= a.n) {
#pragma unroll
                    for (int k = 0; k < CT; ++k) x[k][j].zero();
#pragma unroll
                    for (int k = 0; k < 4; ++k) g[k][j].zero();
                }
        }
        grad_products<0>(x, g, acc[0]);
        grad_products<1>(x, g, acc[1]);
        grad_products<2>(x, g, acc[1]);
        grad_products<3>(x, g, acc[1]);
    }
    // degrees of the quarters: 0 1 | 2 2 | 2 3 | 3 3.  The third hands its sums to the others.
    v4f* give = reinterpret_cast<v4f*>(sh) + side * 2 * CT * 4 * 64 + lane;
    __syncthreads();
    if (quarter == 2) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int k = 0; k < CT; ++k)
#pragma unroll
                for (int o = 0; o < 4; ++o) give[((i * CT + k) * 4 + o) * 64] = acc[i][k][o];
    }
    __syncthreads();
    if (quarter == 2) return;
#pragma unroll
    for (int k = 0; k < CT; ++k)
#pragma unroll
        for (int o = 0; o < 4; ++o) {
            v4f u = acc[0][k][o], v = acc[1][k][o];
            if (quarter) u += v + give[((quarter / 2 * CT + k) * 4 + o) * 64];
            const int l = quarter ? quarter / 2 + 2 : 0;
            float* part = a.part + (split * 4 + l) * a.K * a.M;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int c = c0 + (side * CT + k) * 16 + 4 * q + r, m = o0 + o * 16 + at;
                if (c >= a.K || m >= a.M) continue;
                part[(int64_t)c * a.M + m] = u[r];
                if (!quarter) part[((int64_t)a.K + c) * a.M + m] = v[r];
            }
        }
}

// Sums of part over the splits: 64 columns of four a workgroup, four threads a column
__global__ __launch_bounds__(256) void mix_weight_sum_kernel(const float* __restrict__ part, int splits,
                                                             int64_t cols, float* __restrict__ out) {
    __shared__ float4 sh[4][64];
    const int lane = threadIdx.x & 63, k = threadIdx.x >> 6;
    const int64_t col = ((int64_t)blockIdx.x * 64 + lane) * 4;
    float4 s = make_float4(0, 0, 0, 0);
    if (col < cols) {
#pragma unroll 8
        for (int r = k; r < splits; r += 4) {
            const float4 v = *reinterpret_cast<const float4*>(part + r * cols + col);
            s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
        }
    }
    sh[k][lane] = s;
    __syncthreads();
    if (k || col >= cols) return;
#pragma unroll
    for (int i = 1; i < 4; ++i) {
        const float4 v = sh[i][lane];
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    *reinterpret_cast<float4*>(out + col) = s;
}

static bool mix_shape_ok(int64_t N, int C, int O, int dtype) {
    return N >= 0 && N < ((int64_t)1 << 31) && C >= 1 && C <= kMixMaxC && O >= 1 && O <= kMixMaxC &&
           (dtype == 0 || dtype == 1);
}

template <typename T>
static void mix_tiles(int M, MixArgs& a) {
    constexpr int kOT = MixTile<T>::kOT;
    a.chunks = (M + kOT * 16 - 1) / (kOT * 16);
    a.tiles = a.chunks * kOT;
}
template <typename T>
static size_t mix_bytes(int K, int M) {
    if (K <= kStayMost<T>) return 16;
    MixArgs a{};
    mix_tiles<T>(M, a);
    return (size_t)((K + 31) / 32) * 4 * a.tiles * MixTile<T>::kPW * 64 * 16;
}

// The general kernel's launch: at most 2^22 workgroups (and the last 8 units' of a chunk) of 512 threads.  Beyond
// that features and results do not fit a card's memory.
template <typename T>
static bool mix_launch_ok(int64_t n, int K, int M) {
    MixArgs a{};
    mix_tiles<T>(M, a);
    return K <= kStayMost<T> || n * a.chunks <= (int64_t)1 << 27;
}

// More than 64 KB of LDS for a kernel, allowed once on each device
static int mix_allow_lds(const void* kernel, int bytes, std::atomic<uint64_t>& allowed) {
    int device = 0;
    hipError_t rc = hipGetDevice(&device);
    if (rc != hipSuccess) return (int)rc;
    const uint64_t bit = device < 64 ? (uint64_t)1 << device : 0;
    if (allowed.load(std::memory_order_relaxed) & bit) return 0;
    rc = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (rc != hipSuccess) return (int)rc;
    allowed.fetch_or(bit, std::memory_order_relaxed);
    return 0;
}

template <typename T, int KS, int OT, int OG>
static int stay_launch(MixArgs a, hipStream_t s) {
    constexpr int kBytes = StayShape<T>::bytes(OG), kPer = std::min(8 / (2 * OG), 163840 / kBytes);
    auto kernel = mix_stay_kernel<T, KS, OT, OG>;
    static std::atomic<uint64_t> allowed{0};
    if (const int rc = mix_allow_lds((const void*)kernel, kBytes, allowed)) return rc;
    a.chunks = (a.M + OG * OT * 16 - 1) / (OG * OT * 16);
    const int64_t tiles = ceil_div(a.n, 16), most = std::max(1, 32 * kPer / a.chunks);
    const int64_t streams = 8 * std::min(most, ceil_div(tiles, 8));
    kernel<<<(unsigned)(streams * a.chunks), 128 * OG, kBytes, s>>>(a);
    return (int)hipGetLastError();
}
template <typename T, int KS, int OT>
static int stay_groups(const MixArgs& a, hipStream_t s) {
    if (a.M <= OT * 16) return stay_launch<T, KS, OT, 1>(a, s);
    return stay_launch<T, KS, OT, 2>(a, s);
}
template <typename T>
static int stay_run(const MixArgs& a, hipStream_t s) {
    if constexpr (sizeof(T) == 2) {
        if (a.K > 128) return stay_groups<T, 8, 1>(a, s);
        if (a.K > 64) return stay_groups<T, 4, 2>(a, s);
    }
    return stay_groups<T, 2, 2>(a, s);
}

template <typename T>
static int mix_run(MixArgs a, void* ws, hipStream_t s) {
    if (a.K <= kStayMost<T>) return stay_run<T>(a, s);
    using S = MixTile<T>;
    static std::atomic<uint64_t> allowed{0};
    if (const int rc = mix_allow_lds((const void*)&mix_kernel<T>, S::kBytes, allowed)) return rc;
    mix_tiles<T>(a.M, a);
    const int total = (a.K + 31) / 32 * 4 * a.tiles * 64;
    mix_pack_kernel<S::kPW><<<(total + 255) / 256, 256, 0, s>>>(a.weight, (v4u*)ws, a.K, a.M, a.sk,
                                                               a.sm, a.tiles, total);
    a.w = (const v4u*)ws;
    a.units = ceil_div(a.n, 16 * S::kNG);
    mix_kernel<T><<<mix_grid(a.units, a.chunks), 256 * S::kNG, S::kBytes, s>>>(a);
    return (int)hipGetLastError();
}

// Most ranges of atoms of gW: a workgroup for each compute unit, of one or two steps at least, 64 MB of
// partial sums at most
static int mix_splits(int64_t N, int C, int O) {
    const int64_t tiles = ceil_div(C, C > 64 ? 128 : 64) * ceil_div(O, 64);
    const int64_t most = std::max<int64_t>(1, ((int64_t)1 << 24) / ((int64_t)4 * C * O));
    return (int)std::max<int64_t>(1, std::min({ceil_div(256, tiles), ceil_div(N, 16), most}));
}

template <typename T, bool KEPT, int CT>
static int mix_weight_run(MixArgs& a, hipStream_t s) {
    using S = GradShape<T, KEPT, CT>;
    auto kernel = mix_weight_kernel<T, KEPT, CT>;
    static std::atomic<uint64_t> allowed{0};
    if (const int rc = mix_allow_lds((const void*)kernel, S::kBytes, allowed)) return rc;
    a.tiles = (a.K + S::kIn - 1) / S::kIn;
    a.chunks = (a.M + S::kOut - 1) / S::kOut;
    a.splits = std::min(a.splits, (int)ceil_div(256, a.tiles * a.chunks));
    a.per_split = (int)ceil_div(ceil_div(a.n, S::kAtoms), a.splits);
    kernel<<<mix_grid(a.splits, a.tiles * a.chunks), 512, S::kBytes, s>>>(a);
    return (int)hipGetLastError();
}
template <typename T>
static int mix_weight_pick(MixArgs& a, hipStream_t s) {
    if (a.x) return mix_weight_run<T, false, 2>(a, s);
    // 128 channels in for 64 out where g would else be read once more (50,000 x 128 x 128: 94 against 106 us)
    if constexpr (sizeof(T) == 2)
        if (a.K > 64) return mix_weight_run<T, true, 4>(a, s);
    return mix_weight_run<T, true, 2>(a, s);
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
    const int K = transposed ? O : C, M = transposed ? C : O;
    if (!(dtype == 0 ? mix_launch_ok<float>(N, K, M) : mix_launch_ok<uint16_t>(N, K, M))) return BM_ERR_ARG;
    if (N == 0) return BM_OK;
    if (workspace_bytes < batteries_channel_mixing_workspace_bytes(C, O, transposed, dtype) || !workspace)
        return BM_ERR_WORKSPACE;
    MixArgs a{};
    a.x = x; a.y = y; a.n = N; a.K = K; a.M = M;
    a.weight = weight; a.sk = transposed ? 1 : O; a.sm = transposed ? O : 1;
    return dtype == 0 ? mix_run<float>(a, workspace, stream) : mix_run<uint16_t>(a, workspace, stream);
}

extern "C" size_t batteries_channel_mixing_weight_grad_workspace_bytes(int64_t N, int C, int O) {
    if (!mix_shape_ok(N, C, O, 0)) return 0;
    return (size_t)mix_splits(N, C, O) * 4 * C * O * sizeof(float);
}

extern "C" int batteries_channel_mixing_weight_grad(const void* x, const uint8_t* codes,
                                                    const uint8_t* exps, const void* g, float* gweight,
                                                    int64_t N, int C, int O, int dtype, void* workspace,
                                                    size_t workspace_bytes, hipStream_t stream) {
    if (!mix_shape_ok(N, C, O, dtype) || !gweight || (N > 0 && (!g || (!x && (!codes || !exps)))))
        return BM_ERR_ARG;
    if (!aligned_to({x, g, codes, gweight, workspace}, 16)) return BM_ERR_ARG;
    if (workspace_bytes < batteries_channel_mixing_weight_grad_workspace_bytes(N, C, O) || !workspace)
        return BM_ERR_WORKSPACE;
    MixArgs a{};
    a.x = x; a.codes = codes; a.exps = exps; a.g = g; a.part = (float*)workspace; a.n = N; a.K = C;
    a.M = O; a.splits = mix_splits(N, C, O);
    if (N > 0) {
        const int rc = dtype == 0 ? mix_weight_pick<float>(a, stream) : mix_weight_pick<uint16_t>(a, stream);
        if (rc) return rc;
    }
    const int64_t cols = (int64_t)4 * C * O;
    mix_weight_sum_kernel<<<(unsigned)ceil_div(cols, 256), 256, 0, stream>>>(
        a.part, N > 0 ? a.splits : 0, cols, gweight);
    return (int)hipGetLastError();
}
