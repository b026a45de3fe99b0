// Softmax attention of every row (destination) over its neighbours (sources) on the edges of a
// graph, forward (no reference counterpart: the reference sums its messages,
// src/message_passing/fused_message_passing.cu).
//
//   x_eh = scale <q[i,h], k[j,g]> + b[e,h]      edge e: j -> i, g = h / (H / H_kv)
//   p_eh = exp(x_eh - m_ih) / l_ih              m, l: maximum and sum of exponentials over
//                                               the edges of row i
//   o_ih = sum_e p_eh v[j,g]
//
// An edge whose b or x is -inf is left out; a row without an edge gives o = 0.
//
// One pass over a tile's columns (attention.h) with a running reference (the maximum, or up to 8
// below it) in m's place and the sum relative to it, which are kept for the backward.  x is formed in natural units and the maximum taken off before the factor
// log2 e, so that a bias of the type's lowest value does not become infinite.
#include "attention.h"

namespace bmhip {

struct AttnFwd {
    AttnSide side;
    const void *q, *k, *v;
    EdgeBias bias;
    void* out;
    float *stats;                          // [n_dst, H, 2]: reference and sum
    float *part_o, *part_ml;               // [parts, H, 16, Dv], [parts, H, 16, 2]
    uint32_t qs, ks, vs;                   // rows' strides in bytes
    int H, group, Dk, Dv;
    float scale;
};

// An item's rows one after the other, each over its own edges alone: infinities or NaN among the
// values.
template <typename T>
__device__ __forceinline__ void attn_fwd_rows(const AttnFwd& a, int item, int h, int tile,
                                              int part_at) {
    constexpr float kInf = __builtin_inff();
    const int kv = h / a.group;
    for (int r = 0; r < kAttnRows; ++r) {
        const int row = a.side.rows[tile * kAttnRows + r];
        if (row < 0) continue;
        const T* q = row_of<T>(a.q, row, a.qs) + (int64_t)h * a.Dk;
        float m = -kInf, l = 0.0f, o[4] = {0, 0, 0, 0};
        each_edge(a.side, item, r, [&](int e, int col) {
            const float b = a.bias.value ? a.bias.at(e, h) : 0.0f;
            const T* k = row_of<T>(a.k, col, a.ks) + (int64_t)kv * a.Dk;
            float s = 0.0f;
            for (int d = threadIdx.x; d < a.Dk; d += 64) s = fmaf(attn_f32(q[d]), attn_f32(k[d]), s);
            const float x = fmaf(attn_wave_sum(s), a.scale, b);
            if (b == -kInf || x == -kInf) return;
            const float top = fmaxf(m, x), f = attn_exp(m - top);
            const float p = attn_exp(x - top);
            m = top;
            l = l * f + p;
#pragma unroll
            for (int c = 0; c < 4; ++c) o[c] *= f;
            add_row<T>(o, p, row_of<T>(a.v, col, a.vs) + (int64_t)kv * a.Dv, a.Dv);
        });
        const int64_t part = ((int64_t)part_at * a.H + h) * kAttnRows + r;
        const int64_t at = (int64_t)row * a.H + h;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int d = c * 64 + threadIdx.x;
            if (d >= a.Dv) continue;
            if (part_at >= 0) a.part_o[part * a.Dv + d] = o[c];
            else attn_st((T*)a.out + at * a.Dv + d, o[c] * inv);
        }
        float* ml = part_at >= 0 ? a.part_ml + part * 2 : a.stats ? a.stats + at * 2 : nullptr;
        if (ml && threadIdx.x == 0) {
            ml[0] = m;
            ml[1] = l;
        }
    }
}

// A step's loads are in flight over most of the step before: k goes to LDS while the softmax and
// the second product of the step before run, v to registers over the first product and the
// softmax.  All reads from LDS stand before the loads to LDS.
//
// Measured, atoms with 28 neighbours (GB/s of q, k, v and o once):
//   5000, 8 heads of 128, f32           51 us   1.7 TB/s   one round of waves; a tile has 4.7
//                                                          chunks of columns, the longest 7
//   20,011, 8 on 2 heads of 128, bf16   64 us              issue: waves wait for it 36 % of their
//                                                          time, 31 % for memory
//   50,000, 8 heads of 256, bf16       353 us   2.5 TB/s   1.17 GB from HBM and Infinity Cache
//   5000, random, 4 heads of 24 by 256 106 us   6.3 TB/s   of rows from Infinity Cache
// Rows of k loaded straight to registers in row form, where 16 lanes ask for 16 cache lines, made an
// earlier form take 79 us at the first size instead of 65.
// Registers for two waves a SIMD at least, unless the tiles of k and v in f32 need more than that
// leaves (LDS holds 7 waves a CU at 256 by 256, 12 at 128 by 128): 20,000 atoms, 8 heads of 256 in bf16 100 us against 122 without the bound, 5000 in f32
// 66 us with it against 64.
template <typename T, int KP, int VP, bool FULL, bool BIAS, bool WIDE>
__global__ __launch_bounds__(64, (KP + VP) * sizeof(T) <= 1536 ? 2 : 1) void attn_fwd_kernel(
    AttnFwd a) {
    constexpr int kT = Attn<T>::kTiles;
    constexpr float kInf = __builtin_inff(), kSlack = 8.0f;
    using Rows = RowTile<T, KP, kT>;
    __shared__ __attribute__((aligned(1024))) char k_lds[
        Rows::kBytes > OutTile<T, VP>::kBytes ? Rows::kBytes : OutTile<T, VP>::kBytes];
    __shared__ float b_lds[BIAS ? kTileEdges + 1 : 1];
    int item, h;
    if (!attn_unit(blockIdx.x, a.side.n_items, a.H, item, h)) return;
    const int lane = threadIdx.x, n = lane & 15, g = lane >> 4;
    const int kv = uniform_quotient(h, a.group);
    const Item it(a.side, item, lane);
    const int row = it.row, steps = it.steps(kT);
    const T* kbase = (const T*)a.k + (int64_t)kv * a.Dk;
    const T* vbase = (const T*)a.v + (int64_t)kv * a.Dv;
    v4f acc[ColFrag<T, VP>::kAcc];
    float m = -kInf, l = 0.0f;
#pragma unroll
    for (int i = 0; i < ColFrag<T, VP>::kAcc; ++i) acc[i] = v4f{0, 0, 0, 0};
    {
        int done = 0;                      // row n's edges of earlier steps
        ColFrag<T, VP> vf;
        uint32_t mask = 0;
        int ids = 0;
        const Steps<kT> step(a.side, it, lane);
        // v of step i, whose columns `ids` holds; then those of the next step
        auto load_v = [&](int i) {
            const StepCols<T> cols(ids, g);
            ids = step.ids(i + 1);
            load_fence();
            vf.load([&](int j) { return row_of<T>(vbase, cols.col[j], a.vs); }, a.Dv, n);
            load_fence();
        };
        if (steps > 0) {
            ids = step.ids(0);
            mask = step.mask(0);
        }
        RowFrag<T, KP> q;
        // (a slot past the last row computes with row 0 and stores nothing)
        q.template load<FULL>(row_of<T>(a.q, max(row, 0), a.qs) + (int64_t)h * a.Dk, a.Dk, g);
        if (steps > 0) {
            Rows::template fill<FULL, WIDE>(k_lds, ids, kbase, a.ks, a.Dk, lane);
            load_v(0);
        }
        if constexpr (BIAS) {
            auto keep = [&](int i, int, float b, int) { b_lds[i] = b; };
            if (a.bias.eid)
                it.each<float>(a.side, lane, [&](int e) { return a.bias.at(e, h); }, keep);
            else
                it.each<float>(a.side, lane, [&](int e) {
                    return a.bias.value[(int64_t)e * a.bias.edge_step + h * a.bias.head_step];
                }, keep);
        }
        for (int i = 0; i < steps; ++i) {
            float b[4 * kT], x[4 * kT];
            bool on[4 * kT];
            Rows::template arrived<ColFrag<T, VP>::kLoads>();
#pragma unroll
            for (int t = 0; t < kT; ++t) {
                RowFrag<T, KP> kf;
                Rows::template read<FULL>(kf, k_lds, t, a.Dk, n, g);
                const v4f s = row_product<T, KP>(kf, q);
#pragma unroll
                for (int r = 0; r < 4; ++r) x[4 * t + r] = s[r];
                // two tiles' fragments at a time would leave no room for a second wave
                if (kT > 1 && KP + VP > 256) asm volatile("" : "+v"(x[4 * t]) : : "memory");
            }
#pragma unroll
            for (int t = 0; t < kT; ++t) {
                int at[4];
                edge_places(mask, t, g, it.off + done, at, on + 4 * t);
#pragma unroll
                for (int r = 0; r < 4; ++r) b[4 * t + r] = BIAS ? b_lds[at[r]] : 0.0f;
            }
            Rows::reads_done();
            Rows::template fill<FULL, WIDE>(k_lds, ids, kbase, a.ks, a.Dk, lane);
            float top = m;
#pragma unroll
            for (int j = 0; j < 4 * kT; ++j) {
                // (b = -inf and a product that is infinite or NaN: the sums will tell)
                x[j] = on[j] ? fmaf(x[j], a.scale, b[j]) : -kInf;
                top = fmaxf(top, x[j]);
            }
            top = max_over_groups(top);
            // The sums are scaled to a new reference only where the maximum has left the old one by
            // more than kSlack: p then stays below e^kSlack, which the fp32 sums have room for.
            if (__any(top > m + kSlack)) {
                const float to = top > m + kSlack ? top : m;
                const float f = m == -kInf ? 0.0f : attn_exp(m - to);
                l *= f;
#pragma unroll
                for (int j = 0; j < ColFrag<T, VP>::kAcc; ++j) acc[j] *= f;
                m = to;
            }
            const float ref = m == -kInf ? 0.0f : m;
            float p[4 * kT];
#pragma unroll
            for (int j = 0; j < 4 * kT; ++j) {
                p[j] = attn_exp(x[j] - ref);
                l += p[j];
            }
            vf.mac(p, acc);
            done += __popc(mask);
            mask = step.mask(i + 1);
            load_v(i + 1);
        }
    }
    // (the last fill of k, which nothing read, must not land in the results)
    Rows::template arrived<0>();
    l = sum_over_groups(l);
    if (__builtin_expect(any_not_finite<ColFrag<T, VP>::kAcc>(acc), 0)) {
        attn_fwd_rows<T>(a, item, h, it.tile, it.part);
        return;
    }
    if (it.part >= 0) {
        if (row < 0) return;
        const int64_t at = ((int64_t)it.part * a.H + h) * kAttnRows + n;
        store_part<T, VP>(a.part_o + at * a.Dv, acc, 1.0f, a.Dv, g);
        if (g == 0) {
            a.part_ml[at * 2] = m;
            a.part_ml[at * 2 + 1] = l;
        }
        return;
    }
    if (a.stats && g == 0 && row >= 0)
        *reinterpret_cast<float2*>(a.stats + ((int64_t)row * a.H + h) * 2) = make_float2(m, l);
    // l is 0 only without an edge; a NaN stays one
    OutTile<T, VP>::store(k_lds, (T*)a.out + (int64_t)h * a.Dv, (int64_t)a.H * a.Dv, row, acc,
                          l == 0.0f ? 0.0f : 1.0f / l, a.Dv, lane);
}

// Joins the parts of a cut tile, row by row: workgroup p of the parts takes rows p, p + parts of
// its tile, ...; groups of D / 4 lanes take the parts in turn, a lane four components.  Latency:
// 9.0 us for 8 rows of 25,000 edges, 4 heads of 128 components.
template <typename T>
__global__ __launch_bounds__(1024) void attn_join_kernel(AttnFwd a) {
    constexpr float kInf = __builtin_inff();
    __shared__ float sm[16], sl[16], so[1024][4];
    const int h = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int wide = a.Dv / 4, groups = 1024 / wide, k = threadIdx.x / wide, c4 = threadIdx.x % wide;
    int first, parts;
    const int tile = tile_of_part(a.side, blockIdx.x, first, parts);
    for (int slot = (int)blockIdx.x - first; slot < kAttnRows; slot += parts) {
        const int row = a.side.rows[tile * kAttnRows + slot];
        if (row < 0) continue;
        auto at = [&](int p) { return ((int64_t)(first + p) * a.H + h) * kAttnRows + slot; };
        float m = -kInf, l = 0.0f;
        for (int p = threadIdx.x; p < parts; p += 1024) m = fmaxf(m, a.part_ml[at(p) * 2]);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
        __syncthreads();
        if (lane == 0) sm[w] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; ++i) m = fmaxf(m, sm[i]);
        const float ref = m == -kInf ? 0.0f : m;
        for (int p = threadIdx.x; p < parts; p += 1024) {
            const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + at(p) * 2);
            l = fmaf(ml.y, attn_exp(ml.x - ref), l);
        }
        l = attn_wave_sum(l);
        if (lane == 0) sl[w] = l;
        float o[4] = {0, 0, 0, 0};
        if (k < groups) {
#pragma unroll 4
            for (int p = k; p < parts; p += groups) {
                // a part without an edge of this row holds zeros, and the factor 0
                const float f = attn_exp(a.part_ml[at(p) * 2] - ref);
                const float4 x = *reinterpret_cast<const float4*>(a.part_o + at(p) * a.Dv + 4 * c4);
                o[0] = fmaf(x.x, f, o[0]);
                o[1] = fmaf(x.y, f, o[1]);
                o[2] = fmaf(x.z, f, o[2]);
                o[3] = fmaf(x.w, f, o[3]);
            }
        }
        *reinterpret_cast<float4*>(so[threadIdx.x]) = make_float4(o[0], o[1], o[2], o[3]);
        __syncthreads();
        if (k != 0) continue;
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) l += sl[i];
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        for (int i = 1; i < groups; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(so[i * wide + c4]);
            o[0] += x.x;
            o[1] += x.y;
            o[2] += x.z;
            o[3] += x.w;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) o[c] *= inv;
        const int64_t to = (int64_t)row * a.H + h;
        attn_store_w<4>((T*)a.out + to * a.Dv + 4 * c4, o);
        if (a.stats && threadIdx.x == 0) {
            a.stats[to * 2] = m;
            a.stats[to * 2 + 1] = l;
        }
    }
}

template <typename T, int KP, int VP>
static void attn_fwd_launch(const AttnFwd& a, bool wide, hipStream_t s) {
    const unsigned grid = attn_grid(a.side.n_items, a.H);
    const bool full = a.Dk == KP;
    if (wide && a.bias.value) attn_fwd_kernel<T, KP, VP, false, true, true><<<grid, 64, 0, s>>>(a);
    else if (wide) attn_fwd_kernel<T, KP, VP, false, false, true><<<grid, 64, 0, s>>>(a);
    else if (a.bias.value && full) attn_fwd_kernel<T, KP, VP, true, true, false><<<grid, 64, 0, s>>>(a);
    else if (a.bias.value) attn_fwd_kernel<T, KP, VP, false, true, false><<<grid, 64, 0, s>>>(a);
    else if (full) attn_fwd_kernel<T, KP, VP, true, false, false><<<grid, 64, 0, s>>>(a);
    else attn_fwd_kernel<T, KP, VP, false, false, false><<<grid, 64, 0, s>>>(a);
}
template <typename T, int KP>
static void attn_fwd_pick_v(const AttnFwd& a, bool wide, hipStream_t s) {
    if (a.Dv <= 64) attn_fwd_launch<T, KP, 64>(a, wide, s);
    else if (a.Dv <= 128) attn_fwd_launch<T, KP, 128>(a, wide, s);
    else attn_fwd_launch<T, KP, 256>(a, wide, s);
}
template <typename T>
static void attn_fwd_run(const AttnFwd& a, bool wide, int parts, hipStream_t s) {
    if (a.Dk <= 64) attn_fwd_pick_v<T, 64>(a, wide, s);
    else if (a.Dk <= 128) attn_fwd_pick_v<T, 128>(a, wide, s);
    else attn_fwd_pick_v<T, 256>(a, wide, s);
    if (parts)
        attn_join_kernel<T><<<dim3((unsigned)parts, (unsigned)a.H), 1024, 0, s>>>(a);
}

}  // namespace bmhip

using namespace bmhip;

// in [E, H] (row edge_id e) <-> out [H, E]: 256 edges and up to 16 heads a workgroup, through LDS,
// so that both sides are contiguous.  A thread takes up to 4 heads of an edge, 16 bytes where H
// allows.  Memory bound; when to take it is the caller's choice (binding_block.cpp measures both).
template <bool TO_HEADS>
__global__ __launch_bounds__(256) void attn_edges_kernel(const float* __restrict__ in,
                                                         const int* __restrict__ eid,
                                                         float* __restrict__ out, int64_t edges,
                                                         int H) {
    __shared__ float t[16][257];
    const int64_t e0 = (int64_t)blockIdx.x * 256;
    const int h0 = blockIdx.y * 16, n = (int)min((int64_t)256, edges - e0), w = min(16, H - h0);
    const int groups = w <= 4 ? 1 : w <= 8 ? 2 : 4, g = threadIdx.x & (groups - 1);
    const int per = 256 / groups, h = 4 * g, nh = min(4, w - h);
    const bool vec = (H & 3) == 0;
    auto rows = [&]() {
        for (int k = 0; k < groups; ++k) {
            const int e = k * per + threadIdx.x / groups;
            if (e >= n || nh <= 0) continue;
            const int64_t at = (eid ? (int64_t)eid[e0 + e] : e0 + e) * H + h0 + h;
            if (TO_HEADS) {
                float4 v = make_float4(0, 0, 0, 0);
                if (vec) {
                    v = *reinterpret_cast<const float4*>(in + at);
                } else {
                    v.x = in[at];
                    if (nh > 1) v.y = in[at + 1];
                    if (nh > 2) v.z = in[at + 2];
                    if (nh > 3) v.w = in[at + 3];
                }
                t[h][e] = v.x;
                t[h + 1][e] = v.y;
                t[h + 2][e] = v.z;
                t[h + 3][e] = v.w;
            } else {
                const float4 v = make_float4(t[h][e], t[h + 1][e], t[h + 2][e], t[h + 3][e]);
                if (vec) {
                    *reinterpret_cast<float4*>(out + at) = v;
                } else {
                    out[at] = v.x;
                    if (nh > 1) out[at + 1] = v.y;
                    if (nh > 2) out[at + 2] = v.z;
                    if (nh > 3) out[at + 3] = v.w;
                }
            }
        }
    };
    auto cols = [&]() {
        const int e = threadIdx.x;
        if (e >= n) return;
#pragma unroll 4
        for (int i = 0; i < w; ++i) {
            const int64_t at = (int64_t)(h0 + i) * edges + e0 + e;
            if (TO_HEADS) out[at] = t[i][e];
            else t[i][e] = in[at];
        }
    };
    if (TO_HEADS) rows(); else cols();
    __syncthreads();
    if (TO_HEADS) cols(); else rows();
}

// Heads of any size and strides <-> dense rows of heads padded with zeros to whole 16-byte pieces,
// up to four matrices a launch (blockIdx.y).  Packing: a thread a piece; cutting: an element.
// Memory bound on large inputs, a launch on small ones: a training step of 725 atoms with one head
// of 15 by 17 takes 62 us (46 at 16 by 16, where nothing is packed; 127 with a fill and a copy for
// every matrix).
struct AttnPacks {
    batmobile_attention_pack m[4];
};

template <typename T, bool CUT>
__global__ __launch_bounds__(256) void attn_pack_kernel(AttnPacks all) {
    constexpr int kE = 16 / (int)sizeof(T);
    const batmobile_attention_pack& a = all.m[blockIdx.y];
    const uint32_t Dp = (uint32_t)(a.D + kE - 1) / kE * kE;
    const int64_t step = (int64_t)gridDim.x * 256, i0 = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (CUT) {
        const T* in = (const T*)a.in;
        T* out = (T*)a.out;
        const int64_t n = a.rows * a.heads * a.D;
        for (int64_t i = i0; i < n; i += step) {
            const int64_t rh = i / a.D;
            out[i] = in[rh * Dp + (i - rh * a.D)];
        }
        return;
    }
    const uint32_t pieces = Dp / kE;
    const int64_t n = a.rows * a.heads * pieces;
    for (int64_t i = i0; i < n; i += step) {
        const int64_t rh = i / pieces;
        const int d0 = (int)(i - rh * pieces) * kE;
        const int64_t row = rh / a.heads, head = rh - row * a.heads;
        const T* in = (const T*)a.in + row * a.row_stride + head * a.head_stride;
        T v[kE];
#pragma unroll
        for (int k = 0; k < kE; ++k) v[k] = d0 + k < a.D ? in[(d0 + k) * a.step] : (T)0;
        v4u w;
        __builtin_memcpy(&w, v, 16);
        *reinterpret_cast<v4u*>((T*)a.out + i * kE) = w;
    }
}

extern "C" int batteries_attention_pack(const batmobile_attention_pack* packs, int count,
                                        int dtype, int cut, hipStream_t stream) {
    if (count < 0 || count > 4 || (count > 0 && !packs) || (dtype != 0 && dtype != 1))
        return BM_ERR_ARG;
    AttnPacks all{};
    int64_t most = 0;
    for (int i = 0; i < count; ++i) {
        const batmobile_attention_pack& p = packs[i];
        if (p.rows < 0 || p.heads <= 0 || p.D <= 0 || p.D > 256 ||
            (p.rows > 0 && (!p.in || !p.out)) || (!cut && !aligned_to({p.out}, 16)))
            return BM_ERR_ARG;
        all.m[i] = p;
        most = std::max(most, p.rows * p.heads * (cut ? p.D : ceil_div(p.D * (dtype ? 2 : 4), 16)));
    }
    if (most == 0) return BM_OK;
    const dim3 grid((unsigned)std::min<int64_t>(ceil_div(most, 256), 4096), (unsigned)count);
    if (dtype == 0 && cut) attn_pack_kernel<float, true><<<grid, 256, 0, stream>>>(all);
    else if (dtype == 0) attn_pack_kernel<float, false><<<grid, 256, 0, stream>>>(all);
    else if (cut) attn_pack_kernel<uint16_t, true><<<grid, 256, 0, stream>>>(all);
    else attn_pack_kernel<uint16_t, false><<<grid, 256, 0, stream>>>(all);
    return (int)hipGetLastError();
}

extern "C" int batteries_attention_edges_by_head(const float* values, const int32_t* edge_id,
                                                 float* out, int64_t n_edges, int H, int back,
                                                 hipStream_t stream) {
    if (n_edges < 0 || H <= 0 || H > 65535 || n_edges >= INT32_MAX / 4 ||
        !aligned_to({values, out}, 16) || (n_edges > 0 && (!values || !out)))
        return BM_ERR_ARG;
    if (n_edges == 0) return BM_OK;
    const dim3 grid((unsigned)ceil_div(n_edges, 256), (unsigned)ceil_div(H, 16));
    if (back) attn_edges_kernel<false><<<grid, 256, 0, stream>>>(values, edge_id, out, n_edges, H);
    else attn_edges_kernel<true><<<grid, 256, 0, stream>>>(values, edge_id, out, n_edges, H);
    return (int)hipGetLastError();
}

extern "C" size_t batteries_neighbor_attention_workspace_bytes(int64_t n_parts, int H, int Dv) {
    if (n_parts <= 0 || H <= 0 || Dv <= 0) return 0;
    return (size_t)n_parts * H * kAttnRows * (Dv + 2) * sizeof(float);
}

extern "C" int batteries_neighbor_attention(const void* q, const void* k, const void* v,
                                            const float* bias, const int32_t* edge_id,
                                            int bias_by_head,
                                            const batmobile_attention_side* side, void* out,
                                            float* stats, int H, int Hkv, int Dk, int Dv,
                                            int64_t q_stride, int64_t k_stride, int64_t v_stride,
                                            float scale, int dtype, void* workspace,
                                            size_t workspace_bytes, hipStream_t stream) {
    if (!side || !attn_shape_ok(*side, H, Hkv, Dk, Dv, dtype)) return BM_ERR_ARG;
    const int align = dtype == 0 ? 4 : 8;
    if (Dk % align || Dv % align || q_stride % align || k_stride % align || v_stride % align ||
        !attn_strides_ok({q_stride, k_stride, v_stride}) || !aligned_to({q, k, v, out}, 16))
        return BM_ERR_ARG;
    if (side->n_rows == 0) return BM_OK;
    if (!q || !out || (side->n_edges > 0 && (!k || !v))) return BM_ERR_ARG;
    const size_t need = batteries_neighbor_attention_workspace_bytes(side->n_parts, H, Dv);
    if (workspace_bytes < need || (need && !workspace)) return BM_ERR_WORKSPACE;
    AttnFwd a{};
    a.side = side_args(*side);
    a.q = q; a.k = k; a.v = v; a.out = out;
    a.bias = edge_bias(bias, edge_id, side->n_edges, H, bias_by_head != 0);
    a.stats = stats;
    a.part_o = (float*)workspace;
    a.part_ml = a.part_o + (size_t)side->n_parts * H * kAttnRows * Dv;
    const int64_t size = dtype == 0 ? 4 : 2;
    a.qs = (uint32_t)(q_stride * size); a.ks = (uint32_t)(k_stride * size);
    a.vs = (uint32_t)(v_stride * size);
    a.H = H; a.group = H / Hkv; a.Dk = Dk; a.Dv = Dv; a.scale = scale;
    const bool wide = attn_wide(side->n_cols, k_stride * size);
    if (dtype == 0) attn_fwd_run<float>(a, wide, side->n_parts, stream);
    else attn_fwd_run<uint16_t>(a, wide, side->n_parts, stream);
    return (int)hipGetLastError();
}
