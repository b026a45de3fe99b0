// Gradients of the attention over a graph's edges (attention.hip), go the gradient of o:
//
//   dp_eh = <go[i,h], v[j,g]>,  D_ih = sum_e p_eh dp_eh,  ds_eh = p_eh (dp_eh - D_ih)
//   gb = ds,  gq[i,h] = scale sum_e ds k[j,g],  gk[j,g] = scale sum ds q[i,h],
//   gv[j,g] = sum p go[i,h]
//
// with p formed again from the rows' kept references and sums (attention.hip).
//
//   attn_scores  a tile and head at a time, both products of its pairs: p and dp per edge, kept
//                in LDS, D and ds; p and ds go to the workspace, ds to gb
//   attn_ds      D and ds of the rows of cut tiles
//   attn_sum     tiles of either side: gq (ds and k), gk (ds and q), gv (p and go)
//
// D comes from the same fp32 p and dp: formed from the rounded o it would put o's rounding into
// gb, which is fp32.  p and ds take 8 bytes an edge and head in the workspace; the source side
// would otherwise read two rows and form both products again.  No atomics: sums run in the
// plan's order.
#include "attention.h"

namespace bmhip {

struct AttnScores {
    AttnSide side;
    const void *q, *k, *v, *go;
    EdgeBias bias;
    const float* stats;
    float* gbias;                          // [E, H], or NULL
    const int *eid, *place;                // edge -> its row of gbias, its place among the sources'
    float2* ws;                            // [H][E], sources' order: p, ds (of cut tiles first dp)
    float* wd;                             // [H][E], destinations' order: ds
    uint32_t qs, ks, vs, gs;               // rows' strides in bytes
    int64_t edges;
    int H, group, Dk, Dv;
    float scale;
};

// A step takes 16 columns: with 32 the rows of k and v would leave LDS for 6 waves a CU only.
// k and v of a step go to LDS while the products of the step before run; p and dp of the step
// before are written to LDS first, as are all reads done (attn_fwd_kernel).
//
// Measured, atoms with 28 neighbours: 5000, 8 heads of 128 in f32 69 us; 20,011, 8 on 2 heads of
// 128 in bf16 101 us (111 in steps of 32 columns), waves waiting 43 % of their time for memory
// and 29 % for issue; 5000 with random neighbours, 4 heads of 24 by 256 in f32, 138 us (rows from
// Infinity Cache).  Registers for two waves a SIMD give 2 % at 128 components in bf16; LDS
// holds 9 waves a CU there, 6 at 128 in f32, 3 at 256 in f32 (less than one a SIMD).
template <typename T, int KP, int VP, bool FULL, bool WIDE>
__global__ __launch_bounds__(64, 2) void attn_scores_kernel(AttnScores a) {
    constexpr int kT = 1;                      // (see the kernel's head)
    constexpr float kInf = __builtin_inff();
    using KRows = RowTile<T, KP, kT>;
    using VRows = RowTile<T, VP, kT>;
    __shared__ __attribute__((aligned(1024))) char k_lds[KRows::kBytes];
    __shared__ __attribute__((aligned(1024))) char v_lds[VRows::kBytes];
    __shared__ float p_lds[kTileEdges + 1];          // the bias, then p
    __shared__ float dp_lds[kTileEdges + 1];
    int item, h;
    if (!attn_unit(blockIdx.x, a.side.n_items, a.H, item, h)) return;
    const int lane = threadIdx.x, n = lane & 15, g = lane >> 4;
    const int kv = uniform_quotient(h, a.group);
    const Item it(a.side, item, lane);
    const int row = it.row, steps = it.steps(kT);
    if (steps == 0) return;
    const T* kbase = (const T*)a.k + (int64_t)kv * a.Dk;
    const T* vbase = (const T*)a.v + (int64_t)kv * a.Dv;
    const Steps<kT> step(a.side, it, lane);
    int ids = step.ids(0);
    uint32_t mask = step.mask(0);
    RowFrag<T, KP> q;
    RowFrag<T, VP> go;
    q.template load<FULL>(row_of<T>(a.q, max(row, 0), a.qs) + (int64_t)h * a.Dk, a.Dk, g);
    go.template load<FULL>(row_of<T>(a.go, max(row, 0), a.gs) + (int64_t)h * a.Dv, a.Dv, g);
    const float2 ml =
        *reinterpret_cast<const float2*>(a.stats + ((int64_t)max(row, 0) * a.H + h) * 2);
    const float ref = ml.x == -kInf ? 0.0f : ml.x, inv = ml.y == 0.0f ? 0.0f : 1.0f / ml.y;
    KRows::template fill<FULL, WIDE>(k_lds, ids, kbase, a.ks, a.Dk, lane);
    VRows::template fill<FULL, WIDE>(v_lds, ids, vbase, a.vs, a.Dv, lane);
    ids = step.ids(1);
    auto keep_bias = [&](int i, int, float b, int) { p_lds[i] = b; };
    if (!a.bias.value)
        it.each<float>(a.side, lane, [](int) { return 0.0f; }, keep_bias);
    else if (a.bias.eid)
        it.each<float>(a.side, lane, [&](int e) { return a.bias.at(e, h); }, keep_bias);
    else
        it.each<float>(a.side, lane, [&](int e) {
            return a.bias.value[(int64_t)e * a.bias.edge_step + h * a.bias.head_step];
        }, keep_bias);
    float2* ws = a.ws + (int64_t)h * a.edges;
    float d = 0.0f, p[4 * kT], dp[4 * kT];
    int done = 0;                              // row n's edges of earlier steps
    int at[4 * kT];
    bool on[4 * kT], was[4 * kT] = {};
    auto keep = [&]() {
#pragma unroll
        for (int j = 0; j < 4 * kT; ++j)
            if (was[j]) {
                p_lds[at[j]] = p[j];
                dp_lds[at[j]] = dp[j];
            }
    };
    for (int i = 0; i < steps; ++i) {
        RowFrag<T, KP> kf[kT];
        RowFrag<T, VP> vf[kT];
        KRows::template arrived<0>();
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            KRows::template read<FULL>(kf[t], k_lds, t, a.Dk, n, g);
            VRows::template read<FULL>(vf[t], v_lds, t, a.Dv, n, g);
        }
        keep();
        float b[4 * kT];
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            edge_places(mask, t, g, it.off + done, at + 4 * t, on + 4 * t);
#pragma unroll
            for (int r = 0; r < 4; ++r) b[4 * t + r] = p_lds[at[4 * t + r]];
        }
        KRows::reads_done();
        KRows::template fill<FULL, WIDE>(k_lds, ids, kbase, a.ks, a.Dk, lane);
        VRows::template fill<FULL, WIDE>(v_lds, ids, vbase, a.vs, a.Dv, lane);
        ids = step.ids(i + 2);
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            const v4f s = row_product<T, KP>(kf[t], q);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = 4 * t + r;
                const float x = fmaf(s[r], a.scale, b[j]);
                p[j] = attn_exp(x - ref) * inv;
                p[j] = on[j] & (b[j] != -kInf) & (x != -kInf) ? p[j] : 0.0f;
                was[j] = on[j];
            }
        }
#pragma unroll
        for (int t = 0; t < kT; ++t) {
            const v4f y = row_product<T, VP>(vf[t], go);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int j = 4 * t + r;
                dp[j] = p[j] == 0.0f ? 0.0f : y[r];
                d = fmaf(p[j], dp[j], d);
            }
        }
        done += __popc(mask);
        mask = step.mask(i + 1);
    }
    keep();
    KRows::template arrived<0>();              // the last fills, which nothing reads
    auto place = [&](int e) { return a.place[e]; };
    if (it.part >= 0) {                        // the rest once all parts of the row are there
        it.each<int>(a.side, lane, place, [&](int i, int, int to, int) {
            ws[to] = make_float2(p_lds[i], dp_lds[i]);
        });
        return;
    }
    d = sum_over_groups(d);
    float dr[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) dr[k] = __shfl(d, 4 * k + g);
    float* wd = a.wd + (int64_t)h * a.edges;
    it.each<int>(a.side, lane, place, [&](int i, int e, int to, int k) {
        const float pe = p_lds[i], ds = pe == 0.0f ? 0.0f : pe * (dp_lds[i] - dr[k]);
        ws[to] = make_float2(pe, ds);
        wd[e] = ds;
        if (a.gbias) a.gbias[(int64_t)(a.eid ? a.eid[e] : e) * a.H + h] = ds;
    });
}

struct AttnDs {
    AttnSide side;
    const int64_t* row_ptr;
    const int *eid, *place;
    float2* ws;
    float *wd, *gbias;
    int64_t edges;
    int H;
};

// Rows of cut tiles: workgroup p of the parts takes rows p, p + parts of its tile, ...; a pass for
// D and one for ds over a row's edges, each a latency of memory per 1024 edges.
__global__ __launch_bounds__(1024) void attn_ds_kernel(AttnDs a) {
    __shared__ float sh[16];
    const int h = blockIdx.y;
    int first, parts;
    const int tile = tile_of_part(a.side, blockIdx.x, first, parts);
    for (int slot = (int)blockIdx.x - first; slot < kAttnRows; slot += parts) {
        const int row = a.side.rows[tile * kAttnRows + slot];
        if (row < 0) continue;
        const int64_t e0 = a.row_ptr[row], e1 = a.row_ptr[row + 1];
        float2* ws = a.ws + (int64_t)h * a.edges;
        float d = 0.0f;
        for (int64_t e = e0 + threadIdx.x; e < e1; e += 1024) {
            const float2 w = ws[a.place[e]];
            d += w.x == 0.0f ? 0.0f : w.x * w.y;
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) d += __shfl_xor(d, o);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = d;
        __syncthreads();
        d = 0.0f;
        for (int i = 0; i < 16; ++i) d += sh[i];
        for (int64_t e = e0 + threadIdx.x; e < e1; e += 1024) {
            float2* at = ws + a.place[e];
            const float ds = at->x == 0.0f ? 0.0f : at->x * (at->y - d);
            at->y = ds;
            a.wd[(int64_t)h * a.edges + e] = ds;
            if (a.gbias) a.gbias[(int64_t)(a.eid ? a.eid[e] : e) * a.H + h] = ds;
        }
    }
}

// out[row, head] = f sum over the row's edges and the head's group of w x[column, head of x]
struct AttnSum {
    AttnSide side;
    const void* x;
    void* out;
    float* part;                           // [parts, heads, 16, D]
    const float* w;                        // [H][E], w_step apart, in the side's order
    uint32_t xs;                           // row stride in bytes
    int w_step;
    int64_t edges;
    int heads, group, D;                   // heads of out; heads of w per head of out
    int x_div;                             // head of x = head of ws / x_div
    float f;
};

// An item's rows one after the other, each over its own edges of a factor other than 0.
template <typename T>
__device__ __forceinline__ void attn_sum_rows(const AttnSum& a, int item, int head,
                                              const Item& it) {
    for (int r = 0; r < kAttnRows; ++r) {
        const int row = a.side.rows[it.tile * kAttnRows + r];
        if (row < 0) continue;
        float o[4] = {0, 0, 0, 0};
        for (int hh = head * a.group; hh < (head + 1) * a.group; ++hh)
            each_edge(a.side, item, r, [&](int e, int col) {
                const float w = a.w[((int64_t)hh * a.edges + e) * a.w_step];
                if (w != 0.0f)
                    add_row<T>(o, w, row_of<T>(a.x, col, a.xs) + (int64_t)(hh / a.x_div) * a.D,
                               a.D);
            });
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int d = c * 64 + threadIdx.x;
            if (d >= a.D) continue;
            if (it.part >= 0)
                a.part[(((int64_t)it.part * a.heads + head) * kAttnRows + r) * a.D + d] = o[c] * a.f;
            else
                attn_st((T*)a.out + ((int64_t)row * a.heads + head) * a.D + d, o[c] * a.f);
        }
    }
}

// Up to three sums in one launch, so that one's last workgroups run beside the next one's first.
struct AttnSums {
    AttnSum sum[3];
    unsigned first[4];                     // first workgroup of each, and their end
};

// The rows pass through LDS as in the other kernels, the factors (p or ds, one head) lie in LDS by
// edge.  Factors of a bf16 product are taken as two bf16 numbers, hi + lo: in one they would round
// every gradient's terms to 8 bits.  The first two sums share the source side's plan but not its
// rows.
//
// Measured, atoms with 28 neighbours, the three sums: 5000, 8 heads of 128 in f32 69 us; 20,011,
// 8 on 2 heads of 128 in bf16 102 us, 34 % of the waves' time waiting for memory, 29 % for
// issue.  Registers for two waves a SIMD (at 256 in bf16 with 8 bytes a lane of spill): a training step of 20,000 atoms, 8 heads of 256 in bf16, 369 us
// against 418 without the bound; 8 heads of 64 125 against 134.
template <typename T, int P>
__global__ __launch_bounds__(64, 2) void attn_sum_kernel(AttnSums all) {
    const int which = (blockIdx.x >= all.first[1]) + (blockIdx.x >= all.first[2]);
    const AttnSum& a = all.sum[which];
    constexpr int kT = Attn<T>::kTiles, kR = Attn<T>::kRowsPerLane;
    constexpr int kBytes = (kTileEdges + 1) * 4;
    __shared__ __attribute__((aligned(16))) char
        lds[kBytes > OutTile<T, P>::kBytes ? kBytes : OutTile<T, P>::kBytes];
    float* w_lds = reinterpret_cast<float*>(lds);
    int item, head;
    if (!attn_unit(blockIdx.x - all.first[which], a.side.n_items, a.heads, item, head)) return;
    const int lane = threadIdx.x, n = lane & 15, g = lane >> 4;
    const Item it(a.side, item, lane);
    const int row = it.row, steps = it.steps(kT);
    v4f acc[ColFrag<T, P>::kAcc];
    {
#pragma unroll
        for (int i = 0; i < ColFrag<T, P>::kAcc; ++i) acc[i] = v4f{0, 0, 0, 0};
        for (int hh = head * a.group; steps > 0 && hh < (head + 1) * a.group; ++hh) {
            const T* x = (const T*)a.x + (int64_t)(hh / a.x_div) * a.D;
            const float* wh = a.w + (int64_t)hh * a.edges * a.w_step;
            // two steps' rows in turn: one is read while the other is multiplied
            const Steps<kT> step(a.side, it, lane);
            ColFrag<T, P> x0, x1;
            int s0 = step.ids(0), s1 = step.ids(1);
            uint32_t m0 = step.mask(0), m1 = step.mask(1);
            // the rows of the columns in `ids`; then the columns of step `then`
            auto load = [&](ColFrag<T, P>& f, int& ids, int then) {
                const StepCols<T> cols(ids, g);
                ids = step.ids(then);
                load_fence();
                f.load([&](int j) { return row_of<T>(x, cols.col[j], a.xs); }, a.D, n);
                load_fence();
            };
            load(x0, s0, 2);
            __builtin_amdgcn_wave_barrier();
            it.each<float>(a.side, lane, [&](int e) { return wh[(int64_t)e * a.w_step]; },
                           [&](int i, int, float w, int) { w_lds[i] = w; });
            __builtin_amdgcn_wave_barrier();
            int done = 0;                      // row n's edges of earlier steps
            auto mac = [&](uint32_t mask, const ColFrag<T, P>& f) {
                float w[kR];
#pragma unroll
                for (int t = 0; t < kT; ++t) {
                    int at[4];
                    bool on[4];
                    edge_places(mask, t, g, it.off + done, at, on);
#pragma unroll
                    for (int r = 0; r < 4; ++r) w[4 * t + r] = on[r] ? w_lds[at[r]] : 0.0f;
                }
                done += __popc(mask);
                f.mac(w, acc);
            };
            for (int i = 0; i < steps; i += 2) {
                load(x1, s1, i + 3);
                mac(m0, x0);
                m0 = step.mask(i + 2);
                load(x0, s0, i + 4);
                mac(i + 1 < steps ? m1 : 0, x1);
                m1 = step.mask(i + 3);
            }
        }
    }
    if (__builtin_expect(any_not_finite<ColFrag<T, P>::kAcc>(acc), 0)) {
        attn_sum_rows<T>(a, item, head, it);
        return;
    }
    if (it.part >= 0) {
        if (row >= 0)
            store_part<T, P>(
                a.part + (((int64_t)it.part * a.heads + head) * kAttnRows + n) * a.D, acc, a.f,
                a.D, g);
        return;
    }
    OutTile<T, P>::store(lds, (T*)a.out + (int64_t)head * a.D, (int64_t)a.heads * a.D, row, acc,
                         a.f, a.D, lane);
}

// Adds the parts of a cut tile, row by row (as attn_join_kernel, and as long).
template <typename T>
__global__ __launch_bounds__(1024) void attn_sum_join_kernel(AttnSum a) {
    __shared__ float so[1024][4];
    const int head = blockIdx.y, wide = a.D / 4, groups = 1024 / wide;
    const int k = threadIdx.x / wide, c4 = threadIdx.x % wide;
    int first, parts;
    const int tile = tile_of_part(a.side, blockIdx.x, first, parts);
    for (int slot = (int)blockIdx.x - first; slot < kAttnRows; slot += parts) {
        const int row = a.side.rows[tile * kAttnRows + slot];
        if (row < 0) continue;
        float o[4] = {0, 0, 0, 0};
        if (k < groups) {
#pragma unroll 4
            for (int p = k; p < parts; p += groups) {
                const int64_t at = ((int64_t)(first + p) * a.heads + head) * kAttnRows + slot;
                const float4 x = *reinterpret_cast<const float4*>(a.part + at * a.D + 4 * c4);
                o[0] += x.x;
                o[1] += x.y;
                o[2] += x.z;
                o[3] += x.w;
            }
        }
        __syncthreads();
        *reinterpret_cast<float4*>(so[threadIdx.x]) = make_float4(o[0], o[1], o[2], o[3]);
        __syncthreads();
        if (k != 0) continue;
        for (int i = 1; i < groups; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(so[i * wide + c4]);
            o[0] += x.x;
            o[1] += x.y;
            o[2] += x.z;
            o[3] += x.w;
        }
        attn_store_w<4>((T*)a.out + ((int64_t)row * a.heads + head) * a.D + 4 * c4, o);
    }
}

template <typename T, int KP, int VP>
static void attn_scores_launch(const AttnScores& a, bool wide, hipStream_t s) {
    const unsigned grid = attn_grid(a.side.n_items, a.H);
    if (wide) attn_scores_kernel<T, KP, VP, false, true><<<grid, 64, 0, s>>>(a);
    else if (a.Dk == KP && a.Dv == VP)
        attn_scores_kernel<T, KP, VP, true, false><<<grid, 64, 0, s>>>(a);
    else attn_scores_kernel<T, KP, VP, false, false><<<grid, 64, 0, s>>>(a);
}
template <typename T, int KP>
static void attn_scores_run_k(const AttnScores& a, bool wide, hipStream_t s) {
    if (a.Dv <= 64) attn_scores_launch<T, KP, 64>(a, wide, s);
    else if (a.Dv <= 128) attn_scores_launch<T, KP, 128>(a, wide, s);
    else attn_scores_launch<T, KP, 256>(a, wide, s);
}
template <typename T>
static void attn_scores_run(const AttnScores& a, bool wide, hipStream_t s) {
    if (a.Dk <= 64) attn_scores_run_k<T, 64>(a, wide, s);
    else if (a.Dk <= 128) attn_scores_run_k<T, 128>(a, wide, s);
    else attn_scores_run_k<T, 256>(a, wide, s);
}
static int attn_sum_class(int D) { return D <= 64 ? 64 : D <= 128 ? 128 : 256; }

// The n sums of one size class, the later of their parts' joins.
template <typename T>
static void attn_sum_run(const AttnSum* sums, const int* parts, int n, hipStream_t s) {
    AttnSums all{};
    all.first[0] = 0;
    for (int i = 0; i < 3; ++i) {
        all.sum[i] = sums[std::min(i, n - 1)];
        all.first[i + 1] =
            all.first[i] + (i < n ? attn_grid(sums[i].side.n_items, sums[i].heads) : 0);
    }
    const unsigned grid = all.first[3];
    if (grid == 0) return;
    const int P = attn_sum_class(sums[0].D);
    if (P == 64) attn_sum_kernel<T, 64><<<grid, 64, 0, s>>>(all);
    else if (P == 128) attn_sum_kernel<T, 128><<<grid, 64, 0, s>>>(all);
    else attn_sum_kernel<T, 256><<<grid, 64, 0, s>>>(all);
    for (int i = 0; i < n; ++i)
        if (parts[i])
            attn_sum_join_kernel<T><<<dim3((unsigned)parts[i], (unsigned)sums[i].heads), 1024, 0,
                                      s>>>(sums[i]);
}

}  // namespace bmhip

using namespace bmhip;

static size_t bwd_part_floats(int64_t dst_parts, int64_t src_parts, int H, int Hkv, int Dk, int Dv) {
    return (size_t)kAttnRows * ((size_t)dst_parts * H * Dk + (size_t)src_parts * Hkv * (Dk + Dv));
}

extern "C" size_t batteries_neighbor_attention_backward_workspace_bytes(
    int64_t n_edges, int64_t dst_parts, int64_t src_parts, int H, int Hkv, int Dk, int Dv) {
    if (n_edges < 0 || dst_parts < 0 || src_parts < 0 || H <= 0 || Hkv <= 0) return 0;
    return ((size_t)n_edges * H + 3) / 4 * 4 * 3 * sizeof(float) +
           bwd_part_floats(dst_parts, src_parts, H, Hkv, Dk, Dv) * sizeof(float);
}

extern "C" int batteries_neighbor_attention_backward(
    const void* q, const void* k, const void* v, const float* bias, const float* stats,
    const void* grad_out, const int64_t* row_ptr, const int32_t* edge_id,
    int bias_by_head, const batmobile_attention_side* dst, const batmobile_attention_side* src,
    const int32_t* src_place, void* grad_q, void* grad_k, void* grad_v, float* grad_bias, int H,
    int Hkv, int Dk, int Dv, int64_t q_stride, int64_t k_stride, int64_t v_stride,
    int64_t go_stride, float scale, int dtype, void* workspace, size_t workspace_bytes,
    hipStream_t stream) {
    if (!dst || !src || !attn_shape_ok(*dst, H, Hkv, Dk, Dv, dtype) ||
        !attn_shape_ok(*src, H, Hkv, Dk, Dv, dtype) || src->n_rows != dst->n_cols ||
        src->n_cols != dst->n_rows || src->n_edges != dst->n_edges)
        return BM_ERR_ARG;
    const int align = dtype == 0 ? 4 : 8;
    if (Dk % align || Dv % align || q_stride % align || k_stride % align || v_stride % align ||
        go_stride % align || !attn_strides_ok({q_stride, k_stride, v_stride, go_stride}) ||
        !aligned_to({q, k, v, grad_out, grad_q, grad_k, grad_v, workspace}, 16))
        return BM_ERR_ARG;
    const int64_t E = dst->n_edges, size = dtype == 0 ? 4 : 2;
    if ((dst->n_rows > 0 && !grad_q) || (src->n_rows > 0 && (!grad_k || !grad_v)) ||
        (E > 0 && (!q || !k || !v || !stats || !grad_out || !row_ptr || !src_place)))
        return BM_ERR_ARG;
    const size_t need = batteries_neighbor_attention_backward_workspace_bytes(
        E, dst->n_parts, src->n_parts, H, Hkv, Dk, Dv);
    if (workspace_bytes < need || (need && !workspace)) return BM_ERR_WORKSPACE;
    const bool by_head = bias_by_head != 0;
    float2* ws = (float2*)workspace;
    float* wd = (float*)(ws + ((size_t)E * H + 3) / 4 * 4);
    float* part = wd + ((size_t)E * H + 3) / 4 * 4;
    if (E > 0) {
        AttnScores a{};
        a.side = side_args(*dst);
        a.q = q; a.k = k; a.v = v; a.go = grad_out; a.stats = stats;
        a.bias = edge_bias(bias, edge_id, E, H, by_head);
        a.ws = ws;
        a.wd = wd; a.place = src_place;
        a.gbias = by_head ? nullptr : grad_bias;
        a.eid = edge_id;
        a.qs = (uint32_t)(q_stride * size); a.ks = (uint32_t)(k_stride * size);
        a.vs = (uint32_t)(v_stride * size); a.gs = (uint32_t)(go_stride * size); a.edges = E;
        a.H = H; a.group = H / Hkv; a.Dk = Dk; a.Dv = Dv; a.scale = scale;
        const bool wide = attn_wide(dst->n_cols, std::max(k_stride, v_stride) * size);
        if (dtype == 0) attn_scores_run<float>(a, wide, stream);
        else attn_scores_run<uint16_t>(a, wide, stream);
        if (dst->n_parts > 0) {
            AttnDs d{side_args(*dst), row_ptr, edge_id, src_place, ws, wd, a.gbias, E, H};
            attn_ds_kernel<<<dim3((unsigned)dst->n_parts, (unsigned)H), 1024, 0, stream>>>(d);
        }
    }
    if (grad_bias && by_head && E > 0) {
        const int rc = batteries_attention_edges_by_head(wd, edge_id, grad_bias, E, H, 1, stream);
        if (rc != BM_OK) return rc;
    }
    // the sums with the longest work per wave first; cut tiles' parts of each behind the last's
    AttnSum sums[3];
    int parts[3], n = 0;
    auto sum = [&](const batmobile_attention_side& side, const void* x, int64_t xs, void* out,
                   int heads, int group, int x_div, int D, const float* w, int w_step, float f) {
        if (side.n_rows == 0) return;
        AttnSum& a = sums[n];
        a.side = side_args(side);
        a.x = x; a.xs = (uint32_t)(xs * size); a.out = out; a.part = part; a.edges = E;
        a.heads = heads; a.group = group; a.x_div = x_div; a.D = D; a.w = w; a.w_step = w_step;
        a.f = f;
        part += (size_t)side.n_parts * heads * kAttnRows * D;
        parts[n++] = side.n_parts;
    };
    auto run = [&]() {
        if (n == 0) return;
        if (dtype == 0) attn_sum_run<float>(sums, parts, n, stream);
        else attn_sum_run<uint16_t>(sums, parts, n, stream);
        n = 0;
    };
    sum(*src, q, q_stride, grad_k, Hkv, H / Hkv, 1, Dk, &ws->y, 2, scale);
    if (attn_sum_class(Dk) != attn_sum_class(Dv)) run();
    sum(*src, grad_out, go_stride, grad_v, Hkv, H / Hkv, 1, Dv, &ws->x, 2, 1.0f);
    if (attn_sum_class(Dk) != attn_sum_class(Dv)) run();
    sum(*dst, k, k_stride, grad_q, H, 1, H / Hkv, Dk, wd, 1, scale);
    run();
    return (int)hipGetLastError();
}
