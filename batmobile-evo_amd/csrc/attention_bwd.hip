// Gradients of the attention over a graph's edges (attention.hip), go the gradient of o:
//
//   dp_eh = <go[i,h], v[j,g]>,  D_ih = sum_e p_eh dp_eh,  ds_eh = p_eh (dp_eh - D_ih)
//   gb = ds,  gq[i,h] = scale sum_e ds k[j,g],  gk[j,g] = scale sum ds q[i,h],
//   gv[j,g] = sum p go[i,h]
//
// with p recomputed from the rows' maxima and sums.
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
    const float *bias, *stats;
    float* gbias;
    float2* ws;                            // [H][E]: p, ds (of cut tiles first dp)
    int64_t qs, ks, vs, gs, edges;
    int H, group, Dk, Dv;
    float scale;
};

template <typename T, int KP, int VP, bool FULL>
__global__ __launch_bounds__(256, KP + VP <= 256 ? 2 : 1) void attn_scores_kernel(AttnScores a) {
    constexpr int kT = Attn<T>::kTiles;
    constexpr float kInf = __builtin_inff();
    __shared__ float lds_p[4][kTileEdges];           // the bias, then p
    __shared__ float lds_dp[4][kTileEdges];
    __shared__ float lds_d[4][kAttnRows];
    int item, h;
    if (!attn_unit(a.side.n_items, a.H, item, h)) return;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, kv = h / a.group;
    const int4 it4 = a.side.items[item];
    const int row = a.side.rows[it4.x * kAttnRows + n];
    const int steps = it4.z * 2 / kT;
    if (steps == 0) return;
    const T* kbase = (const T*)a.k + (int64_t)kv * a.Dk;
    const T* vbase = (const T*)a.v + (int64_t)kv * a.Dv;
    Step<T> st, next;
    st.load(a.side, it4.y, 0, n, g);
    next.load(a.side, it4.y, min(1, steps - 1), n, g);
    RowFrag<T, KP> kf[kT], q;
    RowFrag<T, VP> go;
#pragma unroll
    for (int t = 0; t < kT; ++t)
        kf[t].template load<FULL>(row_of<T>(kbase, st.row[t], a.ks), a.Dk, g);
    q.template load<FULL>(row_of<T>(a.q, max(row, 0), a.qs) + (int64_t)h * a.Dk, a.Dk, g);
    go.template load<FULL>(row_of<T>(a.go, max(row, 0), a.gs) + (int64_t)h * a.Dv, a.Dv, g);
    const float2 ml =
        *reinterpret_cast<const float2*>(a.stats + ((int64_t)max(row, 0) * a.H + h) * 2);
    const float ref = ml.x == -kInf ? 0.0f : ml.x, inv = ml.y == 0.0f ? 0.0f : 1.0f / ml.y;
    ItemEdges edges;
    edges.load(a.side, item, n);
    float* p_lds = lds_p[threadIdx.x >> 6];
    float* dp_lds = lds_dp[threadIdx.x >> 6];
    const bool staged = edges.total <= kTileEdges;
    auto place = [&](int e) { return (int64_t)(a.side.eid ? a.side.eid[e] : e) * a.H + h; };
    if (staged && a.bias) edges.each([&](int i, int e, int) { p_lds[i] = a.bias[place(e)]; });
    float2* ws = a.ws + (int64_t)h * a.edges;
    float d = 0.0f;
    int done = 0;                              // row n's edges of earlier steps
    for (int i = 0; i < steps; ++i) {
        RowFrag<T, VP> vf[kT];
#pragma unroll
        for (int t = 0; t < kT; ++t)
            vf[t].template load<FULL>(row_of<T>(vbase, st.row[t], a.vs), a.Dv, g);
        v4f s[kT], dp[kT];
#pragma unroll
        for (int t = 0; t < kT; ++t) s[t] = row_product<T, KP>(kf[t], q);
#pragma unroll
        for (int t = 0; t < kT; ++t)
            kf[t].template load<FULL>(row_of<T>(kbase, next.row[t], a.ks), a.Dk, g);
        Step<T> after;
        after.load(a.side, it4.y, min(i + 2, steps - 1), n, g);
        float p[4 * kT];
#pragma unroll
        for (int j = 0; j < 4 * kT; ++j) {
            const int bit = (j >> 2) * 16 + 4 * g + (j & 3);
            const bool on = (st.mask >> bit) & 1;
            const int at = done + st.nth(bit);
            float b = 0.0f;
            if (a.bias) {
                if (staged) b = p_lds[min(edges.off + at, kTileEdges - 1)];
                else if (on) b = a.bias[place(edges.base + at)];
            }
            const float x = fmaf(s[j >> 2][j & 3], a.scale, b);
            p[j] = !on || b == -kInf || x == -kInf ? 0.0f : exp2f((x - ref) * kLog2e) * inv;
        }
#pragma unroll
        for (int t = 0; t < kT; ++t) dp[t] = row_product<T, VP>(vf[t], go);
#pragma unroll
        for (int j = 0; j < 4 * kT; ++j) {
            const int bit = (j >> 2) * 16 + 4 * g + (j & 3);
            const float y = p[j] == 0.0f ? 0.0f : dp[j >> 2][j & 3];
            d = fmaf(p[j], y, d);
            if ((st.mask >> bit) & 1) {
                const int at = done + st.nth(bit);
                if (staged) {
                    p_lds[edges.off + at] = p[j];
                    dp_lds[edges.off + at] = y;
                } else {
                    ws[edges.base + at] = make_float2(p[j], y);
                }
            }
        }
        done += __popc(st.mask);
        st = next;
        next = after;
    }
    if (!staged) return;
    if (it4.w >= 0) {                          // the rest once all parts of the row are there
        edges.each([&](int i, int e, int) { ws[e] = make_float2(p_lds[i], dp_lds[i]); });
        return;
    }
    d += __shfl_xor(d, 16);
    d += __shfl_xor(d, 32);
    float* d_lds = lds_d[threadIdx.x >> 6];
    if (g == 0) d_lds[n] = d;
    __builtin_amdgcn_wave_barrier();
    edges.each([&](int i, int e, int r) {
        const float p = p_lds[i], ds = p == 0.0f ? 0.0f : p * (dp_lds[i] - d_lds[r]);
        ws[e] = make_float2(p, ds);
        if (a.gbias) a.gbias[place(e)] = ds;
    });
}

struct AttnDs {
    AttnSide side;
    const int64_t* row_ptr;
    float2* ws;
    float* gbias;
    int64_t edges;
    int H;
};

// Rows of cut tiles: workgroup p of the parts takes rows p, p + parts of its tile, ...
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
            const float2 w = ws[e];
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
            const float2 w = ws[e];
            const float ds = w.x == 0.0f ? 0.0f : w.x * (w.y - d);
            ws[e].y = ds;
            if (a.gbias) a.gbias[(int64_t)(a.side.eid ? a.side.eid[e] : e) * a.H + h] = ds;
        }
    }
}

// out[row, head] = f sum over the row's edges and the head's group of w x[column, head of x]
struct AttnSum {
    AttnSide side;                         // eid: edge -> its place in ws
    const void* x;
    void* out;
    float* part;                           // [parts, heads, 16, D]
    const float2* ws;
    int64_t xs, edges;
    int heads, group, D, second;           // heads of out; heads of ws per head of out;
                                           // second: the factor is ws.y
    int x_div;                             // head of x = head of ws / x_div
    float f;
};

template <typename T, int P>
__global__ __launch_bounds__(256, 2) void attn_sum_kernel(AttnSum a) {
    constexpr int kT = Attn<T>::kTiles, kR = Attn<T>::kRowsPerLane;
    __shared__ float lds[4][kTileEdges];
    int item, head;
    if (!attn_unit(a.side.n_items, a.heads, item, head)) return;
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int4 it4 = a.side.items[item];
    const int row = a.side.rows[it4.x * kAttnRows + n];
    const int steps = it4.z * 2 / kT;
    float* w_lds = lds[threadIdx.x >> 6];
    ItemEdges edges;
    edges.load(a.side, item, n);
    const bool staged = edges.total <= kTileEdges;
    v4f acc[ColFrag<T, P>::kAcc];
    for (int exact = 0;; ++exact) {
#pragma unroll
        for (int i = 0; i < ColFrag<T, P>::kAcc; ++i) acc[i] = v4f{0, 0, 0, 0};
        for (int hh = head * a.group; steps > 0 && hh < (head + 1) * a.group; ++hh) {
            const T* x = (const T*)a.x + (int64_t)(hh / a.x_div) * a.D;
            const float* ws = reinterpret_cast<const float*>(a.ws + (int64_t)hh * a.edges) +
                              a.second;
            auto factor = [&](int e) {
                return ws[(int64_t)(a.side.eid ? a.side.eid[e] : e) * 2];
            };
            // two steps' rows in turn: one is read while the other is multiplied
            Step<T> s0, s1;
            ColFrag<T, P> x0, x1;
            s0.load(a.side, it4.y, 0, n, g);
            s1.load(a.side, it4.y, min(1, steps - 1), n, g);
            if (steps == 1) s1.mask = 0;
            x0.load([&](int j) { return row_of<T>(x, s0.col[j], a.xs); }, a.D, n);
            __builtin_amdgcn_wave_barrier();
            if (staged) edges.each([&](int i, int e, int) { w_lds[i] = factor(e); });
            __builtin_amdgcn_wave_barrier();
            int done = 0;                      // row n's edges of earlier steps
            auto mac = [&](const Step<T>& s, const ColFrag<T, P>& f) {
                float w[kR];
#pragma unroll
                for (int j = 0; j < kR; ++j) {
                    const int bit = (j >> 2) * 16 + 4 * g + (j & 3);
                    const int at = done + s.nth(bit);
                    const bool on = (s.mask >> bit) & 1;
                    float v = 0.0f;
                    if (staged) v = w_lds[min(edges.off + at, kTileEdges - 1)];
                    else if (on) v = factor(edges.base + at);
                    w[j] = on ? v : 0.0f;
                }
                done += __popc(s.mask);
                if (exact) mac_exact<T, P>(w, s.col, acc, x, a.xs, a.D);
                else f.mac(w, acc);
            };
            for (int i = 0; i < steps; i += 2) {
                x1.load([&](int j) { return row_of<T>(x, s1.col[j], a.xs); }, a.D, n);
                Step<T> s2, s3;
                s2.load(a.side, it4.y, min(i + 2, steps - 1), n, g);
                s3.load(a.side, it4.y, min(i + 3, steps - 1), n, g);
                if (i + 3 >= steps) s3.mask = 0;
                mac(s0, x0);
                x0.load([&](int j) { return row_of<T>(x, s2.col[j], a.xs); }, a.D, n);
                mac(s1, x1);
                s0 = s2;
                s1 = s3;
            }
        }
        if (exact || !any_not_finite<ColFrag<T, P>::kAcc>(acc)) break;
    }
    if (row < 0) return;
    if (it4.w >= 0)
        store_rows<T, P>(a.part + (((int64_t)it4.w * a.heads + head) * kAttnRows + n) * a.D, acc,
                         a.f, a.D, g);
    else
        store_rows<T, P>((T*)a.out + ((int64_t)row * a.heads + head) * a.D, acc, a.f, a.D, g);
}

// Adds the parts of a cut tile, row by row (as attn_join_kernel).
template <typename T>
__global__ __launch_bounds__(256) void attn_sum_join_kernel(AttnSum a) {
    __shared__ float so[4][256];
    const int head = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int first, parts;
    const int tile = tile_of_part(a.side, blockIdx.x, first, parts);
    for (int slot = (int)blockIdx.x - first; slot < kAttnRows; slot += parts) {
        const int row = a.side.rows[tile * kAttnRows + slot];
        if (row < 0) continue;
        float o[4] = {0, 0, 0, 0};
        if (4 * lane < a.D)
            for (int p = w; p < parts; p += 4) {
                const int64_t at = ((int64_t)(first + p) * a.heads + head) * kAttnRows + slot;
                const float4 x = *reinterpret_cast<const float4*>(a.part + at * a.D + 4 * lane);
                o[0] += x.x;
                o[1] += x.y;
                o[2] += x.z;
                o[3] += x.w;
            }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < 4; ++c) so[w][4 * lane + c] = o[c];
        __syncthreads();
        if (w != 0 || 4 * lane >= a.D) continue;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            o[c] = so[0][4 * lane + c] + so[1][4 * lane + c] + so[2][4 * lane + c] +
                   so[3][4 * lane + c];
        attn_store_w<4>((T*)a.out + ((int64_t)row * a.heads + head) * a.D + 4 * lane, o);
    }
}

template <typename T, int KP, int VP>
static void attn_scores_launch(const AttnScores& a, hipStream_t s) {
    const unsigned grid = attn_grid(a.side.n_items, a.H);
    if (a.Dk == KP && a.Dv == VP) attn_scores_kernel<T, KP, VP, true><<<grid, 256, 0, s>>>(a);
    else attn_scores_kernel<T, KP, VP, false><<<grid, 256, 0, s>>>(a);
}
template <typename T, int KP>
static void attn_scores_run_k(const AttnScores& a, hipStream_t s) {
    if (a.Dv <= 64) attn_scores_launch<T, KP, 64>(a, s);
    else if (a.Dv <= 128) attn_scores_launch<T, KP, 128>(a, s);
    else attn_scores_launch<T, KP, 256>(a, s);
}
template <typename T>
static void attn_scores_run(const AttnScores& a, hipStream_t s) {
    if (a.Dk <= 64) attn_scores_run_k<T, 64>(a, s);
    else if (a.Dk <= 128) attn_scores_run_k<T, 128>(a, s);
    else attn_scores_run_k<T, 256>(a, s);
}
template <typename T>
static void attn_sum_run(const AttnSum& a, int parts, hipStream_t s) {
    const unsigned grid = attn_grid(a.side.n_items, a.heads);
    if (grid == 0) return;
    if (a.D <= 64) attn_sum_kernel<T, 64><<<grid, 256, 0, s>>>(a);
    else if (a.D <= 128) attn_sum_kernel<T, 128><<<grid, 256, 0, s>>>(a);
    else attn_sum_kernel<T, 256><<<grid, 256, 0, s>>>(a);
    if (parts)
        attn_sum_join_kernel<T><<<dim3((unsigned)parts, (unsigned)a.heads), 256, 0, s>>>(a);
}

}  // namespace bmhip

using namespace bmhip;

static size_t bwd_part_floats(int64_t dst_parts, int64_t src_parts, int H, int Hkv, int Dk, int Dv) {
    return (size_t)kAttnRows *
           std::max((size_t)dst_parts * H * Dk, (size_t)src_parts * Hkv * std::max(Dk, Dv));
}

extern "C" size_t batteries_neighbor_attention_backward_workspace_bytes(
    int64_t n_edges, int64_t dst_parts, int64_t src_parts, int H, int Hkv, int Dk, int Dv) {
    if (n_edges < 0 || dst_parts < 0 || src_parts < 0 || H <= 0 || Hkv <= 0) return 0;
    return ((size_t)n_edges * H + 1) / 2 * 2 * sizeof(float2) +
           bwd_part_floats(dst_parts, src_parts, H, Hkv, Dk, Dv) * sizeof(float);
}

extern "C" int batteries_neighbor_attention_backward(
    const void* q, const void* k, const void* v, const float* bias, const float* stats,
    const void* grad_out, const int64_t* row_ptr, const int32_t* edge_id,
    const batmobile_attention_side* dst, const batmobile_attention_side* src,
    const int32_t* src_pos, void* grad_q, void* grad_k, void* grad_v, float* grad_bias, int H,
    int Hkv, int Dk, int Dv, int64_t q_stride, int64_t k_stride, int64_t v_stride,
    int64_t go_stride, float scale, int dtype, void* workspace, size_t workspace_bytes,
    hipStream_t stream) {
    if (!dst || !src || !attn_shape_ok(*dst, H, Hkv, Dk, Dv, dtype) ||
        !attn_shape_ok(*src, H, Hkv, Dk, Dv, dtype) || src->n_rows != dst->n_cols ||
        src->n_cols != dst->n_rows || src->n_edges != dst->n_edges)
        return BM_ERR_ARG;
    const int align = dtype == 0 ? 4 : 8;
    if (Dk % align || Dv % align || q_stride % align || k_stride % align || v_stride % align ||
        go_stride % align || !aligned_to({q, k, v, grad_out, grad_q, grad_k, grad_v, workspace}, 16))
        return BM_ERR_ARG;
    const int64_t E = dst->n_edges;
    const size_t need = batteries_neighbor_attention_backward_workspace_bytes(
        E, dst->n_parts, src->n_parts, H, Hkv, Dk, Dv);
    if (workspace_bytes < need || (need && !workspace)) return BM_ERR_WORKSPACE;
    float2* ws = (float2*)workspace;
    float* part = (float*)(ws + ((size_t)E * H + 1) / 2 * 2);
    if (E > 0) {
        AttnScores a{};
        a.side = side_args(*dst, edge_id);
        a.q = q; a.k = k; a.v = v; a.go = grad_out; a.bias = bias; a.stats = stats; a.ws = ws;
        a.gbias = grad_bias;
        a.qs = q_stride; a.ks = k_stride; a.vs = v_stride; a.gs = go_stride; a.edges = E;
        a.H = H; a.group = H / Hkv; a.Dk = Dk; a.Dv = Dv; a.scale = scale;
        if (dtype == 0) attn_scores_run<float>(a, stream);
        else attn_scores_run<uint16_t>(a, stream);
        if (dst->n_parts > 0) {
            AttnDs d{side_args(*dst, edge_id), row_ptr, ws, grad_bias, E, H};
            attn_ds_kernel<<<dim3((unsigned)dst->n_parts, (unsigned)H), 1024, 0, stream>>>(d);
        }
    }
    auto sum = [&](const batmobile_attention_side& side, const int32_t* at, const void* x,
                   int64_t xs, void* out, int heads, int group, int x_div, int D, int second,
                   float f) {
        if (side.n_rows == 0) return;
        AttnSum a{};
        a.side = side_args(side, at);
        a.x = x; a.xs = xs; a.out = out; a.part = part; a.ws = ws; a.edges = E; a.heads = heads;
        a.group = group; a.x_div = x_div; a.D = D; a.second = second; a.f = f;
        if (dtype == 0) attn_sum_run<float>(a, side.n_parts, stream);
        else attn_sum_run<uint16_t>(a, side.n_parts, stream);
    };
    sum(*dst, nullptr, k, k_stride, grad_q, H, 1, H / Hkv, Dk, 1, scale);
    sum(*src, src_pos, q, q_stride, grad_k, Hkv, H / Hkv, 1, Dk, 1, scale);
    sum(*src, src_pos, grad_out, go_stride, grad_v, Hkv, H / Hkv, 1, Dv, 0, 1.0f);
    return (int)hipGetLastError();
}
