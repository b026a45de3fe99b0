// Softmax attention of every row (destination) over its neighbours (sources), forward and
// backward, on the edge list of a graph (no reference counterpart: the reference sums its
// messages, src/message_passing/fused_message_passing.cu).
//
//   x_eh = scale <q[i,h], k[j,g]> + b[e,h]      edge e: j -> i, g = h / (H / H_kv)
//   p_eh = exp(x_eh - m_ih) / l_ih              m, l: maximum and sum of exponentials over
//                                               the edges of row i (b = -inf: no edge)
//   o_ih = sum_e p_eh v[j,g]                    a row without an edge: o = 0
//
// and, with go the gradient of o,
//
//   dp_eh = <go[i,h], v[j,g]>,  D_ih = sum_e p_eh dp_eh,  ds_eh = p_eh (dp_eh - D_ih)
//   gb = ds,  gq[i,h] = scale sum_e ds k[j,g],  gk[j,g] = scale sum ds q[i,h],
//   gv[j,g] = sum p go[i,h]
//
// One wave per (row, head): a lane holds components lane, lane + 64, ... of the head.
#include "common.h"
#include "batmobile_hip.h"

namespace bmhip {

constexpr int kAttnMaxPer = 4;  // components per lane: head sizes up to 256

template <typename T>
__device__ __forceinline__ float attn_ld(const T* p);
template <>
__device__ __forceinline__ float attn_ld<float>(const float* p) { return *p; }
template <>
__device__ __forceinline__ float attn_ld<uint16_t>(const uint16_t* p) {
    return __uint_as_float((uint32_t)*p << 16);
}
__device__ __forceinline__ void attn_st(float* p, float v) { *p = v; }
__device__ __forceinline__ void attn_st(uint16_t* p, float v) {
    *p = (uint16_t)(bf16_pack(v, 0.0f) & 0xffffu);
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

struct AttnArgs {
    const void *q, *k, *v, *go;
    const float* bias;
    const int64_t *row_ptr, *col, *eid;        // edges of a row: [row_ptr[i], row_ptr[i + 1])
    const int64_t *src_ptr, *src_dst, *src_pos;  // of a source: its destinations, edge positions
    void *out, *gq, *gk, *gv;
    float *stats, *gbias;
    float2* ws;                                // [E, H]: p, ds
    int64_t n_dst, n_src, qs, ks, vs, gs;      // rows' strides in elements
    int H, Hkv, Dk, Dv;
    float scale;
};

template <typename T>
__global__ __launch_bounds__(256) void attn_fwd_kernel(AttnArgs a) {
    const int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (u >= a.n_dst * a.H) return;
    const int lane = threadIdx.x & 63, h = (int)(u % a.H), g = h / (a.H / a.Hkv);
    const int64_t i = u / a.H;
    const T* q = (const T*)a.q + i * a.qs + (int64_t)h * a.Dk;
    float qr[kAttnMaxPer], o[kAttnMaxPer], m = -__builtin_inff(), l = 0.0f;
    for (int c = 0; c < kAttnMaxPer; ++c) {
        qr[c] = c * 64 + lane < a.Dk ? attn_ld(q + c * 64 + lane) : 0.0f;
        o[c] = 0.0f;
    }
    for (int64_t e = a.row_ptr[i]; e < a.row_ptr[i + 1]; ++e) {
        const int64_t j = a.col[e];
        const float b = a.bias ? a.bias[(a.eid ? a.eid[e] : e) * a.H + h] : 0.0f;
        if (b == -__builtin_inff()) continue;
        const T* k = (const T*)a.k + j * a.ks + (int64_t)g * a.Dk;
        float s = 0.0f;
        for (int c = 0; c < kAttnMaxPer; ++c)
            if (c * 64 + lane < a.Dk) s = fmaf(qr[c], attn_ld(k + c * 64 + lane), s);
        const float x = wave_sum(s) * a.scale + b;
        if (x == -__builtin_inff()) continue;
        const float mn = fmaxf(m, x);
        const float al = m == mn ? 1.0f : __expf(m - mn), p = __expf(x - mn);
        m = mn;
        l = l * al + p;
        const T* v = (const T*)a.v + j * a.vs + (int64_t)g * a.Dv;
        for (int c = 0; c < kAttnMaxPer; ++c)
            if (c * 64 + lane < a.Dv) o[c] = fmaf(p, attn_ld(v + c * 64 + lane), o[c] * al);
    }
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
    T* out = (T*)a.out + (i * a.H + h) * (int64_t)a.Dv;
    for (int c = 0; c < kAttnMaxPer; ++c)
        if (c * 64 + lane < a.Dv) attn_st(out + c * 64 + lane, o[c] * inv);
    if (a.stats && lane == 0) {
        a.stats[u * 2] = m;
        a.stats[u * 2 + 1] = l;
    }
}

// gq, gbias and the edges' p and ds: a first pass over the row's edges for p, dp and D
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_dst_kernel(AttnArgs a) {
    const int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (u >= a.n_dst * a.H) return;
    const int lane = threadIdx.x & 63, h = (int)(u % a.H), g = h / (a.H / a.Hkv);
    const int64_t i = u / a.H;
    const T* q = (const T*)a.q + i * a.qs + (int64_t)h * a.Dk;
    const T* go = (const T*)a.go + i * a.gs + (int64_t)h * a.Dv;
    const float m = a.stats[u * 2], l = a.stats[u * 2 + 1];
    float qr[kAttnMaxPer], gr[kAttnMaxPer], gq[kAttnMaxPer], D = 0.0f;
    for (int c = 0; c < kAttnMaxPer; ++c) {
        qr[c] = c * 64 + lane < a.Dk ? attn_ld(q + c * 64 + lane) : 0.0f;
        gr[c] = c * 64 + lane < a.Dv ? attn_ld(go + c * 64 + lane) : 0.0f;
        gq[c] = 0.0f;
    }
    const int64_t e0 = a.row_ptr[i], e1 = a.row_ptr[i + 1];
    for (int64_t e = e0; e < e1; ++e) {
        const int64_t j = a.col[e];
        const float b = a.bias ? a.bias[(a.eid ? a.eid[e] : e) * a.H + h] : 0.0f;
        float p = 0.0f, dp = 0.0f;
        if (b != -__builtin_inff()) {
            const T* k = (const T*)a.k + j * a.ks + (int64_t)g * a.Dk;
            const T* v = (const T*)a.v + j * a.vs + (int64_t)g * a.Dv;
            float s = 0.0f;
            for (int c = 0; c < kAttnMaxPer; ++c) {
                if (c * 64 + lane < a.Dk) s = fmaf(qr[c], attn_ld(k + c * 64 + lane), s);
                if (c * 64 + lane < a.Dv) dp = fmaf(gr[c], attn_ld(v + c * 64 + lane), dp);
            }
            const float x = wave_sum(s) * a.scale + b;
            dp = wave_sum(dp);
            if (x != -__builtin_inff()) {
                p = __expf(x - m) / l;
                D += p * dp;
            }
        }
        if (lane == 0) a.ws[e * a.H + h] = make_float2(p, dp);
    }
    __threadfence_block();
    for (int64_t e = e0; e < e1; ++e) {
        const float2 w = a.ws[e * a.H + h];
        const float b = a.bias ? a.bias[(a.eid ? a.eid[e] : e) * a.H + h] : 0.0f;
        const bool live = b != -__builtin_inff();
        const float ds = live ? w.x * (w.y - D) : 0.0f;
        const T* k = (const T*)a.k + a.col[e] * a.ks + (int64_t)g * a.Dk;
        for (int c = 0; c < kAttnMaxPer; ++c)
            if (live && c * 64 + lane < a.Dk)
                gq[c] = fmaf(ds, attn_ld(k + c * 64 + lane), gq[c]);
        if (lane == 0) {
            a.ws[e * a.H + h].y = ds;
            if (a.gbias) a.gbias[(a.eid ? a.eid[e] : e) * a.H + h] = ds;
        }
    }
    T* out = (T*)a.gq + (i * a.H + h) * (int64_t)a.Dk;
    for (int c = 0; c < kAttnMaxPer; ++c)
        if (c * 64 + lane < a.Dk) attn_st(out + c * 64 + lane, gq[c] * a.scale);
}

// gk, gv of one source and key/value head
template <typename T>
__global__ __launch_bounds__(256) void attn_bwd_src_kernel(AttnArgs a) {
    const int64_t u = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (u >= a.n_src * a.Hkv) return;
    const int lane = threadIdx.x & 63, g = (int)(u % a.Hkv), G = a.H / a.Hkv;
    const int64_t j = u / a.Hkv;
    float gk[kAttnMaxPer], gv[kAttnMaxPer];
    for (int c = 0; c < kAttnMaxPer; ++c) gk[c] = gv[c] = 0.0f;
    for (int64_t t = a.src_ptr[j]; t < a.src_ptr[j + 1]; ++t) {
        const int64_t i = a.src_dst[t], e = a.src_pos[t];
        for (int h = g * G; h < g * G + G; ++h) {
            const float b = a.bias ? a.bias[(a.eid ? a.eid[e] : e) * a.H + h] : 0.0f;
            if (b == -__builtin_inff()) continue;
            const float2 w = a.ws[e * a.H + h];
            const T* q = (const T*)a.q + i * a.qs + (int64_t)h * a.Dk;
            const T* go = (const T*)a.go + i * a.gs + (int64_t)h * a.Dv;
            for (int c = 0; c < kAttnMaxPer; ++c) {
                if (c * 64 + lane < a.Dk)
                    gk[c] = fmaf(w.y, attn_ld(q + c * 64 + lane), gk[c]);
                if (c * 64 + lane < a.Dv)
                    gv[c] = fmaf(w.x, attn_ld(go + c * 64 + lane), gv[c]);
            }
        }
    }
    T* ok = (T*)a.gk + (j * a.Hkv + g) * (int64_t)a.Dk;
    T* ov = (T*)a.gv + (j * a.Hkv + g) * (int64_t)a.Dv;
    for (int c = 0; c < kAttnMaxPer; ++c) {
        if (c * 64 + lane < a.Dk) attn_st(ok + c * 64 + lane, gk[c] * a.scale);
        if (c * 64 + lane < a.Dv) attn_st(ov + c * 64 + lane, gv[c]);
    }
}

static bool attn_shape_ok(int64_t n_dst, int64_t n_src, int64_t n_edges, int H, int Hkv, int Dk,
                          int Dv, int dtype) {
    return n_dst >= 0 && n_src >= 0 && n_edges >= 0 && H > 0 && Hkv > 0 && H % Hkv == 0 &&
           Dk > 0 && Dv > 0 && Dk <= 64 * kAttnMaxPer && Dv <= 64 * kAttnMaxPer &&
           (n_edges == 0 || (n_src > 0 && n_dst > 0)) && (dtype == 0 || dtype == 1) &&
           n_dst * (int64_t)H < ((int64_t)1 << 32) && n_src * (int64_t)Hkv < ((int64_t)1 << 32);
}

}  // namespace bmhip

using namespace bmhip;

extern "C" int batteries_neighbor_attention(
    const void* q, const void* k, const void* v, const float* bias, const int64_t* row_ptr,
    const int64_t* col, const int64_t* eid, void* out, float* stats, int64_t n_dst, int64_t n_src,
    int64_t n_edges, int H, int Hkv, int Dk, int Dv, int64_t q_stride, int64_t k_stride,
    int64_t v_stride, float scale, int dtype, hipStream_t stream) {
    if (!attn_shape_ok(n_dst, n_src, n_edges, H, Hkv, Dk, Dv, dtype)) return BM_ERR_ARG;
    if (n_dst == 0) return BM_OK;
    AttnArgs a{};
    a.q = q; a.k = k; a.v = v; a.bias = bias; a.row_ptr = row_ptr; a.col = col; a.eid = eid;
    a.out = out; a.stats = stats; a.n_dst = n_dst; a.n_src = n_src; a.H = H; a.Hkv = Hkv;
    a.Dk = Dk; a.Dv = Dv; a.qs = q_stride; a.ks = k_stride; a.vs = v_stride; a.scale = scale;
    const unsigned grid = (unsigned)ceil_div(n_dst * H, 4);
    if (dtype == 0) attn_fwd_kernel<float><<<grid, 256, 0, stream>>>(a);
    else attn_fwd_kernel<uint16_t><<<grid, 256, 0, stream>>>(a);
    return (int)hipGetLastError();
}

extern "C" size_t batteries_neighbor_attention_backward_workspace_bytes(int64_t n_edges, int H) {
    return (size_t)(n_edges > 0 ? n_edges : 0) * (size_t)H * sizeof(float2);
}

extern "C" int batteries_neighbor_attention_backward(
    const void* q, const void* k, const void* v, const float* bias, const float* stats,
    const void* grad_out, const int64_t* row_ptr, const int64_t* col, const int64_t* eid,
    const int64_t* src_ptr, const int64_t* src_dst, const int64_t* src_pos, void* grad_q,
    void* grad_k, void* grad_v, float* grad_bias, int64_t n_dst, int64_t n_src, int64_t n_edges,
    int H, int Hkv, int Dk, int Dv, int64_t q_stride, int64_t k_stride, int64_t v_stride,
    int64_t go_stride, float scale, int dtype, void* workspace, size_t workspace_bytes,
    hipStream_t stream) {
    if (!attn_shape_ok(n_dst, n_src, n_edges, H, Hkv, Dk, Dv, dtype)) return BM_ERR_ARG;
    if (workspace_bytes < batteries_neighbor_attention_backward_workspace_bytes(n_edges, H) ||
        (n_edges > 0 && !workspace))
        return BM_ERR_WORKSPACE;
    AttnArgs a{};
    a.q = q; a.k = k; a.v = v; a.go = grad_out; a.bias = bias; a.row_ptr = row_ptr; a.col = col;
    a.eid = eid; a.src_ptr = src_ptr; a.src_dst = src_dst; a.src_pos = src_pos;
    a.gq = grad_q; a.gk = grad_k; a.gv = grad_v; a.gbias = grad_bias;
    a.stats = const_cast<float*>(stats); a.ws = (float2*)workspace;
    a.n_dst = n_dst; a.n_src = n_src; a.H = H; a.Hkv = Hkv; a.Dk = Dk; a.Dv = Dv;
    a.qs = q_stride; a.ks = k_stride; a.vs = v_stride; a.gs = go_stride; a.scale = scale;
    const unsigned gd = (unsigned)ceil_div(n_dst * H, 4), gs = (unsigned)ceil_div(n_src * Hkv, 4);
    if (gd) {
        if (dtype == 0) attn_bwd_dst_kernel<float><<<gd, 256, 0, stream>>>(a);
        else attn_bwd_dst_kernel<uint16_t><<<gd, 256, 0, stream>>>(a);
    }
    if (gs) {
        if (dtype == 0) attn_bwd_src_kernel<float><<<gs, 256, 0, stream>>>(a);
        else attn_bwd_src_kernel<uint16_t><<<gs, 256, 0, stream>>>(a);
    }
    return (int)hipGetLastError();
}
