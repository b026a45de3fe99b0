// The operators of an equivariant transformer block in the _batmobile extension (registered by
// binding.cpp): attention over the edges of a graph, norms by degree with gate and residual,
// gradient clipping.  No reference counterpart.  Host code only, over include/batmobile_hip.h.
#include "binding_ops.h"

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <tuple>
#include <vector>

using namespace bmops;

namespace {

const int64_t* index_ptr(const Tensor& t, const Tensor& as, int64_t n, const char* name) {
    TORCH_CHECK(t.device() == as.device(), name, " must be on ", as.device());
    TORCH_CHECK(t.scalar_type() == torch::kInt64, name, " must be int64");
    TORCH_CHECK(t.is_contiguous() && t.dim() == 1, name, " must be contiguous and 1D");
    TORCH_CHECK(t.numel() == n, name, " must have ", n, " entries");
    return t.data_ptr<int64_t>();
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------

// Matrices [n, heads, D] as the kernels read them: heads of a row dense, rows at any stride below
// 2^30 elements, everything in units of 16 bytes.  Others are packed (head sizes padded with zeros, which add
// nothing to a product), all in one launch.
class Packer {
public:
    Tensor add(const Tensor& t) {
        const int64_t unit = 16 / t.element_size(), D = t.size(2);
        const bool dense = t.stride(2) == 1 && (t.size(1) == 1 || t.stride(1) == D) &&
                           (t.size(0) <= 1 ||
                            (t.stride(0) >= t.size(1) * D && t.stride(0) % unit == 0 &&
                             t.stride(0) < (int64_t)1 << 30)) &&
                           (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0;
        if (D % unit == 0 && (dense || t.numel() == 0)) return t.numel() ? t : t.contiguous();
        Tensor out = torch::empty({t.size(0), t.size(1), (D + unit - 1) / unit * unit}, t.options());
        packs_[count_++] = {t.data_ptr(), out.data_ptr(), t.size(0), t.stride(0), t.stride(1),
                            t.stride(2), (int32_t)t.size(1), (int32_t)D};
        return out;
    }
    // padded results cut to D
    Tensor cut(const Tensor& t, int64_t D) {
        if (t.size(2) == D) return t;
        Tensor out = torch::empty({t.size(0), t.size(1), D}, t.options());
        packs_[count_++] = {t.data_ptr(), out.data_ptr(), t.size(0), 0, 0, 0, (int32_t)t.size(1),
                            (int32_t)D};
        return out;
    }
    void run(int dtype, bool cut, const Tensor& as, const char* what) {
        if (count_)
            check_status(batteries_attention_pack(packs_, count_, dtype, cut, stream_of(as)), what);
        count_ = 0;
    }

private:
    batmobile_attention_pack packs_[4];
    int count_ = 0;
};
int64_t row_stride(const Tensor& t) {
    return t.size(0) <= 1 ? t.size(1) * t.size(2) : t.stride(0);
}
// An output of head size D made in units of 16 bytes, and cut to D
Tensor heads_like(const Tensor& as, int64_t n, int64_t heads, int64_t D) {
    const int64_t unit = 16 / as.element_size();
    return torch::empty({n, heads, (D + unit - 1) / unit * unit}, as.options());
}
// A side of a plan: (plan, items, parts) as attention_plan returns them.
batmobile_attention_side attn_side(const Tensor& plan, int64_t items, int64_t parts, int64_t rows,
                                   int64_t cols, int64_t edges, const Tensor& as) {
    TORCH_CHECK(plan.device() == as.device(), "the plan must be on ", as.device());
    TORCH_CHECK(plan.scalar_type() == torch::kInt32 && plan.is_contiguous() &&
                    (size_t)plan.numel() * 4 >= batteries_attention_plan_bytes(rows, edges),
                "the plan is not one of this many rows and edges");
    batmobile_attention_side s;
    s.n_rows = rows, s.n_cols = cols, s.n_edges = edges;
    s.plan = plan.data_ptr<int32_t>();
    s.n_items = (int32_t)items, s.n_parts = (int32_t)parts;
    return s;
}
const int32_t* opt_index32(const OptTensor& t, const Tensor& as, int64_t n, const char* name) {
    if (!t) return nullptr;
    TORCH_CHECK(t->device() == as.device() && t->scalar_type() == torch::kInt32 &&
                    t->is_contiguous() && t->numel() == n,
                name, " must be a contiguous int32 vector of ", n, " entries on ", as.device());
    return t->data_ptr<int32_t>();
}

// (plan, items, parts, flags): waits for the GPU to read the numbers back
std::tuple<Tensor, int64_t, int64_t, int64_t> attention_plan(const Tensor& row_ptr,
                                                             const Tensor& col,
                                                             const OptTensor& order,
                                                             int64_t n_cols, bool check) {
    TORCH_CHECK(row_ptr.is_cuda(), "row_ptr must be a CUDA tensor");
    TORCH_CHECK(row_ptr.numel() >= 1, "row_ptr must have at least one entry");
    const int64_t rows = row_ptr.numel() - 1, edges = col.numel();
    const int64_t* rp = index_ptr(row_ptr, row_ptr, rows + 1, "row_ptr");
    const int64_t* cp = index_ptr(col, row_ptr, edges, "col");
    const int64_t* op = order ? index_ptr(*order, row_ptr, rows, "order") : nullptr;
    const c10::DeviceGuard guard(row_ptr.device());
    const size_t n = batteries_attention_plan_bytes(rows, edges);
    TORCH_CHECK(n > 0 && n_cols >= 0, "attention_plan: up to 2^29 edges and 2^26 rows");
    Tensor plan = torch::empty({(int64_t)(n / 4)}, row_ptr.options().dtype(torch::kInt32));
    check_status(batteries_attention_plan(rp, cp, op, rows, n_cols, edges, check, plan.data_ptr(),
                                          n, stream_of(row_ptr)),
                 "attention_plan");
    const Tensor head = plan.slice(0, 0, 4).cpu();
    const int32_t* h = head.data_ptr<int32_t>();
    return {plan, h[0], h[1], h[2]};
}

struct AttnShape {
    int dtype, H, Hkv, Dk, Dv;
    int64_t n_dst, n_src, E;
};

AttnShape attn_shape(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& bias,
                     int64_t E) {
    AttnShape s;
    s.dtype = dtype_of(q, "q");
    TORCH_CHECK(q.dim() == 3, "q must be 3D [N_dst, H, Dk]");
    TORCH_CHECK(k.dim() == 3, "k must be 3D [N_src, H_kv, Dk]");
    TORCH_CHECK(v.dim() == 3, "v must be 3D [N_src, H_kv, Dv]");
    check_like(k, q, "k");
    check_like(v, q, "v");
    s.n_dst = q.size(0), s.n_src = k.size(0), s.E = E;
    TORCH_CHECK(v.size(0) == s.n_src, "k and v must have the same number of rows");
    TORCH_CHECK(k.size(1) == v.size(1), "k and v must have the same number of heads");
    TORCH_CHECK(q.size(1) > 0 && k.size(1) > 0 && q.size(1) % k.size(1) == 0,
                "the heads of q must be a multiple of those of k and v");
    TORCH_CHECK(q.size(2) == k.size(2), "q and k must have the same head size");
    TORCH_CHECK(q.size(2) >= 1 && q.size(2) <= 256 && v.size(2) >= 1 && v.size(2) <= 256,
                "head sizes must be in [1, 256]");
    s.H = (int)q.size(1), s.Hkv = (int)k.size(1), s.Dk = (int)q.size(2), s.Dv = (int)v.size(2);
    if (bias) {
        check_f32(*bias, q, "bias");
        TORCH_CHECK(bias->dim() == 2 && bias->size(0) == E && bias->size(1) == s.H,
                    "bias must be [E, H]");
    }
    return s;
}

// Edges x heads from which the bias (and its gradient) is brought to [H, E] by a kernel of its
// own: a wave takes one head of a tile, whose values lie H apart in [E, H], so every head reads
// (writes) all cache lines of the array, which shows once the array leaves the L2s.  A training
// step, heads of 32 in f32, as it lies and by head: 20,000 rows of 28, 2 heads 60 and 66 us, 4
// heads 96 and 98, 8 heads 191 and 170, 16 heads 517 and 354; 5000 rows, 8 heads 62 and 66, 16
// heads 104 and 102.
constexpr int64_t kByHead = 1 << 21;

// values [E, H] -> [H, E] in the order of edge_id, or back
Tensor attention_edges_by_head(const Tensor& values, const OptTensor& edge_id, bool back) {
    TORCH_CHECK(values.is_cuda(), "values must be a CUDA tensor");
    TORCH_CHECK(values.scalar_type() == torch::kFloat32 && values.dim() == 2 &&
                    values.is_contiguous(),
                "values must be a contiguous float32 matrix");
    const int64_t E = values.size(back ? 1 : 0), H = values.size(back ? 0 : 1);
    const c10::DeviceGuard guard(values.device());
    const int32_t* eid = opt_index32(edge_id, values, E, "edge_id");
    Tensor out = back ? torch::empty({E, H}, values.options()) : torch::empty({H, E}, values.options());
    if (E == 0 || H == 0) return out;
    check_status(batteries_attention_edges_by_head(values.data_ptr<float>(), eid,
                                                   out.data_ptr<float>(), E, (int)H, back,
                                                   stream_of(values)),
                 "attention_edges_by_head");
    return out;
}

// (out, stats, bias by head): the last two for the backward, if kept
std::tuple<Tensor, Tensor, Tensor> neighbor_attention(const Tensor& q_, const Tensor& k_,
                                                      const Tensor& v_, const OptTensor& bias_,
                                                      const Tensor& plan, int64_t items,
                                                      int64_t parts, int64_t E,
                                                      const OptTensor& edge_id, double scale,
                                                      bool keep_stats) {
    const AttnShape s = attn_shape(q_, k_, v_, bias_, E);
    const c10::DeviceGuard guard(q_.device());
    const batmobile_attention_side side = attn_side(plan, items, parts, s.n_dst, s.n_src, E, q_);
    const int32_t* eid = opt_index32(edge_id, q_, E, "edge_id");
    Packer packer;
    const Tensor q = packer.add(q_), k = packer.add(k_), v = packer.add(v_);
    packer.run(s.dtype, false, q, "neighbor_attention");
    Tensor bias, by_head;
    if (bias_) bias = bias_->contiguous();
    if (bias.defined() && (reinterpret_cast<uintptr_t>(bias.data_ptr()) & 15))
        bias = bias.clone(at::MemoryFormat::Contiguous);
    if (bias.defined() && s.H > 1 && E * s.H >= kByHead) {
        by_head = torch::empty({s.H, E}, bias.options());
        check_status(batteries_attention_edges_by_head(bias.data_ptr<float>(), eid,
                                                       by_head.data_ptr<float>(), E, s.H, 0,
                                                       stream_of(q)),
                     "neighbor_attention");
        bias = by_head;
    }
    const Tensor out = heads_like(q, s.n_dst, s.H, s.Dv);
    Tensor stats;
    if (keep_stats) stats = torch::empty({s.n_dst, s.H, 2}, q.options().dtype(torch::kFloat32));
    const int Dk = (int)q.size(2), Dv = (int)v.size(2);
    const size_t wsb = batteries_neighbor_attention_workspace_bytes(parts, s.H, Dv);
    Tensor ws;
    if (wsb) ws = bytes_on(q, wsb);
    check_status(batteries_neighbor_attention(
                     q.data_ptr(), k.data_ptr(), v.data_ptr(),
                     bias.defined() ? bias.data_ptr<float>() : nullptr, eid, by_head.defined(),
                     &side, out.data_ptr(), keep_stats ? stats.data_ptr<float>() : nullptr, s.H,
                     s.Hkv, Dk, Dv, row_stride(q), row_stride(k), row_stride(v), (float)scale,
                     s.dtype, wsb ? ws.data_ptr() : nullptr, wsb, stream_of(q)),
                 "neighbor_attention");
    const Tensor result = packer.cut(out, s.Dv);
    packer.run(s.dtype, true, q, "neighbor_attention");
    return {result, stats, keep_stats ? by_head : Tensor()};
}

// by_head: the forward's, in place of the bias.  src_*: the side of the sources, src_place the
// place of every edge in its order.
std::tuple<Tensor, Tensor, Tensor, Tensor> neighbor_attention_backward(
    const Tensor& q_, const Tensor& k_, const Tensor& v_, const OptTensor& bias_,
    const OptTensor& by_head, const Tensor& stats, const Tensor& grad_, const Tensor& row_ptr,
    const Tensor& plan,
    int64_t items, int64_t parts, const OptTensor& edge_id, const Tensor& src_plan,
    int64_t src_items, int64_t src_parts, const Tensor& src_place, double scale, bool need_bias) {
    const int64_t E = src_place.numel();
    const AttnShape s = attn_shape(q_, k_, v_, bias_, E);
    check_like(grad_, q_, "grad_out");
    TORCH_CHECK(grad_.dim() == 3 && grad_.size(0) == s.n_dst && grad_.size(1) == s.H &&
                    grad_.size(2) == s.Dv,
                "grad_out must have the shape of the output");
    check_f32(stats, q_, "stats");
    TORCH_CHECK(stats.is_contiguous() && stats.numel() == s.n_dst * s.H * 2,
                "stats must be [N_dst, H, 2]");
    const c10::DeviceGuard guard(q_.device());
    const batmobile_attention_side dst = attn_side(plan, items, parts, s.n_dst, s.n_src, E, q_);
    const batmobile_attention_side src =
        attn_side(src_plan, src_items, src_parts, s.n_src, s.n_dst, E, q_);
    const int32_t* eid = opt_index32(edge_id, q_, E, "edge_id");
    const int32_t* pos = opt_index32(src_place, q_, E, "src_place");
    const int64_t* rp = index_ptr(row_ptr, q_, s.n_dst + 1, "row_ptr");
    Packer packer;
    const Tensor q = packer.add(q_), k = packer.add(k_), v = packer.add(v_), go = packer.add(grad_);
    packer.run(s.dtype, false, q, "neighbor_attention_backward");
    Tensor bias, gbias;
    if (bias_) bias = bias_->contiguous();
    if (by_head) {
        check_f32(*by_head, q_, "bias by head");
        TORCH_CHECK(by_head->is_contiguous() && by_head->dim() == 2 && by_head->size(0) == s.H &&
                        by_head->size(1) == E,
                    "bias by head must be [H, E]");
        bias = *by_head;
    }
    if (need_bias && bias.defined())
        gbias = torch::empty({E, s.H}, q.options().dtype(torch::kFloat32));
    const Tensor gq = heads_like(q, s.n_dst, s.H, s.Dk);
    const Tensor gk = heads_like(q, s.n_src, s.Hkv, s.Dk);
    const Tensor gv = heads_like(q, s.n_src, s.Hkv, s.Dv);
    const int Dk = (int)q.size(2), Dv = (int)v.size(2);
    const size_t wsb = batteries_neighbor_attention_backward_workspace_bytes(
        E, parts, src_parts, s.H, s.Hkv, Dk, Dv);
    const Tensor ws = bytes_on(q, wsb);
    check_status(
        batteries_neighbor_attention_backward(
            q.data_ptr(), k.data_ptr(), v.data_ptr(),
            bias.defined() ? bias.data_ptr<float>() : nullptr, stats.data_ptr<float>(),
            go.data_ptr(), rp, eid, by_head.has_value(), &dst, &src, pos, gq.data_ptr(),
            gk.data_ptr(), gv.data_ptr(),
            gbias.defined() ? gbias.data_ptr<float>() : nullptr, s.H, s.Hkv, Dk, Dv,
            row_stride(q), row_stride(k), row_stride(v), row_stride(go), (float)scale, s.dtype,
            ws.data_ptr(), wsb, stream_of(q)),
        "neighbor_attention_backward");
    const Tensor rq = packer.cut(gq, s.Dk), rk = packer.cut(gk, s.Dk), rv = packer.cut(gv, s.Dv);
    packer.run(s.dtype, true, q, "neighbor_attention_backward");
    return {rq, rk, rv, gbias};
}

// ---------------------------------------------------------------------------
// norms by degree
// ---------------------------------------------------------------------------

void check_features(const Tensor& x, const char* name) {
    TORCH_CHECK(x.dim() == 3 && x.size(2) == 16, name, " must be 3D [N, C, 16]");
    TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= 2048, name, " must have 1 to 2048 channels");
}
Tensor weight4(const Tensor& w, const Tensor& x, const char* name) {
    check_f32(w, x, name);
    TORCH_CHECK(w.dim() == 2 && w.size(0) == 4 && w.size(1) == x.size(1), name,
                " must be [4, C]");
    return w.contiguous();
}
// (h, n, rs); y none: n = norm(x) alone, h undefined
std::tuple<Tensor, Tensor, Tensor> gated_residual_norm(const Tensor& x_, const OptTensor& y_,
                                                       const OptTensor& gate_,
                                                       const OptTensor& scale_,
                                                       const OptTensor& w_post_,
                                                       const OptTensor& w_pre_, double eps,
                                                       bool keep_stats) {
    const int dt = dtype_of(x_, "x");
    check_features(x_, "x");
    TORCH_CHECK(y_ || w_pre_, "one of y and weight_pre is needed");
    TORCH_CHECK(eps >= 0.0, "eps must not be negative");
    const int64_t N = x_.size(0);
    const int C = (int)x_.size(1);
    const c10::DeviceGuard guard(x_.device());
    const Tensor x = rows4(x_);
    Tensor y, gate, scale, w_post, w_pre, h, n, rs;
    if (y_) {
        TORCH_CHECK(scale_ && w_post_, "y needs scale and weight_post");
        check_same(*y_, x_, "y");
        y = rows4(*y_);
        check_f32(*scale_, x_, "scale");
        TORCH_CHECK(scale_->dim() == 1 && scale_->size(0) == C, "scale must be [C]");
        scale = scale_->contiguous();
        w_post = weight4(*w_post_, x_, "weight_post");
        if (gate_) {
            check_like(*gate_, x_, "gate");
            TORCH_CHECK(gate_->dim() == 3 && gate_->size(0) == N && gate_->size(1) == C &&
                            gate_->size(2) == 4,
                        "gate must be [N, C, 4]");
            gate = gate_->contiguous();
        }
        h = torch::empty_like(x);
    }
    if (w_pre_) {
        w_pre = weight4(*w_pre_, x_, "weight_pre");
        n = torch::empty_like(x);
    }
    if (keep_stats) rs = torch::empty({N, 8}, x.options().dtype(torch::kFloat32));
    // a tensor without elements has no address, which would read as "not given"
    if (N > 0)
        check_status(batteries_gated_residual_norm(x.data_ptr(), opt_ptr(y), opt_ptr(gate),
                                                   opt_f32(scale), opt_f32(w_post),
                                                   opt_f32(w_pre), opt_ptr(h), opt_ptr(n),
                                                   opt_f32(rs), N, C, (float)eps, dt,
                                                   stream_of(x)),
                     "gated_residual_norm");
    return {h, n, rs};
}

// (gx, gy, ggate, gscale, gw_post, gw_pre)
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor, Tensor> gated_residual_norm_backward(
    const OptTensor& gh_, const OptTensor& gn_, const Tensor& x_, const OptTensor& y_,
    const OptTensor& gate_, const OptTensor& scale_, const OptTensor& w_post_,
    const OptTensor& w_pre_, const Tensor& rs) {
    const int dt = dtype_of(x_, "x");
    check_features(x_, "x");
    const int64_t N = x_.size(0);
    const int C = (int)x_.size(1);
    TORCH_CHECK(y_ || w_pre_, "one of y and weight_pre is needed");
    TORCH_CHECK(!w_pre_ || gn_, "weight_pre needs the gradient of n");
    TORCH_CHECK(w_pre_ || gh_, "the gradient of h is needed");
    check_f32(rs, x_, "rs");
    TORCH_CHECK(rs.is_contiguous() && rs.numel() == N * 8, "rs must be [N, 8]");
    const c10::DeviceGuard guard(x_.device());
    const Tensor x = rows4(x_);
    Tensor gh, gn, y, gate, scale, w_post, w_pre, gx, gy, ggate, gscale, gw_post, gw_pre;
    gx = torch::empty_like(x);
    if (gh_) check_same(*gh_, x_, "grad_h"), gh = rows4(*gh_);
    if (w_pre_) {
        check_same(*gn_, x_, "grad_n");
        gn = rows4(*gn_);
        w_pre = weight4(*w_pre_, x_, "weight_pre");
        gw_pre = torch::empty_like(w_pre);
    }
    if (y_) {
        TORCH_CHECK(scale_ && w_post_, "y needs scale and weight_post");
        check_same(*y_, x_, "y");
        y = rows4(*y_);
        check_f32(*scale_, x_, "scale");
        TORCH_CHECK(scale_->numel() == C, "scale must be [C]");
        scale = scale_->contiguous();
        w_post = weight4(*w_post_, x_, "weight_post");
        gy = torch::empty_like(y);
        gscale = torch::empty_like(scale);
        gw_post = torch::empty_like(w_post);
        if (gate_) {
            check_like(*gate_, x_, "gate");
            TORCH_CHECK(gate_->numel() == N * C * 4, "gate must be [N, C, 4]");
            gate = gate_->contiguous();
            ggate = torch::empty_like(gate);
        }
    }
    if (N == 0) {
        for (Tensor* t : {&gscale, &gw_post, &gw_pre})
            if (t->defined()) t->zero_();
        return {gx, gy, ggate, gscale, gw_post, gw_pre};
    }
    const size_t wsb = batteries_gated_residual_norm_backward_workspace_bytes(N, C);
    const Tensor ws = bytes_on(x, wsb);
    check_status(batteries_gated_residual_norm_backward(
                     opt_ptr(gh), opt_ptr(gn), x.data_ptr(), opt_ptr(y), opt_ptr(gate),
                     opt_f32(scale), opt_f32(w_post), opt_f32(w_pre), rs.data_ptr<float>(),
                     gx.data_ptr(), opt_ptr(gy), opt_ptr(ggate), opt_f32(gscale),
                     opt_f32(gw_post), opt_f32(gw_pre), N, C, dt, ws.data_ptr(), wsb,
                     stream_of(x)),
                 "gated_residual_norm_backward");
    return {gx, gy, ggate, gscale, gw_post, gw_pre};
}

// ---------------------------------------------------------------------------
// autograd of both.  Nodes in C++: a training step of a small system is the host's time, and
// Python's part of a node takes longer than the kernels (a step through the norm of 141 atoms, 8
// channels: 61 us against 83 with a node in Python, its two calls 15 us of either; attention of 39
// atoms, 16 heads, 88 against 112; the norm of 1000 atoms without gradients 4.8 against 7.5).
// ---------------------------------------------------------------------------

// A plan as the Python class holds it: both sides, (plan, items, parts), and its index arrays.
struct PlanRef {
    Tensor plan, row_ptr, edge_id, src_plan, src_place;
    int64_t items, parts, src_items, src_parts, edges;
};

struct AttentionNode : torch::autograd::Function<AttentionNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                          const OptTensor& bias, const PlanRef& p, double scale) {
        auto [out, stats, by_head] = neighbor_attention(q, k, v, bias, p.plan, p.items, p.parts,
                                                        p.edges, opt_of(p.edge_id), scale, true);
        const bool need_bias = bias && bias->requires_grad();
        // a bias brought to [H, E] takes the place of the caller's
        ctx->save_for_backward({q, k, v, by_head.defined() ? Tensor() : tensor_of(bias), by_head,
                                stats});
        // not saved variables: a plan may have been made under inference mode
        ctx->saved_data["plan"] =
            std::vector<Tensor>{p.row_ptr, p.plan, p.edge_id, p.src_plan, p.src_place};
        ctx->saved_data["sizes"] =
            std::vector<int64_t>{p.items, p.parts, p.src_items, p.src_parts, need_bias};
        ctx->saved_data["scale"] = scale;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const bool create_graph = at::GradMode::is_enabled();
        const torch::NoGradGuard no_grad;
        refuse_tangents({&grads[0]}, "the gradient of neighbor_attention");
        const variable_list s = ctx->get_saved_variables();
        const std::vector<Tensor> p = ctx->saved_data["plan"].toTensorVector();
        const std::vector<int64_t> n = ctx->saved_data["sizes"].toIntVector();
        auto [gq, gk, gv, gb] = neighbor_attention_backward(
            s[0], s[1], s[2], opt_of(s[3]), opt_of(s[4]), s[5], grads[0], p[0], p[1], n[0], n[1],
            opt_of(p[2]), p[3], n[2], n[3], p[4], ctx->saved_data["scale"].toDouble(), n[4] != 0);
        variable_list g =
            first_order({gq, gk, gv, gb}, create_graph, "neighbor_attention");
        g.resize(6);
        return g;
    }
};

// source_side: called for the sources' side (plan, items, parts, place) where gradients are wanted
Tensor neighbor_attention_autograd(const Tensor& q, const Tensor& k, const Tensor& v,
                                   const OptTensor& bias, const Tensor& plan, int64_t items,
                                   int64_t parts, int64_t E, const OptTensor& edge_id,
                                   const Tensor& row_ptr, const pybind11::function& source_side,
                                   double scale) {
    refuse_tangents({&q, &k, &v, ptr_of(bias)}, "neighbor_attention");
    if (!wants_grad({&q, &k, &v, ptr_of(bias)}))
        return std::get<0>(neighbor_attention(q, k, v, bias, plan, items, parts, E, edge_id, scale,
                                              false));
    const auto src = source_side().cast<std::tuple<Tensor, int64_t, int64_t, Tensor>>();
    return AttentionNode::apply(q, k, v, bias,
                                PlanRef{plan, row_ptr, tensor_of(edge_id), std::get<0>(src),
                                        std::get<3>(src), items, parts, std::get<1>(src),
                                        std::get<2>(src), E},
                                scale);
}

struct NormNode : torch::autograd::Function<NormNode> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& y,
                                 const OptTensor& gate, const OptTensor& scale,
                                 const OptTensor& w_post, const OptTensor& w_pre, double eps) {
        auto [h, n, rs] = gated_residual_norm(x, y, gate, scale, w_post, w_pre, eps, true);
        ctx->save_for_backward({x, tensor_of(y), tensor_of(gate), tensor_of(scale),
                                tensor_of(w_post), tensor_of(w_pre), rs});
        ctx->set_materialize_grads(false);
        if (!h.defined()) return {n};
        if (!n.defined()) return {h};
        return {h, n};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const bool create_graph = at::GradMode::is_enabled();
        const torch::NoGradGuard no_grad;
        refuse_tangents({&grads.front(), &grads.back()}, "the gradient of gated_residual_norm");
        const variable_list s = ctx->get_saved_variables();
        const Tensor gh = s[1].defined() ? grads.front() : Tensor();
        const Tensor gn = s[5].defined() ? grads.back() : Tensor();
        if (!gh.defined() && !gn.defined()) return variable_list(7);
        // only h is used further on: no part of n
        const Tensor w_pre = gn.defined() ? s[5] : Tensor();
        auto [gx, gy, gg, gs, gpost, gpre] = gated_residual_norm_backward(
            opt_of(gh), opt_of(gn), s[0], opt_of(s[1]), opt_of(s[2]), opt_of(s[3]), opt_of(s[4]),
            opt_of(w_pre), s[6]);
        if (s[5].defined() && !gn.defined()) gpre = torch::zeros_like(s[5]);
        variable_list g = first_order({gx, gy, gg, gs, gpost, gpre}, create_graph,
                                      "gated_residual_norm");
        g.resize(7);
        return g;
    }
};

// [n], [h] or [h, n]
variable_list gated_residual_norm_autograd(const Tensor& x, const OptTensor& y,
                                           const OptTensor& gate, const OptTensor& scale,
                                           const OptTensor& w_post, const OptTensor& w_pre,
                                           double eps) {
    refuse_tangents({&x, ptr_of(y), ptr_of(gate), ptr_of(scale), ptr_of(w_post), ptr_of(w_pre)},
                    "gated_residual_norm");
    if (wants_grad({&x, ptr_of(y), ptr_of(gate), ptr_of(scale), ptr_of(w_post), ptr_of(w_pre)}))
        return NormNode::apply(x, y, gate, scale, w_post, w_pre, eps);
    auto [h, n, rs] = gated_residual_norm(x, y, gate, scale, w_post, w_pre, eps, false);
    if (!h.defined()) return {n};
    if (!n.defined()) return {h};
    return {h, n};
}

// ---------------------------------------------------------------------------
// gradient clipping
// ---------------------------------------------------------------------------

// Which outs share memory with another out, with another gradient, or with their own gradient at
// another place (empty: none): the kernels' workgroups read and write in no order, so those go through
// a buffer.  in, out: the addresses of dense tensors.
std::vector<bool> overlapping_outs(const std::vector<const void*>& in,
                                   const std::vector<void*>& out,
                                   const std::vector<int64_t>& bytes) {
    struct Range {
        uintptr_t begin;
        size_t i;                          // of a gradient, or behind those of an out
    };
    const size_t n = in.size();
    std::vector<Range> all;
    all.reserve(2 * n);
    for (size_t i = 0; i < n; ++i) {
        if (bytes[i] == 0) continue;
        all.push_back({reinterpret_cast<uintptr_t>(out[i]), n + i});
        if (in[i] != out[i]) all.push_back({reinterpret_cast<uintptr_t>(in[i]), i});
    }
    std::sort(all.begin(), all.end(),
              [](const Range& a, const Range& b) { return a.begin < b.begin; });
    std::vector<bool> overlaps;
    auto end_of = [&](size_t k) { return all[k].begin + (uintptr_t)bytes[all[k].i < n ? all[k].i : all[k].i - n]; };
    for (size_t i = 0, j; i < all.size(); i = j) {     // runs of ranges that overlap
        uintptr_t end = end_of(i);
        for (j = i + 1; j < all.size() && all[j].begin < end; ++j) end = std::max(end, end_of(j));
        if (j - i == 1) continue;
        overlaps.resize(n);
        for (size_t k = i; k < j; ++k)
            if (all[k].i >= n) overlaps[all[k].i - n] = true;
    }
    return overlaps;
}

// (norm, clipped): the norm as a tensor without dimensions; the clipped gradients in outs
// (which may be the gradients; then nothing is returned for them) or in new tensors.  A strided
// view with gaps, an out of another layout than its gradient, or one that shares memory with
// others, goes through a dense copy: every gradient is read before any result is seen.
std::tuple<Tensor, std::vector<Tensor>> clip_grad_norm(
    const std::vector<Tensor>& grads, double max_norm,
    const c10::optional<std::vector<Tensor>>& outs) {
    TORCH_CHECK(max_norm >= 0.0, "max_norm must not be negative");
    TORCH_CHECK(!grads.empty(), "at least one tensor is needed");
    TORCH_CHECK(!outs || outs->size() == grads.size(), "out must hold one tensor per gradient");
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode())
        for (const Tensor& g : grads) refuse_tangent(&g, "clip_grad_norm");
    const torch::NoGradGuard no_grad;
    const size_t n = grads.size();
    std::vector<const void*> in(n);
    std::vector<void*> out(n);
    std::vector<int64_t> numel(n), bytes(n);
    std::vector<int> dt(n);
    std::vector<Tensor> dense(n), into(n);
    TORCH_CHECK(grads[0].is_cuda(), "a gradient must be a CUDA tensor");
    const c10::DeviceGuard guard(grads[0].device());
    for (size_t i = 0; i < n; ++i) {
        const Tensor* g = &grads[i];
        dt[i] = dtype_of(*g, "a gradient");
        TORCH_CHECK(g->device() == grads[0].device(), "the gradients must be on one device");
        if (!g->is_non_overlapping_and_dense()) dense[i] = g->contiguous(), g = &dense[i];
        const Tensor* o = outs ? &(*outs)[i] : nullptr;
        if (o) {
            check_like(*o, *g, "out");
            TORCH_CHECK(o->sizes() == g->sizes(), "out must have the shapes of the gradients");
        }
        if (!o || o->strides() != g->strides()) into[i] = torch::empty_like(*g), o = &into[i];
        in[i] = g->data_ptr(), out[i] = o->data_ptr(), numel[i] = g->numel();
        bytes[i] = numel[i] * (dt[i] ? 2 : 4);
    }
    if (outs) {
        const std::vector<bool> overlaps = overlapping_outs(in, out, bytes);
        for (size_t i = 0; i < overlaps.size(); ++i)
            if (overlaps[i] && !into[i].defined())
                into[i] = torch::empty_like((*outs)[i]), out[i] = into[i].data_ptr();
    }
    Tensor norm = torch::empty({}, grads[0].options().dtype(torch::kFloat32));
    int64_t elements = 0;
    for (const int64_t k : numel) elements += k;
    const size_t wsb = batteries_clip_grad_norm_workspace_bytes((int64_t)n, elements);
    const Tensor ws = bytes_on(grads[0], wsb);
    check_status(batteries_clip_grad_norm(in.data(), out.data(), numel.data(), dt.data(),
                                          (int64_t)n, (float)max_norm, norm.data_ptr<float>(),
                                          ws.data_ptr(), wsb, stream_of(grads[0])),
                 "clip_grad_norm");
    if (!outs) return {norm, into};
    for (size_t i = 0; i < n; ++i) {
        const Tensor& o = (*outs)[i];
        if (into[i].defined()) o.copy_(into[i]);
        // written by address: whoever saved it for a backward is told as by torch's own operators
        else if (!o.is_inference()) torch::autograd::impl::bump_version(o);
    }
    return {norm, {}};
}

}  // namespace

void register_block_ops(pybind11::module_& m) {
    namespace py = pybind11;
    m.def("attention_plan", &attention_plan, py::arg("row_ptr"), py::arg("col"),
          py::arg("order"), py::arg("n_cols"), py::arg("check") = true,
          "tiles of a graph side for the attention -> (plan, items, parts, flags)");
    m.def("attention_edges_by_head", &attention_edges_by_head, py::arg("values"),
          py::arg("edge_id") = py::none(), py::arg("back") = false,
          "values [E, H] (row edge_id[e] of edge e) -> [H, E]; back: the other way");
    m.def("neighbor_attention", &neighbor_attention, py::arg("q"), py::arg("k"), py::arg("v"),
          py::arg("bias"), py::arg("plan"), py::arg("items"), py::arg("parts"),
          py::arg("num_edges"), py::arg("edge_id"), py::arg("scale"),
          py::arg("keep_stats") = false,
          "softmax attention over the edges of each row -> (out, stats or None, bias [H, E] or None)");
    m.def("neighbor_attention_backward", &neighbor_attention_backward, py::arg("q"), py::arg("k"),
          py::arg("v"), py::arg("bias"), py::arg("by_head"), py::arg("stats"), py::arg("grad_out"),
          py::arg("row_ptr"), py::arg("plan"), py::arg("items"), py::arg("parts"),
          py::arg("edge_id"), py::arg("src_plan"), py::arg("src_items"), py::arg("src_parts"),
          py::arg("src_place"), py::arg("scale"), py::arg("need_bias") = true,
          "(grad_q, grad_k, grad_v, grad_bias or None)");
    m.def("gated_residual_norm", &gated_residual_norm, py::arg("x"), py::arg("y"),
          py::arg("gate"), py::arg("scale"), py::arg("weight_post"), py::arg("weight_pre"),
          py::arg("eps"), py::arg("keep_stats") = false,
          "h = x + scale sigmoid(gate) norm(y), n = norm(h) -> (h, n, rs); y None: n = norm(x)");
    m.def("gated_residual_norm_backward", &gated_residual_norm_backward, py::arg("grad_h"),
          py::arg("grad_n"), py::arg("x"), py::arg("y"), py::arg("gate"), py::arg("scale"),
          py::arg("weight_post"), py::arg("weight_pre"), py::arg("rs"),
          "(grad_x, grad_y, grad_gate, grad_scale, grad_weight_post, grad_weight_pre)");
    m.def("neighbor_attention_autograd", &neighbor_attention_autograd, py::arg("q"), py::arg("k"),
          py::arg("v"), py::arg("bias"), py::arg("plan"), py::arg("items"), py::arg("parts"),
          py::arg("num_edges"), py::arg("edge_id"), py::arg("row_ptr"), py::arg("source_side"),
          py::arg("scale"), "neighbor_attention with gradients -> out");
    m.def("gated_residual_norm_autograd", &gated_residual_norm_autograd, py::arg("x"),
          py::arg("y"), py::arg("gate"), py::arg("scale"), py::arg("weight_post"),
          py::arg("weight_pre"), py::arg("eps"),
          "gated_residual_norm with gradients -> [n], [h] or [h, n]");
    m.def("clip_grad_norm", &clip_grad_norm, py::arg("grads"), py::arg("max_norm"),
          py::arg("out") = py::none(),
          "(norm of all tensors together, the tensors scaled to max_norm)");
}
