// The operators beside attention in the _batmobile extension (registered by binding.cpp): the learned
// bias by distance, layer norm, channel mixing by degree, the gated activation and the 8-bit form of
// activations.  No reference counterpart.  Host code only, over include/batmobile_hip.h.
#include "binding_ops.h"

#include <string>
#include <tuple>
#include <vector>

using namespace bmops;

namespace {

void check_features(const Tensor& x, const char* name) {
    TORCH_CHECK(x.dim() == 3 && x.size(2) == 16, name, " must be 3D [N, C, 16]");
    TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= 2048, name, " must have 1 to 2048 channels");
}
// Whether a layer keeps its input in 8 bits for the backward
bool keeps_8bit(const c10::optional<std::string>& checkpoint) {
    TORCH_CHECK(!checkpoint || *checkpoint == "e4m3", "checkpoint must be None or \"e4m3\"");
    return checkpoint.has_value();
}

// ---------------------------------------------------------------------------
// bias by distance
// ---------------------------------------------------------------------------

void check_bias(const Tensor& lengths, const Tensor& boundaries, const Tensor& table,
                c10::optional<double> cutoff) {
    TORCH_CHECK(lengths.is_cuda(), "lengths must be a CUDA tensor");
    check_f32(lengths, lengths, "lengths");
    check_f32(boundaries, lengths, "boundaries");
    check_f32(table, lengths, "table");
    TORCH_CHECK(lengths.dim() == 1, "lengths must be 1D [E]");
    TORCH_CHECK(table.dim() == 2 && table.size(0) >= 1 && table.size(0) <= 4096 && table.size(1) >= 1 &&
                    table.size(1) <= 1024,
                "table must be [B, H], up to 4096 buckets and 1024 heads");
    TORCH_CHECK(boundaries.dim() == 1 && boundaries.size(0) == table.size(0) - 1,
                "boundaries must be [B - 1]");
    TORCH_CHECK(!cutoff || ((float)*cutoff >= 1e-30f && (float)*cutoff <= 1e30f),
                "cutoff must be positive and finite (1e-30 to 1e30)");
}

// (bias [E, H], buckets [E] int16 or none)
std::tuple<Tensor, Tensor> distance_bias(const Tensor& lengths_, const Tensor& boundaries_,
                                         const Tensor& table_, c10::optional<double> cutoff,
                                         bool keep_buckets) {
    check_bias(lengths_, boundaries_, table_, cutoff);
    const c10::DeviceGuard guard(lengths_.device());
    const Tensor lengths = lengths_.contiguous(), boundaries = boundaries_.contiguous(),
                 table = rows4(table_);
    const int64_t E = lengths.size(0), B = table.size(0), H = table.size(1);
    const Tensor bias = torch::empty({E, H}, lengths.options());
    Tensor buckets;
    if (keep_buckets) buckets = torch::empty({E}, lengths.options().dtype(torch::kInt16));
    check_status(batteries_distance_bias(opt_f32(lengths), opt_f32(boundaries), table.data_ptr<float>(),
                                         bias.data_ptr<float>(), (uint16_t*)opt_ptr(buckets), E, (int)H,
                                         (int)B, (float)cutoff.value_or(0.0), stream_of(lengths)),
                 "distance_bias");
    return {bias, buckets};
}

// (grad_table, grad_lengths), each if wanted
std::tuple<Tensor, Tensor> distance_bias_backward(const OptTensor& lengths_, const OptTensor& buckets,
                                                  const Tensor& grad_, int64_t B, double cutoff,
                                                  bool need_table, bool need_lengths) {
    TORCH_CHECK(grad_.is_cuda(), "grad must be a CUDA tensor");
    check_f32(grad_, grad_, "grad");
    TORCH_CHECK(grad_.dim() == 2 && B >= 1, "grad must be [E, H]");
    const int64_t E = grad_.size(0), H = grad_.size(1);
    if (need_table)
        TORCH_CHECK(buckets && buckets->device() == grad_.device() &&
                        buckets->scalar_type() == torch::kInt16 && buckets->is_contiguous() &&
                        buckets->numel() == E,
                    "buckets must be int16 [E]");
    const c10::DeviceGuard guard(grad_.device());
    const Tensor grad = rows4(grad_);
    Tensor lengths, gt, gl, ws;
    if (need_lengths) {
        TORCH_CHECK(lengths_ && lengths_->dim() == 1 && lengths_->size(0) == E, "lengths must be [E]");
        check_f32(*lengths_, grad_, "lengths");
        lengths = lengths_->contiguous();
    }
    size_t wsb = 0;
    if (need_table) {
        gt = torch::empty({B, H}, grad.options());
        wsb = batteries_distance_bias_backward_workspace_bytes(E, (int)H, (int)B);
        ws = bytes_on(grad, wsb);
    }
    if (need_lengths) gl = torch::empty({E}, grad.options());
    check_status(batteries_distance_bias_backward(
                     opt_f32(lengths), need_table ? (const uint16_t*)buckets->data_ptr() : nullptr,
                     opt_f32(grad), opt_f32(gt), opt_f32(gl), E, (int)H, (int)B, (float)cutoff,
                     opt_ptr(ws), wsb, stream_of(grad)),
                 "distance_bias_backward");
    return {gt, gl};
}

struct BiasNode : torch::autograd::Function<BiasNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& lengths, const Tensor& boundaries,
                          const Tensor& table, c10::optional<double> cutoff) {
        const bool need_table = table.requires_grad(), need_lengths = lengths.requires_grad();
        auto [bias, buckets] = distance_bias(lengths, boundaries, table, cutoff, need_table);
        const bool by_cutoff = need_lengths && cutoff.has_value();
        ctx->save_for_backward({by_cutoff ? lengths : Tensor(), buckets});
        ctx->saved_data["cutoff"] = cutoff.value_or(0.0);
        ctx->saved_data["sizes"] = std::vector<int64_t>{table.size(0), need_table, need_lengths};
        return bias;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const bool create_graph = at::GradMode::is_enabled();
        const torch::NoGradGuard no_grad;
        refuse_tangents({&grads[0]}, "the gradient of distance_bias");
        const variable_list s = ctx->get_saved_variables();
        const std::vector<int64_t> n = ctx->saved_data["sizes"].toIntVector();
        const double cutoff = ctx->saved_data["cutoff"].toDouble();
        auto [gt, gl] = distance_bias_backward(opt_of(s[0]), opt_of(s[1]), grads[0], n[0], cutoff,
                                               n[1] != 0, n[2] != 0 && cutoff > 0.0);
        if (n[2] && !gl.defined()) gl = torch::zeros({grads[0].size(0)}, grads[0].options());
        variable_list g = first_order({gl, Tensor(), gt}, create_graph, "distance_bias");
        g.resize(4);
        return g;
    }
};

Tensor distance_bias_autograd(const Tensor& lengths, const Tensor& boundaries, const Tensor& table,
                              c10::optional<double> cutoff) {
    refuse_tangents({&lengths, &boundaries, &table}, "distance_bias");
    if (!wants_grad({&lengths, &boundaries, &table}))
        return std::get<0>(distance_bias(lengths, boundaries, table, cutoff, false));
    TORCH_CHECK(!boundaries.requires_grad(), "distance_bias: boundaries have no gradient");
    return BiasNode::apply(lengths, boundaries, table, cutoff);
}

// ---------------------------------------------------------------------------
// layer norm
// ---------------------------------------------------------------------------

struct Rows {
    Tensor t;
    int64_t rows, stride, step;
    int D;
};
// x [..., D] as rows at one stride, packed if there is none
Rows rows_of(const Tensor& x) {
    Rows r;
    const int64_t d = x.size(-1);
    r.t = x, r.D = (int)d, r.rows = x.numel() / d;
    r.step = d > 1 ? x.stride(-1) : 1;
    r.stride = d;
    int64_t next = -1;                                  // stride that the next outer dimension must have
    for (int64_t i = x.dim() - 2; i >= 0; --i) {
        if (x.size(i) == 1) continue;
        if (next < 0) r.stride = x.stride(i);
        else if (x.stride(i) != next) {
            r.t = x.contiguous(), r.stride = d, r.step = 1;
            return r;
        }
        next = x.stride(i) * x.size(i);
    }
    return r;
}

void check_layer_norm(const Tensor& x, const Tensor& weight, const OptTensor& bias, double eps) {
    dtype_of(x, "x");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= 8192, "x must be [..., D], D in [1, 8192]");
    check_f32(weight, x, "weight");
    TORCH_CHECK(weight.dim() == 1 && weight.size(0) == x.size(-1), "weight must be [D]");
    if (bias) {
        check_f32(*bias, x, "bias");
        TORCH_CHECK(bias->dim() == 1 && bias->size(0) == x.size(-1), "bias must be [D]");
    }
    TORCH_CHECK(eps >= 0.0, "eps must not be negative");
}

Tensor layer_norm(const Tensor& x, const Tensor& weight_, const OptTensor& bias_, double eps) {
    check_layer_norm(x, weight_, bias_, eps);
    const c10::DeviceGuard guard(x.device());
    const Rows r = rows_of(x);
    const Tensor weight = weight_.contiguous();
    Tensor bias;
    if (bias_) bias = bias_->contiguous();
    const Tensor y = torch::empty(x.sizes(), x.options());
    check_status(batteries_layer_norm(opt_ptr(r.t), weight.data_ptr<float>(), opt_f32(bias), opt_ptr(y),
                                      r.rows, r.D, r.stride, r.step, (float)eps, dtype_of(x, "x"),
                                      stream_of(x)),
                 "layer_norm");
    return y;
}

// (grad_x, grad_weight, grad_bias or none)
std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const Tensor& grad_, const Tensor& x,
                                                       const Tensor& weight_, bool need_bias,
                                                       double eps) {
    check_layer_norm(x, weight_, OptTensor(), eps);
    check_same(grad_, x, "grad");
    const c10::DeviceGuard guard(x.device());
    const Rows r = rows_of(x);
    const Tensor weight = weight_.contiguous(), grad = grad_.contiguous();
    const Tensor gx = torch::empty(x.sizes(), x.options()), gw = torch::empty_like(weight);
    Tensor gb;
    if (need_bias) gb = torch::empty_like(weight);
    const size_t wsb = batteries_layer_norm_backward_workspace_bytes(r.rows, r.D);
    const Tensor ws = bytes_on(x, wsb);
    check_status(batteries_layer_norm_backward(opt_ptr(r.t), weight.data_ptr<float>(), opt_ptr(grad),
                                               opt_ptr(gx), gw.data_ptr<float>(), opt_f32(gb), r.rows,
                                               r.D, r.stride, r.step, (float)eps, dtype_of(x, "x"),
                                               ws.data_ptr(), wsb, stream_of(x)),
                 "layer_norm_backward");
    return {gx, gw, gb};
}

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                          const OptTensor& bias, double eps) {
        const Tensor y = layer_norm(x, weight, bias, eps);
        ctx->save_for_backward({x, weight});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["bias"] = bias.has_value();
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const bool create_graph = at::GradMode::is_enabled();
        const torch::NoGradGuard no_grad;
        refuse_tangents({&grads[0]}, "the gradient of layer_norm");
        const variable_list s = ctx->get_saved_variables();
        auto [gx, gw, gb] = layer_norm_backward(grads[0], s[0], s[1], ctx->saved_data["bias"].toBool(),
                                                ctx->saved_data["eps"].toDouble());
        variable_list g = first_order({gx, gw, gb}, create_graph, "layer_norm");
        g.resize(4);
        return g;
    }
};

Tensor layer_norm_autograd(const Tensor& x, const Tensor& weight, const OptTensor& bias, double eps) {
    refuse_tangents({&x, &weight, ptr_of(bias)}, "layer_norm");
    if (wants_grad({&x, &weight, ptr_of(bias)})) return LayerNormNode::apply(x, weight, bias, eps);
    return layer_norm(x, weight, bias, eps);
}

// ---------------------------------------------------------------------------
// activations in 8 bits
// ---------------------------------------------------------------------------

Tensor codes_like(const Tensor& x) {
    return torch::empty(x.sizes(), x.options().dtype(torch::kFloat8_e4m3fn));
}
Tensor exponents_like(const Tensor& x) {
    return torch::empty({x.size(0), (x.size(1) + 7) / 8}, x.options().dtype(torch::kUInt8));
}
uint8_t* code_ptr(const Tensor& t) { return t.defined() ? (uint8_t*)t.data_ptr() : nullptr; }

std::tuple<Tensor, Tensor> checkpoint_encode(const Tensor& x_) {
    refuse_tangents({&x_}, "checkpoint_encode");
    const int dt = dtype_of(x_, "x");
    check_features(x_, "x");
    const c10::DeviceGuard guard(x_.device());
    const Tensor x = rows4(x_);
    const Tensor codes = codes_like(x), exps = exponents_like(x);
    check_status(batteries_checkpoint_encode(opt_ptr(x), code_ptr(codes), code_ptr(exps), x.size(0),
                                             (int)x.size(1), dt, stream_of(x)),
                 "checkpoint_encode");
    return {codes, exps};
}

void check_codes(const Tensor& codes, const Tensor& exps) {
    TORCH_CHECK(codes.is_cuda(), "codes must be a CUDA tensor");
    check_features(codes, "codes");
    TORCH_CHECK(codes.scalar_type() == torch::kFloat8_e4m3fn && codes.is_contiguous(),
                "codes must be contiguous float8_e4m3fn");
    TORCH_CHECK((reinterpret_cast<uintptr_t>(codes.data_ptr()) & 15) == 0,
                "codes must be aligned to 16 bytes");
    TORCH_CHECK(exps.device() == codes.device() && exps.scalar_type() == torch::kUInt8 &&
                    exps.is_contiguous() && exps.dim() == 2 && exps.size(0) == codes.size(0) &&
                    exps.size(1) == (codes.size(1) + 7) / 8,
                "exponents must be contiguous uint8 [N, ceil(C / 8)] on the device of codes");
}

Tensor checkpoint_decode(const Tensor& codes, const Tensor& exps, c10::ScalarType dtype) {
    check_codes(codes, exps);
    TORCH_CHECK(dtype == torch::kFloat32 || dtype == torch::kBFloat16,
                "dtype must be float32 or bfloat16");
    const c10::DeviceGuard guard(codes.device());
    const Tensor x = torch::empty(codes.sizes(), codes.options().dtype(dtype));
    check_status(batteries_checkpoint_decode(code_ptr(codes), code_ptr(exps), opt_ptr(x), x.size(0),
                                             (int)x.size(1), dtype == torch::kBFloat16, stream_of(x)),
                 "checkpoint_decode");
    return x;
}

// ---------------------------------------------------------------------------
// channel mixing
// ---------------------------------------------------------------------------

void check_mixing(const Tensor& x, const Tensor& weight, bool transposed) {
    dtype_of(x, "x");
    check_features(x, "x");
    check_f32(weight, x, "weight");
    TORCH_CHECK(weight.dim() == 3 && weight.size(0) == 4 && weight.size(transposed ? 2 : 1) == x.size(1),
                "weight must be [4, C_in, C_out]");
    TORCH_CHECK(weight.size(1) >= 1 && weight.size(1) <= 2048 && weight.size(2) >= 1 &&
                    weight.size(2) <= 2048,
                "weight must have 1 to 2048 channels on either side");
}

// transposed: of features [N, C_out, 16] to [N, C_in, 16], as the gradient goes
Tensor channel_mixing(const Tensor& x_, const Tensor& weight_, bool transposed) {
    check_mixing(x_, weight_, transposed);
    const c10::DeviceGuard guard(x_.device());
    const Tensor x = rows4(x_), weight = weight_.contiguous();
    const int dt = dtype_of(x, "x"), C = (int)weight.size(1), O = (int)weight.size(2);
    const Tensor y = torch::empty({x.size(0), transposed ? C : O, 16}, x.options());
    if (x.size(0) == 0) return y;
    const size_t wsb = batteries_channel_mixing_workspace_bytes(C, O, transposed, dt);
    const Tensor ws = bytes_on(x, wsb);
    check_status(batteries_channel_mixing(x.data_ptr(), weight.data_ptr<float>(), y.data_ptr(), x.size(0),
                                          C, O, transposed, dt, ws.data_ptr(), wsb, stream_of(x)),
                 "channel_mixing");
    return y;
}

// x: the layer's input, or none: its codes
Tensor channel_mixing_weight_grad(const OptTensor& x_, const OptTensor& codes, const OptTensor& exps,
                                  const Tensor& grad_) {
    const int dt = dtype_of(grad_, "grad");
    check_features(grad_, "grad");
    TORCH_CHECK(x_ || (codes && exps), "one of x and codes is needed");
    const c10::DeviceGuard guard(grad_.device());
    const Tensor grad = rows4(grad_);
    Tensor x;
    if (x_) {
        check_like(*x_, grad, "x");
        check_features(*x_, "x");
        x = rows4(*x_);
    } else {
        check_codes(*codes, *exps);
        TORCH_CHECK(codes->device() == grad.device(), "codes must be on ", grad.device());
    }
    const Tensor& in = x_ ? x : *codes;
    TORCH_CHECK(in.size(0) == grad.size(0), "x and grad must have the same number of rows");
    const int64_t N = grad.size(0);
    const int C = (int)in.size(1), O = (int)grad.size(1);
    const Tensor gw = torch::empty({4, C, O}, grad.options().dtype(torch::kFloat32));
    const size_t wsb = batteries_channel_mixing_weight_grad_workspace_bytes(N, C, O);
    const Tensor ws = bytes_on(grad, wsb);
    check_status(batteries_channel_mixing_weight_grad(
                     opt_ptr(x), x_ ? nullptr : code_ptr(*codes), x_ ? nullptr : code_ptr(*exps),
                     opt_ptr(grad), gw.data_ptr<float>(), N, C, O, dt, ws.data_ptr(), wsb,
                     stream_of(grad)),
                 "channel_mixing_weight_grad");
    return gw;
}

struct MixingNode : torch::autograd::Function<MixingNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, bool kept) {
        const bool need_x = x.requires_grad(), need_w = weight.requires_grad();
        Tensor codes, exps;
        if (need_w && kept) std::tie(codes, exps) = checkpoint_encode(x);
        const Tensor y = channel_mixing(x, weight, false);
        ctx->save_for_backward({need_w && !kept ? x : Tensor(), need_x ? weight : Tensor(), codes, exps});
        ctx->saved_data["needs"] = std::vector<int64_t>{need_x, need_w};
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const bool create_graph = at::GradMode::is_enabled();
        const torch::NoGradGuard no_grad;
        refuse_tangents({&grads[0]}, "the gradient of channel_mixing");
        const variable_list s = ctx->get_saved_variables();
        const std::vector<int64_t> needs = ctx->saved_data["needs"].toIntVector();
        Tensor gx, gw;
        if (needs[1])
            gw = channel_mixing_weight_grad(opt_of(s[0]), opt_of(s[2]), opt_of(s[3]), grads[0]);
        if (needs[0]) gx = channel_mixing(grads[0], s[1], true);
        variable_list g = first_order({gx, gw}, create_graph, "channel_mixing");
        g.resize(3);
        return g;
    }
};

Tensor channel_mixing_autograd(const Tensor& x, const Tensor& weight,
                               const c10::optional<std::string>& checkpoint) {
    refuse_tangents({&x, &weight}, "channel_mixing");
    const bool kept = keeps_8bit(checkpoint);
    check_mixing(x, weight, false);
    if (wants_grad({&x, &weight})) return MixingNode::apply(x, weight, kept);
    return channel_mixing(x, weight, false);
}

// ---------------------------------------------------------------------------
// gated activation
// ---------------------------------------------------------------------------

// (y, codes, exponents): the last two if kept
std::tuple<Tensor, Tensor, Tensor> gate_activation(const Tensor& x_, bool keep) {
    const int dt = dtype_of(x_, "x");
    check_features(x_, "x");
    const c10::DeviceGuard guard(x_.device());
    const Tensor x = rows4(x_), y = torch::empty_like(x);
    Tensor codes, exps;
    if (keep) codes = codes_like(x), exps = exponents_like(x);
    check_status(batteries_gate_activation(opt_ptr(x), opt_ptr(y), code_ptr(codes), code_ptr(exps),
                                           x.size(0), (int)x.size(1), dt, stream_of(x)),
                 "gate_activation");
    return {y, codes, exps};
}

Tensor gate_activation_backward(const Tensor& grad_, const OptTensor& x_, const OptTensor& codes,
                                const OptTensor& exps) {
    const int dt = dtype_of(grad_, "grad");
    check_features(grad_, "grad");
    TORCH_CHECK(x_ || (codes && exps), "one of x and codes is needed");
    const c10::DeviceGuard guard(grad_.device());
    const Tensor grad = rows4(grad_), gx = torch::empty_like(grad);
    Tensor x;
    if (x_) {
        check_same(*x_, grad, "x");
        x = rows4(*x_);
    } else {
        check_codes(*codes, *exps);
        TORCH_CHECK(codes->device() == grad.device() && codes->sizes() == grad.sizes(),
                    "codes must have the shape of grad, on ", grad.device());
    }
    check_status(batteries_gate_activation_backward(
                     opt_ptr(x), x_ ? nullptr : code_ptr(*codes), x_ ? nullptr : code_ptr(*exps),
                     opt_ptr(grad), opt_ptr(gx), grad.size(0), (int)grad.size(1), dt, stream_of(grad)),
                 "gate_activation_backward");
    return gx;
}

struct GateNode : torch::autograd::Function<GateNode> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, bool kept) {
        auto [y, codes, exps] = gate_activation(x, kept);
        ctx->save_for_backward({kept ? Tensor() : x, codes, exps});
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const bool create_graph = at::GradMode::is_enabled();
        const torch::NoGradGuard no_grad;
        refuse_tangents({&grads[0]}, "the gradient of gate_activation");
        const variable_list s = ctx->get_saved_variables();
        variable_list g = first_order(
            {gate_activation_backward(grads[0], opt_of(s[0]), opt_of(s[1]), opt_of(s[2]))},
            create_graph, "gate_activation");
        g.resize(2);
        return g;
    }
};

Tensor gate_activation_autograd(const Tensor& x, const c10::optional<std::string>& checkpoint) {
    refuse_tangents({&x}, "gate_activation");
    const bool kept = keeps_8bit(checkpoint);
    if (wants_grad({&x})) return GateNode::apply(x, kept);
    return std::get<0>(gate_activation(x, false));
}

}  // namespace

void register_layer_ops(pybind11::module_& m) {
    namespace py = pybind11;
    m.def("distance_bias", &distance_bias, py::arg("lengths"), py::arg("boundaries"), py::arg("table"),
          py::arg("cutoff") = py::none(), py::arg("keep_buckets") = false,
          "bias [E, H] of a table by buckets of length -> (bias, buckets or None)");
    m.def("distance_bias_backward", &distance_bias_backward, py::arg("lengths"), py::arg("buckets"),
          py::arg("grad"), py::arg("num_buckets"), py::arg("cutoff"), py::arg("need_table") = true,
          py::arg("need_lengths") = true, "(grad_table, grad_lengths), None where not wanted");
    m.def("distance_bias_autograd", &distance_bias_autograd, py::arg("lengths"), py::arg("boundaries"),
          py::arg("table"), py::arg("cutoff") = py::none(), "distance_bias with gradients -> bias");
    m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight"), py::arg("bias"), py::arg("eps"),
          "layer norm over the last dimension");
    m.def("layer_norm_backward", &layer_norm_backward, py::arg("grad"), py::arg("x"), py::arg("weight"),
          py::arg("need_bias"), py::arg("eps"), "(grad_x, grad_weight, grad_bias or None)");
    m.def("layer_norm_autograd", &layer_norm_autograd, py::arg("x"), py::arg("weight"), py::arg("bias"),
          py::arg("eps"), "layer_norm with gradients -> y");
    m.def("checkpoint_encode", &checkpoint_encode, py::arg("x"),
          "features in 8 bits -> (codes, exponents)");
    m.def(
        "checkpoint_decode",
        [](const Tensor& codes, const Tensor& exps, py::object dtype) {
            return checkpoint_decode(codes, exps, torch::python::detail::py_object_to_dtype(dtype));
        },
        py::arg("codes"), py::arg("exponents"), py::arg("dtype"), "the features that the codes hold");
    m.def("channel_mixing", &channel_mixing, py::arg("x"), py::arg("weight"),
          py::arg("transposed") = false, "channels mixed degree by degree (transposed: back)");
    m.def("channel_mixing_weight_grad", &channel_mixing_weight_grad, py::arg("x"), py::arg("codes"),
          py::arg("exponents"), py::arg("grad"), "gradient of the weight from x, or from its codes");
    m.def("channel_mixing_autograd", &channel_mixing_autograd, py::arg("x"), py::arg("weight"),
          py::arg("checkpoint") = py::none(), "channel_mixing with gradients -> y");
    m.def("gate_activation", &gate_activation, py::arg("x"), py::arg("keep") = false,
          "sigmoid(x[c, 0]) x[c, m] -> (y, codes or None, exponents or None)");
    m.def("gate_activation_backward", &gate_activation_backward, py::arg("grad"), py::arg("x"),
          py::arg("codes"), py::arg("exponents"), "grad_x from x, or from its codes");
    m.def("gate_activation_autograd", &gate_activation_autograd, py::arg("x"),
          py::arg("checkpoint") = py::none(), "gate_activation with gradients -> y");
}
