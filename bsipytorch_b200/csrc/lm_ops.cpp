// Host side of the operators around a language model's logits (token log probabilities, distillation) and of the 4-bit linear
// layers, as functions of the `bsi_ops` module. Checks, row plans and allocations; every kernel lives in libbsi_b200.so.
#include "lm_ops.h"

#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <vector>

#include "block.h"
#include "bsi_b200.h"

namespace py = pybind11;

namespace {

using OptTensor = c10::optional<torch::Tensor>;

void check_status(int rc, const char* what) {
    TORCH_CHECK(rc == BSI_OK, what, " failed: ", bsi_b200_status_string(rc), " (", bsi_b200_last_error(), ")");
}

bsi_stream_t current_stream() { return static_cast<bsi_stream_t>(at::cuda::getCurrentCUDAStream().stream()); }

at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, at::Device dev) {
    return at::detail::empty_cuda(sizes, type, dev, c10::nullopt);
}

int dtype_code(const at::Tensor& t, const char* what) {
    switch (t.scalar_type()) {
        case at::kFloat: return BSI_DTYPE_F32;
        case at::kHalf: return BSI_DTYPE_F16;
        case at::kBFloat16: return BSI_DTYPE_BF16;
        default: TORCH_CHECK(false, what, " must be float32, float16 or bfloat16, got ", t.scalar_type());
    }
}

// A plain tensor that wants no gradients needs no detached alias.
at::Tensor plain(const at::Tensor& t) { return t.requires_grad() ? t.detach() : t; }

void on_device(const at::Tensor& t, at::Device dev, const char* what) {
    TORCH_CHECK(t.device() == dev, what, " must live on the logits' device ", dev, ", got ", t.device());
}

std::vector<int64_t> with_last(at::IntArrayRef lead, int64_t last) {
    std::vector<int64_t> s(lead.begin(), lead.end());
    s.push_back(last);
    return s;
}

// Where the rows of t lie, taking `inner` trailing dimensions as the row (0 or 1). t is replaced by a copy where two strides do not
// describe its rows.
bsi_row_plan plan_rows(at::Tensor& t, int inner) {
    for (int attempt = 0;; ++attempt) {
        // the leading dimensions, those that lie evenly behind one another as one
        std::vector<int64_t> size, stride;
        for (int64_t d = 0; d < t.dim() - inner; ++d) {
            const int64_t n = t.size(d), s = t.stride(d);
            if (n == 1) continue;
            if (!size.empty() && stride.back() == n * s) {
                size.back() *= n;
                stride.back() = s;
            } else {
                size.push_back(n);
                stride.push_back(s);
            }
        }
        if (size.empty()) return bsi_row_plan{0, 0, 0};
        if (size.size() == 1) return bsi_row_plan{0, 0, stride[0]};
        if (size.size() == 2) return bsi_row_plan{size[1], stride[0], stride[1]};
        TORCH_INTERNAL_ASSERT(attempt == 0);
        t = t.contiguous();
    }
}

struct Logits {
    at::Tensor t;
    bsi_row_plan plan;
    int64_t rows, V;
    int code;
    std::vector<int64_t> lead;

    explicit Logits(const at::Tensor& given) : t(plain(given)) {
        TORCH_CHECK(t.is_cuda(), "logits must be a CUDA tensor: there is no CPU path");
        TORCH_CHECK(t.dim() >= 1 && t.size(-1) >= 1, "logits must be [..., vocabulary]");
        code = dtype_code(t, "logits");
        V = t.size(-1);
        if (V > 1 && t.stride(-1) != 1) t = t.contiguous();
        lead.assign(t.sizes().begin(), t.sizes().end() - 1);
        rows = 1;
        for (int64_t n : lead) rows *= n;
        plan = rows == 0 ? bsi_row_plan{0, 0, 0} : plan_rows(t, 1);
    }
};

py::tuple token_logprobs(const torch::Tensor& logits, const OptTensor& tokens, int64_t top_k) {
    const Logits z(logits);
    c10::cuda::CUDAGuard guard(z.t.device());
    TORCH_CHECK(top_k >= 0 && top_k <= 128 && top_k <= z.V, "top_k must be in [0, min(128, ", z.V, ")], got ", top_k);
    at::Tensor ids;
    bsi_row_plan ids_at{0, 0, 0};
    if (tokens.has_value()) {
        ids = plain(*tokens);
        on_device(ids, z.t.device(), "tokens");
        TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, "tokens must be int64 or int32, got ", ids.scalar_type());
        TORCH_CHECK(ids.sizes() == at::IntArrayRef(z.lead), "tokens must have the logits' leading shape ", at::IntArrayRef(z.lead), ", got ", ids.sizes());
        if (ids.scalar_type() != at::kLong) ids = ids.to(at::kLong);
        if (z.rows > 0) ids_at = plan_rows(ids, 0);
    }
    const at::Device dev = z.t.device();
    Block block(Block::room(z.rows * 4) * 2 + Block::room(z.rows * 8) + Block::room(z.rows * top_k * 4) + Block::room(z.rows * top_k * 8) + 256, dev);
    const std::vector<int64_t> with_top = with_last(z.lead, top_k);
    at::Tensor logprobs = block.take(z.lead, at::kFloat), ranks = block.take(z.lead, at::kLong), entropy = block.take(z.lead, at::kFloat);
    at::Tensor top = block.take(with_top, at::kFloat), top_ids = block.take(with_top, at::kLong);
    check_status(bsi_b200_token_logprobs(z.t.data_ptr(), z.code, z.rows, z.V, &z.plan, ids.defined() ? ids.data_ptr<int64_t>() : nullptr, &ids_at,
                                         static_cast<int>(top_k), logprobs.data_ptr<float>(), ranks.data_ptr<int64_t>(), entropy.data_ptr<float>(),
                                         top.data_ptr<float>(), top_ids.data_ptr<int64_t>(), current_stream()),
                 "bsi_b200_token_logprobs");
    return py::make_tuple(logprobs, ranks, entropy, top, top_ids);
}

// What the distillation calls share beside the logits.
struct Teacher {
    at::Tensor ids, values, weights;
    int K, code;

    Teacher(const Logits& z, const at::Tensor& given_ids, const at::Tensor& given, const OptTensor& w) {
        const at::Device dev = z.t.device();
        ids = plain(given_ids);
        values = plain(given);
        on_device(ids, dev, "ids");
        on_device(values, dev, "the teacher's values");
        TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, "ids must be int64 or int32, got ", ids.scalar_type());
        code = dtype_code(values, "the teacher's values");
        TORCH_CHECK(ids.dim() == z.t.dim() && ids.sizes() == values.sizes() && ids.sizes().slice(0, z.lead.size()) == at::IntArrayRef(z.lead),
                    "ids and the teacher's values must both be ", at::IntArrayRef(z.lead), " by entries, got ", ids.sizes(), " and ", values.sizes());
        TORCH_CHECK(ids.size(-1) >= 1 && ids.size(-1) <= 512, "1 to 512 teacher entries a row are taken, got ", ids.size(-1));
        K = static_cast<int>(ids.size(-1));
        if (ids.scalar_type() != at::kLong) ids = ids.to(at::kLong);
        if (!ids.is_contiguous()) ids = ids.contiguous();
        if (!values.is_contiguous()) values = values.contiguous();
        if (w.has_value()) {
            weights = plain(*w);
            on_device(weights, dev, "weights");
            TORCH_CHECK(weights.sizes() == at::IntArrayRef(z.lead), "weights must have the logits' leading shape ", at::IntArrayRef(z.lead), ", got ", weights.sizes());
            if (weights.scalar_type() != at::kFloat) weights = weights.to(at::kFloat);
            if (!weights.is_contiguous()) weights = weights.contiguous();
        }
    }
    const float* weight() const { return weights.defined() ? weights.data_ptr<float>() : nullptr; }
};

void check_temperature(double t) {
    TORCH_CHECK(t >= 1.0e-30 && t <= 1.0e30, "temperature must be positive (1e-30 to 1e30), got ", t);
}

// reduction: 0 none, 1 sum, 2 mean
enum { kNone = 0, kSum = 1, kMean = 2 };

struct Forward {
    at::Tensor loss, saved, sum;       // saved: what the backward pass takes; sum: of the weights, where the mean is taken
};

Forward distill_forward(const at::Tensor& logits, const at::Tensor& given_ids, const at::Tensor& values, double temperature, bool tail,
                        const OptTensor& weights, int reduction, bool save) {
    const Logits z(logits);
    check_temperature(temperature);
    c10::cuda::CUDAGuard guard(z.t.device());
    const Teacher t(z, given_ids, values, weights);
    const at::Device dev = z.t.device();
    // The loss on an allocation of its own: a caller keeps it long after what the backward pass takes.
    Forward f;
    f.loss = reduction == kNone ? fresh(z.lead, at::kFloat, dev) : fresh({}, at::kFloat, dev);
    Block block(Block::room(z.rows * 4) + Block::room(z.rows * 16) + 512, dev);
    const at::Tensor row_loss = reduction == kNone ? f.loss : block.take(z.lead, at::kFloat);
    if (save) f.saved = block.take({z.rows, 4}, at::kFloat);
    if (reduction == kMean) f.sum = block.take({}, at::kFloat);
    check_status(bsi_b200_distill_forward(z.t.data_ptr(), z.code, z.rows, z.V, &z.plan, t.ids.data_ptr<int64_t>(), t.values.data_ptr(), t.code, t.K,
                                          temperature, tail ? 1 : 0, t.weight(), reduction == kMean ? 1 : 0,
                                          row_loss.data_ptr<float>(), save ? f.saved.data_ptr<float>() : nullptr,
                                          reduction != kNone ? f.loss.data_ptr<float>() : nullptr, f.sum.defined() ? f.sum.data_ptr<float>() : nullptr,
                                          current_stream()),
                 "bsi_b200_distill_forward");
    return f;
}

at::Tensor distill_backward(const torch::Tensor& logits, const torch::Tensor& given_ids, const torch::Tensor& values, double temperature, bool tail,
                            const OptTensor& weights, const torch::Tensor& saved, const torch::Tensor& upstream, const OptTensor& sum) {
    const Logits z(logits);
    check_temperature(temperature);
    c10::cuda::CUDAGuard guard(z.t.device());
    const Teacher t(z, given_ids, values, weights);
    TORCH_CHECK(saved.is_cuda() && saved.scalar_type() == at::kFloat && saved.is_contiguous() && saved.numel() == z.rows * 4, "saved is not this forward pass's");
    TORCH_CHECK(upstream.numel() == 1 || upstream.numel() == z.rows, "one gradient, or one a row");
    on_device(upstream, z.t.device(), "the loss's gradient");
    const at::Tensor up = upstream.detach().to(at::kFloat).contiguous();
    at::Tensor grad = fresh(with_last(z.lead, z.V), z.t.scalar_type(), z.t.device());
    check_status(bsi_b200_distill_backward(z.t.data_ptr(), z.code, z.rows, z.V, &z.plan, t.ids.data_ptr<int64_t>(), t.values.data_ptr(), t.code, t.K,
                                           temperature, tail ? 1 : 0, t.weight(), saved.data_ptr<float>(),
                                           up.data_ptr<float>(), up.numel() == 1 ? 0 : 1, sum.has_value() ? sum->data_ptr<float>() : nullptr,
                                           grad.data_ptr(), z.V, current_stream()),
                 "bsi_b200_distill_backward");
    return grad;
}

// The loss as autograd has it. A node in C++: with one in Python a forward and backward pass took 88 us of host time, with this 69.
struct DistillationLoss : public torch::autograd::Function<DistillationLoss> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& values,
                              const OptTensor& weights, double temperature, bool tail, int64_t reduction) {
        const Forward f = distill_forward(logits, ids, values, temperature, tail, weights, static_cast<int>(reduction), true);
        ctx->save_for_backward({logits, ids, values, weights.has_value() ? *weights : at::Tensor(), f.saved, f.sum});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["tail"] = tail;
        return f.loss;
    }
    static torch::autograd::tensor_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::tensor_list upstream) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "distillation_loss is differentiable once: its gradient cannot be differentiated again");
        const auto kept = ctx->get_saved_variables();
        at::Tensor grad = distill_backward(kept[0], kept[1], kept[2], ctx->saved_data["temperature"].toDouble(), ctx->saved_data["tail"].toBool(),
                                           kept[3].defined() ? OptTensor(kept[3]) : OptTensor(), kept[4], upstream[0],
                                           kept[5].defined() ? OptTensor(kept[5]) : OptTensor());
        const at::Tensor none;
        return {grad, none, none, none, none, none, none};
    }
};

at::Tensor distill_loss(const torch::Tensor& logits, const torch::Tensor& ids, const torch::Tensor& values, double temperature, bool tail,
                        const OptTensor& weights, int reduction) {
    const bool grad = at::GradMode::is_enabled();
    TORCH_CHECK(!(grad && (values.requires_grad() || (weights.has_value() && weights->requires_grad()))),
                "teacher and weights must not require gradients: the loss is differentiated for the student's logits only");
    if (grad && logits.requires_grad())
        return DistillationLoss::apply(logits, ids, values, weights, temperature, tail, static_cast<int64_t>(reduction));
    return distill_forward(logits, ids, values, temperature, tail, weights, reduction, false).loss;
}

py::tuple distill_fused(const torch::Tensor& logits, const torch::Tensor& given_ids, const torch::Tensor& values, double temperature, bool tail,
                        const OptTensor& weights, int reduction) {
    const Logits z(logits);
    check_temperature(temperature);
    c10::cuda::CUDAGuard guard(z.t.device());
    const Teacher t(z, given_ids, values, weights);
    const at::Device dev = z.t.device();
    at::Tensor row_loss = fresh(z.lead, at::kFloat, dev), loss = fresh({}, at::kFloat, dev), sum = fresh({}, at::kFloat, dev);
    at::Tensor grad = fresh(with_last(z.lead, z.V), z.t.scalar_type(), dev);
    check_status(bsi_b200_distill_fused(z.t.data_ptr(), z.code, z.rows, z.V, &z.plan, t.ids.data_ptr<int64_t>(), t.values.data_ptr(), t.code, t.K,
                                        temperature, tail ? 1 : 0, t.weight(), reduction == kMean ? 1 : 0,
                                        row_loss.data_ptr<float>(), loss.data_ptr<float>(), sum.data_ptr<float>(), grad.data_ptr(), z.V,
                                        current_stream()),
                 "bsi_b200_distill_fused");
    return py::make_tuple(reduction == kNone ? row_loss : loss, grad);
}

// ---- microscaled 4-bit floating point ----------------------------------------------------------------------------------------

// The tensors of a packed matrix: codes [rows, ld] uint8, scales uint8, row_scale [rows] float32 (nvfp4) or undefined.
struct Fp4 {
    at::Tensor codes, scales, row_scale;
    int64_t rows, K;
    int format;

    const float* row() const { return row_scale.defined() ? row_scale.data_ptr<float>() : nullptr; }

    // Nothing but room.
    Fp4(int64_t r, int64_t k, int f, at::Device dev) : rows(r), K(k), format(f) {
        const int64_t ld = (K + 31) / 32 * 16, tiles = bsi_b200_fp4_scale_bytes(rows, K, format);
        Block block(Block::room(rows * ld) + Block::room(tiles) + Block::room(rows * 4) + 256, dev);
        codes = block.take({rows, ld}, at::kByte);
        scales = block.take({tiles}, at::kByte);
        if (format == BSI_FP4_NV) row_scale = block.take({rows}, at::kFloat);
    }
    // A matrix that a caller holds.
    Fp4(const at::Tensor& c, const at::Tensor& s, const OptTensor& g, int64_t k, int f) : codes(c), scales(s), rows(c.size(0)), K(k), format(f) {
        TORCH_CHECK(f == BSI_FP4_MX || f == BSI_FP4_NV, "unknown 4-bit format ", f);
        TORCH_CHECK(c.is_cuda() && c.dim() == 2 && c.scalar_type() == at::kByte && c.is_contiguous() && k >= 1 && c.size(1) == (k + 31) / 32 * 16,
                    "codes must be a contiguous uint8 CUDA tensor [rows, ", (k + 31) / 32 * 16, "]");
        TORCH_CHECK(s.device() == c.device() && s.scalar_type() == at::kByte && s.is_contiguous() && s.numel() == bsi_b200_fp4_scale_bytes(rows, k, f),
                    "scales must be ", bsi_b200_fp4_scale_bytes(rows, k, f), " bytes on the codes' device");
        TORCH_CHECK(g.has_value() == (f == BSI_FP4_NV), "nvfp4 matrices, and only they, have row scales");
        if (g.has_value()) {
            TORCH_CHECK(g->device() == c.device() && g->scalar_type() == at::kFloat && g->is_contiguous() && g->numel() == rows, "one float32 row scale per row");
            row_scale = *g;
        }
    }
};

void quantize_into(const at::Tensor& x2d, Fp4& to) {
    check_status(bsi_b200_fp4_quantize(x2d.data_ptr(), dtype_code(x2d, "x"), to.rows, to.K, to.rows > 1 ? x2d.stride(0) : to.K, to.format,
                                       to.codes.data_ptr<uint8_t>(), to.codes.size(1), to.scales.data_ptr<uint8_t>(),
                                       to.row_scale.defined() ? to.row_scale.data_ptr<float>() : nullptr, current_stream()),
                 "bsi_b200_fp4_quantize");
}

at::Tensor as_rows(const at::Tensor& given, const char* what) {
    at::Tensor t = plain(given);
    TORCH_CHECK(t.is_cuda(), what, " must be a CUDA tensor: there is no CPU path");
    TORCH_CHECK(t.dim() >= 1 && t.size(-1) >= 1, what, " must be [..., features]");
    dtype_code(t, what);
    if (t.dim() != 2) t = t.reshape({t.numel() / t.size(-1), t.size(-1)});
    // rows may lie further apart than they are long, elements not
    if ((t.size(1) > 1 && t.stride(1) != 1) || (t.size(0) > 1 && t.stride(0) < t.size(1))) t = t.contiguous();
    return t;
}

py::tuple fp4_quantize(const torch::Tensor& x, int format) {
    const at::Tensor t = as_rows(x, "x");
    TORCH_CHECK(format == BSI_FP4_MX || format == BSI_FP4_NV, "unknown 4-bit format ", format);
    c10::cuda::CUDAGuard guard(t.device());
    Fp4 q(t.size(0), t.size(1), format, t.device());
    quantize_into(t, q);
    return py::make_tuple(q.codes, q.scales, q.row_scale.defined() ? py::cast(q.row_scale) : py::none());
}

at::Tensor fp4_dequantize(const torch::Tensor& codes, const torch::Tensor& scales, const OptTensor& row_scale, int64_t K, int format, py::object dtype) {
    const Fp4 q(codes, scales, row_scale, K, format);
    c10::cuda::CUDAGuard guard(codes.device());
    at::Tensor out = fresh({q.rows, K}, torch::python::detail::py_object_to_dtype(dtype), codes.device());
    check_status(bsi_b200_fp4_dequantize(q.codes.data_ptr<uint8_t>(), q.codes.size(1), q.scales.data_ptr<uint8_t>(), q.row(), q.rows, K, format, out.data_ptr(),
                                         dtype_code(out, "dtype"), K, current_stream()),
                 "bsi_b200_fp4_dequantize");
    return out;
}

// The bias as the product reads it. A cast of its own has to stand in front of the packer, behind which the product starts early.
at::Tensor bias_of(const OptTensor& bias, const Fp4& w) {
    if (!bias.has_value()) return at::Tensor();
    TORCH_CHECK(bias->device() == w.codes.device() && bias->numel() == w.rows, "one bias per output, on the weights' device");
    at::Tensor b = plain(*bias);
    if (b.scalar_type() != at::kFloat) b = b.to(at::kFloat);
    return b.is_contiguous() ? b : b.contiguous();
}

at::Tensor product(const Fp4& x, const Fp4& w, const at::Tensor& bias, bool relu, at::ScalarType type, bool behind_packer) {
    TORCH_CHECK(x.K == w.K, "activations of ", x.K, " features, weights of ", w.K);
    TORCH_CHECK(x.format == w.format, "activations and weights are packed in different 4-bit formats");
    TORCH_CHECK(x.codes.device() == w.codes.device(), "activations and weights live on different devices");
    at::Tensor y = fresh({x.rows, w.rows}, type, w.codes.device());
    check_status(bsi_b200_fp4_linear(x.codes.data_ptr<uint8_t>(), x.codes.size(1), x.scales.data_ptr<uint8_t>(), x.row(), w.codes.data_ptr<uint8_t>(),
                                     w.codes.size(1), w.scales.data_ptr<uint8_t>(), w.row(),
                                     bias.defined() ? bias.data_ptr<float>() : nullptr, x.rows, w.rows, w.K, w.format, y.data_ptr(), w.rows,
                                     dtype_code(y, "the output"), relu ? BSI_ACT_RELU : BSI_ACT_NONE, behind_packer ? 1 : 0,
                                     current_stream()),
                 "bsi_b200_fp4_linear");
    return y;
}

at::Tensor fp4_linear(const torch::Tensor& x, const torch::Tensor& codes, const torch::Tensor& scales, const OptTensor& row_scale, int64_t K, int format,
                      const OptTensor& bias, bool relu, const c10::optional<py::object>& dtype) {
    const Fp4 w(codes, scales, row_scale, K, format);
    const at::Tensor t = as_rows(x, "x");
    TORCH_CHECK(t.size(1) == K, "activations of ", t.size(1), " features, weights of ", K);
    TORCH_CHECK(t.device() == codes.device(), "activations and weights live on different devices");
    c10::cuda::CUDAGuard guard(t.device());
    const at::Tensor b = bias_of(bias, w);
    Fp4 q(t.size(0), K, format, t.device());
    quantize_into(t, q);
    at::Tensor y = product(q, w, b, relu, dtype.has_value() ? torch::python::detail::py_object_to_dtype(*dtype) : x.scalar_type(), true);
    if (x.dim() != 2) y = y.view(with_last(x.sizes().slice(0, x.dim() - 1), w.rows));
    return y;
}

at::Tensor fp4_linear_packed(const torch::Tensor& xc, const torch::Tensor& xs, const OptTensor& xg, const torch::Tensor& codes, const torch::Tensor& scales,
                             const OptTensor& row_scale, int64_t x_K, int64_t K, int x_format, int format, const OptTensor& bias, bool relu, py::object dtype) {
    const Fp4 w(codes, scales, row_scale, K, format), q(xc, xs, xg, x_K, x_format);
    c10::cuda::CUDAGuard guard(codes.device());
    return product(q, w, bias_of(bias, w), relu, torch::python::detail::py_object_to_dtype(dtype), false);
}

}  // namespace

void register_lm_ops(py::module& m) {
    m.def("fp4_quantize", &fp4_quantize, py::arg("x"), py::arg("format"), "(codes, scales, row scales or None) of a matrix in a 4-bit format");
    m.def("fp4_dequantize", &fp4_dequantize, py::arg("codes"), py::arg("scales"), py::arg("row_scale"), py::arg("features"), py::arg("format"),
          py::arg("dtype"));
    m.def("fp4_linear", &fp4_linear, py::arg("x"), py::arg("codes"), py::arg("scales"), py::arg("row_scale"), py::arg("features"), py::arg("format"),
          py::arg("bias"), py::arg("relu"), py::arg("dtype") = py::none(), "Pack x, then the product with a packed weight");
    m.def("fp4_linear_packed", &fp4_linear_packed, py::arg("x_codes"), py::arg("x_scales"), py::arg("x_row_scale"), py::arg("codes"), py::arg("scales"),
          py::arg("row_scale"), py::arg("x_features"), py::arg("features"), py::arg("x_format"), py::arg("format"), py::arg("bias"), py::arg("relu"), py::arg("dtype"));
    m.def("token_logprobs", &token_logprobs, py::arg("logits"), py::arg("tokens") = py::none(), py::arg("top_k") = 0,
          "(logprobs, ranks, entropy, top_logprobs, top_ids) of rows of logits");
    m.def("distill_loss", &distill_loss, py::arg("logits"), py::arg("ids"), py::arg("teacher"), py::arg("temperature"), py::arg("tail"),
          py::arg("weights"), py::arg("reduction"), "The loss, differentiable for the logits");
    m.def("distill_fused", &distill_fused, py::arg("logits"), py::arg("ids"), py::arg("teacher"), py::arg("temperature"), py::arg("tail"),
          py::arg("weights"), py::arg("reduction"), "(loss, the logits' gradient) with the logits read once");
}
