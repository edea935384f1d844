// Host side of the operators around a language model's logits (token log probabilities, distillation), as functions
// of the `bsi_ops` module. Checks, row plans and allocations; every kernel lives in libbsi_b200.so.
#include "lm_ops.h"

#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <vector>

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

    explicit Logits(const at::Tensor& given) : t(given.detach()) {
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
        ids = tokens->detach();
        on_device(ids, z.t.device(), "tokens");
        TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, "tokens must be int64 or int32, got ", ids.scalar_type());
        TORCH_CHECK(ids.sizes() == at::IntArrayRef(z.lead), "tokens must have the logits' leading shape ", at::IntArrayRef(z.lead), ", got ", ids.sizes());
        if (ids.scalar_type() != at::kLong) ids = ids.to(at::kLong);
        if (z.rows > 0) ids_at = plan_rows(ids, 0);
    }
    const at::Device dev = z.t.device();
    at::Tensor logprobs = fresh(z.lead, at::kFloat, dev), ranks = fresh(z.lead, at::kLong, dev), entropy = fresh(z.lead, at::kFloat, dev);
    at::Tensor top = fresh(with_last(z.lead, top_k), at::kFloat, dev), top_ids = fresh(with_last(z.lead, top_k), at::kLong, dev);
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
        ids = given_ids.detach();
        values = given.detach();
        on_device(ids, dev, "ids");
        on_device(values, dev, "the teacher's values");
        TORCH_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, "ids must be int64 or int32, got ", ids.scalar_type());
        code = dtype_code(values, "the teacher's values");
        TORCH_CHECK(ids.dim() == z.t.dim() && ids.sizes() == values.sizes() && ids.sizes().slice(0, z.lead.size()) == at::IntArrayRef(z.lead),
                    "ids and the teacher's values must both be ", at::IntArrayRef(z.lead), " by entries, got ", ids.sizes(), " and ", values.sizes());
        TORCH_CHECK(ids.size(-1) >= 1 && ids.size(-1) <= 512, "1 to 512 teacher entries a row are taken, got ", ids.size(-1));
        K = static_cast<int>(ids.size(-1));
        ids = ids.to(at::kLong).contiguous();
        values = values.contiguous();
        if (w.has_value()) {
            weights = w->detach();
            on_device(weights, dev, "weights");
            TORCH_CHECK(weights.sizes() == at::IntArrayRef(z.lead), "weights must have the logits' leading shape ", at::IntArrayRef(z.lead), ", got ", weights.sizes());
            weights = weights.to(at::kFloat).contiguous();
        }
    }
    const float* weight() const { return weights.defined() ? weights.data_ptr<float>() : nullptr; }
};

void check_temperature(double t) {
    TORCH_CHECK(static_cast<float>(t) > 0.0f && static_cast<float>(t) <= 3.0e38f, "temperature must be positive and finite, got ", t);
}

// reduction: 0 none, 1 sum, 2 mean
enum { kNone = 0, kSum = 1, kMean = 2 };

py::tuple distill_forward(const torch::Tensor& logits, const torch::Tensor& given_ids, const torch::Tensor& values, double temperature, bool tail,
                          const OptTensor& weights, int reduction, bool save) {
    const Logits z(logits);
    check_temperature(temperature);
    c10::cuda::CUDAGuard guard(z.t.device());
    const Teacher t(z, given_ids, values, weights);
    const at::Device dev = z.t.device();
    at::Tensor row_loss = fresh(z.lead, at::kFloat, dev), saved, loss, sum;
    if (save) saved = fresh({z.rows, 4}, at::kFloat, dev);
    if (reduction != kNone) loss = fresh({}, at::kFloat, dev);
    if (reduction == kMean) sum = fresh({}, at::kFloat, dev);
    check_status(bsi_b200_distill_forward(z.t.data_ptr(), z.code, z.rows, z.V, &z.plan, t.ids.data_ptr<int64_t>(), t.values.data_ptr(), t.code, t.K,
                                          static_cast<float>(temperature), tail ? 1 : 0, t.weight(), reduction == kMean ? 1 : 0,
                                          row_loss.data_ptr<float>(), save ? saved.data_ptr<float>() : nullptr,
                                          loss.defined() ? loss.data_ptr<float>() : nullptr, sum.defined() ? sum.data_ptr<float>() : nullptr,
                                          current_stream()),
                 "bsi_b200_distill_forward");
    return py::make_tuple(reduction == kNone ? row_loss : loss, saved.defined() ? py::cast(saved) : py::none(),
                          sum.defined() ? py::cast(sum) : py::none());
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
                                           static_cast<float>(temperature), tail ? 1 : 0, t.weight(), saved.data_ptr<float>(),
                                           up.data_ptr<float>(), up.numel() == 1 ? 0 : 1, sum.has_value() ? sum->data_ptr<float>() : nullptr,
                                           grad.data_ptr(), z.V, current_stream()),
                 "bsi_b200_distill_backward");
    return grad;
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
                                        static_cast<float>(temperature), tail ? 1 : 0, t.weight(), reduction == kMean ? 1 : 0,
                                        row_loss.data_ptr<float>(), loss.data_ptr<float>(), sum.data_ptr<float>(), grad.data_ptr(), z.V,
                                        current_stream()),
                 "bsi_b200_distill_fused");
    return py::make_tuple(reduction == kNone ? row_loss : loss, grad);
}

bool distill_fused_fits(const torch::Tensor& logits, bool tail) {
    return bsi_b200_distill_fused_fits(dtype_code(logits, "logits"), logits.size(-1), tail ? 1 : 0) == 1;
}

}  // namespace

void register_lm_ops(py::module& m) {
    m.def("token_logprobs", &token_logprobs, py::arg("logits"), py::arg("tokens") = py::none(), py::arg("top_k") = 0,
          "(logprobs, ranks, entropy, top_logprobs, top_ids) of rows of logits");
    m.def("distill_forward", &distill_forward, py::arg("logits"), py::arg("ids"), py::arg("teacher"), py::arg("temperature"), py::arg("tail"),
          py::arg("weights"), py::arg("reduction"), py::arg("save"), "(loss, what the backward pass takes or None, the weights' sum or None)");
    m.def("distill_backward", &distill_backward, py::arg("logits"), py::arg("ids"), py::arg("teacher"), py::arg("temperature"), py::arg("tail"),
          py::arg("weights"), py::arg("saved"), py::arg("upstream"), py::arg("weight_sum"), "The logits' gradient");
    m.def("distill_fused", &distill_fused, py::arg("logits"), py::arg("ids"), py::arg("teacher"), py::arg("temperature"), py::arg("tail"),
          py::arg("weights"), py::arg("reduction"), "(loss, the logits' gradient) with the logits read once");
    m.def("distill_fused_fits", &distill_fused_fits, py::arg("logits"), py::arg("tail"));
}
