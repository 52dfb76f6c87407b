// torch_train_ops.cpp -- the training-step operators (layer norm, vocabulary loss, gradient clipping) as
// torch ops of the morphottention namespace, over the C ABI of libmorpho_sm100.so.  Argument checks,
// outputs and workspaces are torch's (caching allocator, current stream, device guard), as in
// torch_ops.cpp.  An input whose rows the kernels cannot address (a last dimension that is not
// contiguous, leading dimensions without one common stride, or an unaligned base where tensor maps
// need 16 bytes) is copied first.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/library.h>

#include <optional>
#include <vector>

#include "../../include/morpho_sm100.h"

namespace {

int dtype_of(const at::Tensor& t, const char* name) {
    switch (t.scalar_type()) {
        case at::kHalf: return MORPHO_DTYPE_F16;
        case at::kBFloat16: return MORPHO_DTYPE_BF16;
        case at::kFloat: return MORPHO_DTYPE_F32;
        default: TORCH_CHECK(false, name, " must be float16, bfloat16 or float32");
    }
}

void on_cuda(const at::Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
}

void same_device(const at::Tensor& t, const at::Tensor& x, const char* name) {
    on_cuda(t, name);
    TORCH_CHECK(t.device() == x.device(), name, " must be on the same device as the other tensors");
}

// [.., dim] as rows of `dim` contiguous elements with one stride: the tensor itself where its leading
// dimensions collapse, else a contiguous copy.
struct Rows {
    at::Tensor t;
    int64_t stride;
};

Rows as_rows(const at::Tensor& t, int64_t align_bytes) {
    const int64_t d = t.dim();
    const bool unit = t.size(d - 1) <= 1 || t.stride(d - 1) == 1;
    int64_t stride = t.size(d - 1), expected = -1;
    bool ok = unit;
    for (int64_t i = d - 2; i >= 0 && ok; --i) {
        if (t.size(i) == 1) continue;
        if (expected < 0) {
            stride = t.stride(i);
            ok = stride >= t.size(d - 1);
        } else {
            ok = t.stride(i) == expected;
        }
        expected = t.stride(i) * t.size(i);
    }
    if (ok && align_bytes > 1)
        ok = reinterpret_cast<uintptr_t>(t.data_ptr()) % align_bytes == 0 && stride * t.element_size() % align_bytes == 0;
    if (ok || t.numel() == 0) return {t, ok ? stride : t.size(d - 1)};
    return {t.clone(at::MemoryFormat::Contiguous), t.size(d - 1)};
}

void* stream_of(const at::Tensor& t) {
    return static_cast<void*>(at::cuda::getCurrentCUDAStream(t.device().index()).stream());
}

void check_rc(int rc, const char* what) {
    TORCH_CHECK(rc == MORPHO_OK, "morphottention ", what, " failed (", rc, "): ", morpho_sm100_last_error());
}

at::Tensor workspace(size_t bytes, const at::Tensor& like) {
    return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

// ---- layer norm --------------------------------------------------------------------------------

morpho_layer_norm_t norm_problem(const at::Tensor& x, const std::optional<at::Tensor>& weight, const char* name) {
    on_cuda(x, name);
    TORCH_CHECK(x.dim() >= 1, name, " must have at least one dimension");
    const int64_t dim = x.size(x.dim() - 1);
    TORCH_CHECK(dim > 0, name, " must not have an empty last dimension");
    TORCH_CHECK(dim <= INT32_MAX, name, " has too long a last dimension (", dim, ")");  // the problem holds 32 bits
    morpho_layer_norm_t p{};
    p.rows = x.numel() / dim;
    p.dim = static_cast<int32_t>(dim);
    p.type = dtype_of(x, name);
    p.weight_type = weight.has_value() ? dtype_of(*weight, "weight") : p.type;
    return p;
}

void check_param(const std::optional<at::Tensor>& w, const at::Tensor& x, const morpho_layer_norm_t& p, const char* name) {
    if (!w.has_value()) return;
    same_device(*w, x, name);
    TORCH_CHECK(w->dim() == 1 && w->size(0) == p.dim, name, " must be [", p.dim, "]");
    TORCH_CHECK(dtype_of(*w, name) == p.weight_type, "weight and bias must have the same type");
    TORCH_CHECK(w->is_contiguous(), name, " must be contiguous");
    TORCH_CHECK(p.weight_type == p.type || p.weight_type == MORPHO_DTYPE_F32, name, " must have x's type or be float32");
}

void* ptr_or_null(const std::optional<at::Tensor>& t) { return t.has_value() ? t->data_ptr() : nullptr; }

std::vector<at::Tensor> layer_norm_forward(const at::Tensor& x, const std::optional<at::Tensor>& weight,
                                           const std::optional<at::Tensor>& bias, double eps,
                                           const std::optional<at::Tensor>& residual) {
    morpho_layer_norm_t p = norm_problem(x, weight, "x");
    TORCH_CHECK(weight.has_value() || !bias.has_value(), "bias needs a weight");
    check_param(weight, x, p, "weight");
    check_param(bias, x, p, "bias");
    p.eps = static_cast<float>(eps);
    const c10::cuda::CUDAGuard guard(x.device());
    const Rows xr = as_rows(x, 1);
    p.stride_x = xr.stride;
    Rows rr{x, 0};
    if (residual.has_value()) {
        same_device(*residual, x, "residual");
        TORCH_CHECK(residual->sizes() == x.sizes(), "residual must have x's shape");
        TORCH_CHECK(residual->scalar_type() == x.scalar_type(), "residual must have x's type");
        rr = as_rows(*residual, 1);
        p.stride_residual = rr.stride;
    }
    auto y = at::empty(x.sizes(), x.options());
    const auto lead = x.sizes().slice(0, x.dim() - 1);
    const auto f32 = x.options().dtype(at::kFloat);
    auto mean = at::empty(lead, f32), rstd = at::empty(lead, f32);
    at::Tensor h;
    if (residual.has_value()) h = at::empty(x.sizes(), x.options());
    check_rc(morpho_sm100_layer_norm_forward(&p, xr.t.data_ptr(), residual.has_value() ? rr.t.data_ptr() : nullptr,
                                             ptr_or_null(weight), ptr_or_null(bias), y.data_ptr(),
                                             residual.has_value() ? h.data_ptr() : nullptr, mean.data_ptr<float>(),
                                             rstd.data_ptr<float>(), stream_of(x)),
             "layer_norm_forward");
    if (residual.has_value()) return {y, mean, rstd, h};
    return {y, mean, rstd};
}

std::vector<at::Tensor> layer_norm_backward(const at::Tensor& grad_y, const at::Tensor& h,
                                            const std::optional<at::Tensor>& weight, const at::Tensor& mean,
                                            const at::Tensor& rstd, const std::optional<at::Tensor>& grad_h) {
    morpho_layer_norm_t p = norm_problem(h, weight, "h");
    check_param(weight, h, p, "weight");
    for (const auto& [t, name] : {std::pair<const at::Tensor*, const char*>{&mean, "mean"}, {&rstd, "rstd"}}) {
        same_device(*t, h, name);
        TORCH_CHECK(t->scalar_type() == at::kFloat && t->is_contiguous() && t->numel() == p.rows, name,
                    " must be the contiguous float32 tensor of the forward");
    }
    same_device(grad_y, h, "grad_y");
    TORCH_CHECK(grad_y.sizes() == h.sizes() && grad_y.scalar_type() == h.scalar_type(), "grad_y must match h's shape and type");
    const c10::cuda::CUDAGuard guard(h.device());
    const Rows hr = as_rows(h, 1), gr = as_rows(grad_y, 1);
    p.stride_x = hr.stride;
    p.stride_grad_y = gr.stride;
    Rows sr{h, 0};
    if (grad_h.has_value()) {
        same_device(*grad_h, h, "grad_h");
        TORCH_CHECK(grad_h->sizes() == h.sizes() && grad_h->scalar_type() == h.scalar_type(), "grad_h must match h's shape and type");
        sr = as_rows(*grad_h, 1);
        p.stride_grad_h = sr.stride;
    }
    auto dx = at::empty(h.sizes(), h.options());
    auto wopt = weight.has_value() ? weight->options() : h.options();
    auto dw = at::empty({p.dim}, wopt), db = at::empty({p.dim}, wopt);
    const size_t bytes = morpho_sm100_layer_norm_backward_workspace_size(&p);
    TORCH_CHECK(bytes > 0, "morphottention layer_norm_backward: unsupported problem: ", morpho_sm100_last_error());
    auto ws = workspace(bytes, h);
    check_rc(morpho_sm100_layer_norm_backward(&p, gr.t.data_ptr(), grad_h.has_value() ? sr.t.data_ptr() : nullptr,
                                              hr.t.data_ptr(), ptr_or_null(weight), mean.data_ptr<float>(),
                                              rstd.data_ptr<float>(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(),
                                              ws.data_ptr(), bytes, stream_of(h)),
             "layer_norm_backward");
    return {dx, dw, db};
}

// ---- vocabulary loss -----------------------------------------------------------------------------

morpho_vocab_loss_t loss_problem(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& target,
                                 int64_t ignore_index, int64_t reduction) {
    on_cuda(hidden, "hidden");
    TORCH_CHECK(hidden.scalar_type() == at::kHalf || hidden.scalar_type() == at::kBFloat16,
                "hidden must be float16 or bfloat16");
    TORCH_CHECK(hidden.dim() >= 1, "hidden must have at least one dimension");
    same_device(weight, hidden, "weight");
    same_device(target, hidden, "target");
    const int64_t D = hidden.size(hidden.dim() - 1);
    TORCH_CHECK(D > 0 && D % 8 == 0, "the last dimension of hidden must be a positive multiple of 8");
    TORCH_CHECK(weight.dim() == 2 && weight.size(1) == D && weight.size(0) > 0, "weight must be [vocab, ", D, "]");
    TORCH_CHECK(weight.size(0) <= (1 << 30) && D <= 16384, "weight is too large: at most 2^30 rows, dim at most 16384");
    TORCH_CHECK(weight.scalar_type() == hidden.scalar_type(), "weight must have hidden's type");
    TORCH_CHECK(target.scalar_type() == at::kLong, "target must be int64");
    TORCH_CHECK(target.sizes() == hidden.sizes().slice(0, hidden.dim() - 1), "target must have hidden's leading shape");
    TORCH_CHECK(reduction >= MORPHO_REDUCTION_NONE && reduction <= MORPHO_REDUCTION_SUM,
                "reduction must be 0 (none), 1 (mean) or 2 (sum)");
    morpho_vocab_loss_t p{};
    p.tokens = target.numel();
    p.vocab = static_cast<int32_t>(weight.size(0));
    p.dim = static_cast<int32_t>(D);
    p.type = dtype_of(hidden, "hidden");
    p.reduction = static_cast<int32_t>(reduction);
    p.ignore_index = ignore_index;
    return p;
}

std::vector<at::Tensor> linear_cross_entropy_forward(const at::Tensor& hidden, const at::Tensor& weight,
                                                     const at::Tensor& target, int64_t ignore_index,
                                                     int64_t reduction) {
    morpho_vocab_loss_t p = loss_problem(hidden, weight, target, ignore_index, reduction);
    const c10::cuda::CUDAGuard guard(hidden.device());
    const Rows hr = as_rows(hidden, 16), wr = as_rows(weight, 16);
    p.stride_hidden = hr.stride;
    p.stride_weight = wr.stride;
    const at::Tensor t = target.contiguous();
    auto f32 = hidden.options().dtype(at::kFloat);
    auto lse = at::empty(target.sizes(), f32);
    auto loss = reduction == MORPHO_REDUCTION_NONE ? at::empty(target.sizes(), f32) : at::empty({}, f32);
    const size_t bytes = morpho_sm100_linear_cross_entropy_forward_workspace_size(&p);
    TORCH_CHECK(bytes > 0, "morphottention linear_cross_entropy_forward: unsupported problem: ", morpho_sm100_last_error());
    auto ws = workspace(bytes, hidden);
    if (p.tokens == 0 && reduction == MORPHO_REDUCTION_NONE) return {loss, lse};
    check_rc(morpho_sm100_linear_cross_entropy_forward(&p, hr.t.data_ptr(), wr.t.data_ptr(), t.data_ptr<int64_t>(),
                                                       loss.data_ptr<float>(), lse.data_ptr<float>(), ws.data_ptr(),
                                                       bytes, stream_of(hidden)),
             "linear_cross_entropy_forward");
    return {loss, lse};
}

std::vector<at::Tensor> linear_cross_entropy_backward(const at::Tensor& grad_loss, const at::Tensor& hidden,
                                                      const at::Tensor& weight, const at::Tensor& target,
                                                      const at::Tensor& lse, int64_t ignore_index, int64_t reduction) {
    morpho_vocab_loss_t p = loss_problem(hidden, weight, target, ignore_index, reduction);
    same_device(grad_loss, hidden, "grad_loss");
    same_device(lse, hidden, "lse");
    TORCH_CHECK(grad_loss.scalar_type() == at::kFloat, "grad_loss must be float32");
    TORCH_CHECK(lse.scalar_type() == at::kFloat && lse.is_contiguous() && lse.numel() == p.tokens,
                "lse must be the contiguous float32 tensor of the forward");
    if (reduction == MORPHO_REDUCTION_NONE) {
        TORCH_CHECK(grad_loss.sizes() == target.sizes(), "grad_loss must have target's shape");
    } else {
        TORCH_CHECK(grad_loss.numel() == 1, "grad_loss must have one element");
    }
    const c10::cuda::CUDAGuard guard(hidden.device());
    const Rows hr = as_rows(hidden, 16), wr = as_rows(weight, 16);
    p.stride_hidden = hr.stride;
    p.stride_weight = wr.stride;
    const at::Tensor t = target.contiguous(), g = grad_loss.contiguous();
    auto dh = at::empty(hidden.sizes(), hidden.options()), dw = at::empty(weight.sizes(), weight.options());
    const size_t bytes = morpho_sm100_linear_cross_entropy_backward_workspace_size(&p);
    TORCH_CHECK(bytes > 0, "morphottention linear_cross_entropy_backward: unsupported problem: ", morpho_sm100_last_error());
    auto ws = workspace(bytes, hidden);
    check_rc(morpho_sm100_linear_cross_entropy_backward(&p, g.data_ptr<float>(), hr.t.data_ptr(), wr.t.data_ptr(),
                                                        t.data_ptr<int64_t>(), lse.data_ptr<float>(), dh.data_ptr(),
                                                        dw.data_ptr(), ws.data_ptr(), bytes, stream_of(hidden)),
             "linear_cross_entropy_backward");
    return {dh, dw};
}

// ---- clipping ------------------------------------------------------------------------------------

at::Tensor clip_grad_norm(at::TensorList grads, at::TensorList out, double max_norm, double loss_scale) {
    TORCH_CHECK(!grads.empty(), "grads must not be empty");
    TORCH_CHECK(grads.size() == out.size(), "out must have as many tensors as grads");
    std::vector<morpho_tensor_pair_t> pairs(grads.size());
    for (size_t i = 0; i < grads.size(); ++i) {
        const at::Tensor &g = grads[i], &o = out[i];
        same_device(g, grads[0], "every gradient");
        same_device(o, grads[0], "every output");
        TORCH_CHECK(g.sizes() == o.sizes(), "out[", i, "] must have the shape of grads[", i, "]");
        // any order of the dimensions will do, as long as both sides have it and leave no gaps
        TORCH_CHECK(g.is_non_overlapping_and_dense() && o.is_non_overlapping_and_dense() &&
                        (g.strides() == o.strides() || (g.is_contiguous() && o.is_contiguous())),
                    "grads[", i, "] and out[", i, "] must be dense and have the same strides");
        pairs[i].in = g.data_ptr();
        pairs[i].out = o.data_ptr();
        pairs[i].count = g.numel();
        pairs[i].in_type = dtype_of(g, "every gradient");
        pairs[i].out_type = dtype_of(o, "every output");
    }
    const c10::cuda::CUDAGuard guard(grads[0].device());
    auto norm = at::empty({}, grads[0].options().dtype(at::kFloat).layout(at::kStrided));
    const int64_t n = static_cast<int64_t>(pairs.size());
    const size_t bytes = morpho_sm100_clip_grad_norm_workspace_size(n);
    auto ws = workspace(bytes, grads[0]);
    check_rc(morpho_sm100_clip_grad_norm(pairs.data(), n, static_cast<float>(max_norm), static_cast<float>(loss_scale),
                                         norm.data_ptr<float>(), ws.data_ptr(), bytes, stream_of(grads[0])),
             "clip_grad_norm");
    // written through raw pointers: a graph that has saved one of them must notice
    for (const at::Tensor& o : out)
        if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
    return norm;
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(morphottention, m) {
    m.def("layer_norm_forward(Tensor x, Tensor? weight, Tensor? bias, float eps, Tensor? residual=None) -> Tensor[]");
    m.def(
        "layer_norm_backward(Tensor grad_y, Tensor h, Tensor? weight, Tensor mean, Tensor rstd, "
        "Tensor? grad_h=None) -> Tensor[]");
    m.def(
        "linear_cross_entropy_forward(Tensor hidden, Tensor weight, Tensor target, int ignore_index=-100, "
        "int reduction=1) -> Tensor[]");
    m.def(
        "linear_cross_entropy_backward(Tensor grad_loss, Tensor hidden, Tensor weight, Tensor target, Tensor lse, "
        "int ignore_index=-100, int reduction=1) -> Tensor[]");
    m.def("clip_grad_norm(Tensor[] grads, Tensor(a!)[] out, float max_norm, float loss_scale=1.0) -> Tensor");
}

TORCH_LIBRARY_IMPL(morphottention, CUDA, m) {
    m.impl("layer_norm_forward", &layer_norm_forward);
    m.impl("layer_norm_backward", &layer_norm_backward);
    m.impl("linear_cross_entropy_forward", &linear_cross_entropy_forward);
    m.impl("linear_cross_entropy_backward", &linear_cross_entropy_backward);
    m.impl("clip_grad_norm", &clip_grad_norm);
}
