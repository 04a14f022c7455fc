// gk_torch.cpp - the training-step operators as PyTorch operators.
//
// Argument checks, allocation, autograd and the calls of the C ABI
// (include/gk.h), on the tensors' device and its current stream. A training
// step calls these many times with small batches, where a Python autograd
// function costs several times the kernels; here a forward and backward pass
// through `linear` takes the host about half the time.
//
// Every tensor argument is marked as used on the stream (record_stream), so
// memory that was allocated on another stream is not reused under a launch.
// What a forward pass saved is used on the same stream by its backward pass.
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/library.h>

#include <tuple>

#include "../../include/gk.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr int64_t kMost = (1ll << 31) - 1;
constexpr int64_t kMostColumns = 1ll << 30;
constexpr int64_t kMostValues = 1ll << 40;

int type_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return GK_FP32;
        case at::kBFloat16: return GK_BF16;
        case at::kHalf: return GK_FP16;
        default: return -1;
    }
}

// Messages are put together as strings, not by streams: a stream formats a
// number with the locale's facets, which failed where another copy of the C++
// runtime had been loaded first.
void ran(const char* name, int status) {
    TORCH_CHECK_VALUE(status != -22, std::string(name) + ": invalid argument");
    TORCH_CHECK(status == 0, std::string(name) + " failed with CUDA error " + std::to_string(status));
}

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }
void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* data(const OptTensor& t) { return has(t) ? t->data_ptr() : nullptr; }

void used(const Tensor& t, const c10::cuda::CUDAStream& stream) {
    if (t.defined()) t.record_stream(stream.unwrap());
}
void used(const OptTensor& t, const c10::cuda::CUDAStream& stream) {
    if (has(t)) used(*t, stream);
}

// The kernels read memory: a lazily negated view (the imaginary part of a
// conjugate) is negated first.
Tensor plain(const Tensor& t) { return t.is_neg() ? t.resolve_neg() : t; }
Tensor dense(const Tensor& t) { return plain(t).contiguous(); }
// [rows, cols] with contiguous rows: a view where the layout allows, else a copy.
Tensor rows_of(const Tensor& given, int64_t cols) {
    const Tensor t = plain(given);
    if (t.dim() != 2) return t.contiguous().view({-1, cols});
    return (t.stride(1) == 1 || cols == 1) && t.stride(0) >= 0 ? t : t.contiguous();
}
// Elements between rows; the row length where there is but one row.
int64_t row_stride(const Tensor& t, int64_t cols) { return t.size(0) == 1 ? cols : t.stride(0); }

Tensor bytes_on(int64_t size, const Tensor& like) {
    return at::empty({size}, like.options().dtype(at::kByte).requires_grad(false));
}

// Gradients under create_graph: usable, but asking for their own gradient raises.
variable_list once(variable_list grads, const char* name) {
    if (!at::GradMode::is_enabled()) return grads;
    for (auto& g : grads) {
        if (!g.defined()) continue;
        Tensor fake = g.detach();
        fake.requires_grad_(true);
        g = (*std::make_shared<torch::autograd::DelayedError>(
            std::string("trying to differentiate twice: ") + name + " is differentiable once", 1))({fake})[0];
    }
    return grads;
}

// There are no forward-mode derivatives. An output without a tangent would stand for a derivative of zero.
bool tangent(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }
bool tangent(const OptTensor& t) { return t.has_value() && tangent(*t); }
template <typename... T>
void no_tangent(const char* name, const T&... inputs) {
    TORCH_CHECK_NOT_IMPLEMENTED(!(tangent(inputs) || ...), std::string(name) + " has no forward-mode derivative");
}

// ------------------------------------------------------------------ pack

// Codes, then scales, of [rows, cols] with rows `stride` elements apart. Rows that lie over one another (an
// expanded or unfolded tensor) are copied apart first, which gk_pack asks for.
std::tuple<Tensor, Tensor> pack_rows(const Tensor& given, int64_t rows, int64_t cols, int64_t given_stride) {
    const bool apart = rows <= 1 || given_stride >= cols;
    const Tensor x = apart ? given : given.contiguous();
    const int64_t stride = apart ? given_stride : cols;
    const int64_t scales = rows * ((cols + 31) / 32);
    Tensor buffer = bytes_on(rows * cols + scales, x);
    Tensor codes = buffer.narrow(0, 0, rows * cols), factor = buffer.narrow(0, rows * cols, scales);
    if (rows > 0 && cols > 0) {
        const c10::cuda::CUDAGuard guard(x.device());
        const auto stream = c10::cuda::getCurrentCUDAStream();
        used(x, stream);
        ran("gk_pack", gk_pack(x.data_ptr(), stride, type_of(x.scalar_type()), rows, cols,
                               static_cast<uint8_t*>(codes.data_ptr()), static_cast<uint8_t*>(factor.data_ptr()),
                               stream.stream()));
    }
    return {codes, factor};
}

std::tuple<Tensor, Tensor> pack(const Tensor& x) {
    TORCH_CHECK_VALUE(x.is_cuda() && type_of(x.scalar_type()) >= 0,
                      "pack_activation packs CUDA tensors of float32, bfloat16 or float16");
    const at::NoGradGuard no_grad;
    const Tensor flat = dense(x);
    return pack_rows(flat, 1, flat.numel(), flat.numel());
}

Tensor unpack(const Tensor& codes, const Tensor& scales, at::IntArrayRef shape, at::ScalarType dtype) {
    const at::NoGradGuard no_grad;
    int64_t count = 1;
    for (const int64_t size : shape) {
        TORCH_CHECK_VALUE(size >= 0 && (size == 0 || count <= kMostValues / size),
                          "a packed activation has up to 2**40 values");
        count *= size;
    }
    TORCH_CHECK_VALUE(type_of(dtype) >= 0, "unpack gives float32, bfloat16 or float16");
    TORCH_CHECK_VALUE(codes.is_cuda() && scales.device() == codes.device() && codes.scalar_type() == at::kByte &&
                          scales.scalar_type() == at::kByte && codes.is_contiguous() && scales.is_contiguous() &&
                          codes.numel() == count && scales.numel() == (count + 31) / 32,
                      "a packed activation holds a contiguous CUDA uint8 code for each of its shape's values, and a "
                      "scale for every 32 of them");
    Tensor out = at::empty(shape, codes.options().dtype(dtype));
    if (out.numel() > 0) {
        const c10::cuda::CUDAGuard guard(out.device());
        const auto stream = c10::cuda::getCurrentCUDAStream();
        used(codes, stream);
        used(scales, stream);
        ran("gk_unpack", gk_unpack(static_cast<const uint8_t*>(codes.data_ptr()),
                                   static_cast<const uint8_t*>(scales.data_ptr()), 1, out.numel(), out.data_ptr(),
                                   out.numel(), type_of(dtype), stream.stream()));
    }
    return out;
}

// ---------------------------------------------------------------- linear

// y and, if asked for, what the derivative takes: the sum before the activation, or tanh in fp32.
std::tuple<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& w, const OptTensor& bias,
                                          const OptTensor& residual, int64_t activation, bool keep_sum,
                                          const Tensor& status) {
    const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
    const auto options = x.options().requires_grad(false);
    Tensor y = at::empty({m, n}, options), pre;
    // Its rows start on 16 bytes whatever n is: it is written and read in whole vectors.
    if (keep_sum)
        pre = at::empty({m, (n + 7) / 8 * 8}, activation == GK_ACT_TANH ? options.dtype(at::kFloat) : options)
                  .narrow(1, 0, n);
    if (m == 0) return {y, pre};
    gk_linear_t p{};
    p.x = x.data_ptr(), p.w = w.data_ptr(), p.bias = data(bias), p.residual = data(residual);
    p.y = y.data_ptr(), p.pre = data(pre);
    p.m = m, p.n = n, p.k = k;
    p.x_stride = row_stride(x, k), p.w_stride = row_stride(w, k);
    p.residual_stride = has(residual) ? row_stride(*residual, n) : 0;
    p.pre_stride = pre.defined() ? pre.stride(0) : 0;
    p.dtype = type_of(x.scalar_type());
    p.activation = (int)activation;
    const c10::cuda::CUDAGuard guard(x.device());
    const auto stream = c10::cuda::getCurrentCUDAStream();
    Tensor workspace;
    const size_t size = gk_linear_workspace_bytes(&p);
    if (size > 0) workspace = bytes_on((int64_t)size, x);
    used(x, stream);
    used(w, stream);
    used(bias, stream);
    used(residual, stream);
    ran("gk_linear_forward", gk_linear_forward(&p, data(workspace), static_cast<uint32_t*>(status.data_ptr()),
                                               stream.stream()));
    return {y, pre};
}

struct Linear : torch::autograd::Function<Linear> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias,
                          const OptTensor& residual, int64_t activation, bool packed, const Tensor& status) {
        auto [y, pre] = linear_forward(x, w, bias, residual, activation,
                                       activation == GK_ACT_GELU || activation == GK_ACT_SILU ||
                                           (activation == GK_ACT_TANH && x.scalar_type() != at::kFloat),
                                       status);
        const int64_t m = x.size(0), k = x.size(1);
        const bool need_x = x.requires_grad(), need_w = w.requires_grad();
        Tensor codes, scales;
        if (need_w && packed) std::tie(codes, scales) = pack_rows(x, m, k, row_stride(x, k));
        ctx->save_for_backward({need_w && !packed ? x : Tensor(), need_x ? w : Tensor(),
                                activation == GK_ACT_NONE ? Tensor() : (pre.defined() ? pre : y), codes, scales});
        ctx->saved_data["status"] = status;  // no saved input: check_linear may clear it before the backward pass
        ctx->saved_data["sizes"] = std::vector<int64_t>{m, w.size(0), k, activation, need_x, need_w,
                                                        has(bias) && bias->requires_grad(),
                                                        has(residual) && residual->requires_grad()};
        return y;
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list saved = ctx->get_saved_variables();
        const auto s = ctx->saved_data["sizes"].toIntVector();
        const int64_t m = s[0], n = s[1], k = s[2], activation = s[3];
        Tensor dx, dw, db, dr;
        {
            const at::NoGradGuard no_grad;
            const Tensor dy = rows_of(grads[0], n);
            const auto options = dy.options();
            if (s[4]) dx = at::empty({m, k}, options);
            if (s[5]) dw = m == 0 ? at::zeros({n, k}, options) : at::empty({n, k}, options);
            if (s[6]) db = m == 0 ? at::zeros({n}, options) : at::empty({n}, options);
            if (s[7]) dr = activation == GK_ACT_NONE ? dy : at::empty({m, n}, options);
            if (m > 0 && (s[4] || s[5] || s[6] || (s[7] && activation != GK_ACT_NONE))) {
                gk_linear_grad_t p{};
                p.dy = dy.data_ptr(), p.kept = data(saved[2]), p.x = data(saved[0]);
                p.x_codes = static_cast<const uint8_t*>(data(saved[3]));
                p.x_scales = static_cast<const uint8_t*>(data(saved[4]));
                p.w = data(saved[1]);
                p.dx = data(dx), p.dw = data(dw), p.db = data(db);
                p.dz = activation == GK_ACT_NONE ? nullptr : data(dr);
                p.m = m, p.n = n, p.k = k;
                p.dy_stride = row_stride(dy, n);
                p.kept_stride = saved[2].defined() ? saved[2].stride(0) : 0;
                p.x_stride = saved[0].defined() ? row_stride(saved[0], k) : 0;
                p.w_stride = saved[1].defined() ? row_stride(saved[1], k) : 0;
                p.dtype = type_of(dy.scalar_type());
                p.activation = (int)activation;
                const c10::cuda::CUDAGuard guard(dy.device());
                const auto stream = c10::cuda::getCurrentCUDAStream();
                Tensor workspace;
                const size_t size = gk_linear_grad_workspace_bytes(&p);
                if (size > 0) workspace = bytes_on((int64_t)size, dy);
                used(dy, stream);
                auto* status = static_cast<uint32_t*>(ctx->saved_data["status"].toTensor().data_ptr());
                ran("gk_linear_backward", gk_linear_backward(&p, data(workspace), status, stream.stream()));
            }
        }
        return once({dx, dw, db, dr, Tensor(), Tensor(), Tensor()}, "linear");
    }
};

void like_x(const char* name, const Tensor& t, const Tensor& x) {
    TORCH_CHECK_VALUE(t.scalar_type() == x.scalar_type() && t.device() == x.device(),
                      std::string(name) + " must have the dtype and device of x");
}

Tensor linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
              int64_t activation, bool packed, const Tensor& status) {
    TORCH_CHECK_VALUE(x.is_cuda(), "linear requires CUDA tensors");
    TORCH_CHECK_VALUE(type_of(x.scalar_type()) >= 0, "linear takes float32, bfloat16 or float16");
    like_x("weight", weight, x);
    TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && weight.numel() > 0 && x.size(-1) == weight.size(1),
                      "x must have shape [..., K] and weight [N, K], with N and K at least 1");
    const int64_t n = weight.size(0), k = weight.size(1);
    if (has(bias)) {
        like_x("bias", *bias, x);
        TORCH_CHECK_VALUE(bias->dim() == 1 && bias->size(0) == n, "bias must have shape (" + std::to_string(n) + ",)");
    }
    if (has(residual)) {
        like_x("residual", *residual, x);
        TORCH_CHECK_VALUE(residual->dim() == x.dim() && residual->size(-1) == n &&
                              residual->sizes().slice(0, x.dim() - 1) == x.sizes().slice(0, x.dim() - 1),
                          "residual must have the output's shape");
    }
    no_tangent("linear", x, weight, bias, residual);
    const Tensor rows = rows_of(x, k), w = rows_of(weight, k);
    TORCH_CHECK_VALUE(rows.size(0) <= kMost && n <= kMost && k <= kMost, "linear takes sizes below 2**31");
    OptTensor b, r;
    if (has(bias)) b = dense(*bias);
    if (has(residual)) r = rows_of(*residual, n);
    Tensor y;
    if (at::GradMode::is_enabled() && (rows.requires_grad() || w.requires_grad() || (has(b) && b->requires_grad()) ||
                                       (has(r) && r->requires_grad())))
        y = Linear::apply(rows, w, b, r, activation, packed, status);
    else
        y = std::get<0>(linear_forward(rows, w, b, r, activation, false, status));
    if (x.dim() == 2) return y;
    auto shape = x.sizes().vec();
    shape.back() = n;
    return y.view(shape);
}

// ----------------------------------------------------------- policy loss

struct LossScalars {
    double clip_low, clip_high, kl_weight, target_weight, denominator;
};

gk_policy_loss_t loss_struct(const Tensor& logits, const Tensor& mask, const Tensor& actions, const Tensor& old,
                             const Tensor& advantages, const Tensor& reference, const Tensor& target,
                             const Tensor& denominator, const LossScalars& o, const Tensor& workspace) {
    gk_policy_loss_t p{};
    p.logits = logits.data_ptr(), p.rows = logits.size(0), p.cols = logits.size(1);
    p.logits_stride = row_stride(logits, p.cols);
    p.logits_type = type_of(logits.scalar_type());
    if (mask.defined()) p.mask = static_cast<const uint8_t*>(mask.data_ptr()), p.mask_stride = row_stride(mask, p.cols);
    if (target.defined()) {
        p.target = target.data_ptr(), p.target_stride = row_stride(target, p.cols);
        p.target_type = type_of(target.scalar_type());
        p.target_weight = (float)o.target_weight;
    }
    if (actions.defined()) {
        p.actions = actions.const_data_ptr<int64_t>();
        p.old_log_probs = old.const_data_ptr<float>(), p.advantages = advantages.const_data_ptr<float>();
        p.clip_low = (float)o.clip_low, p.clip_high = (float)o.clip_high;
    }
    if (reference.defined()) p.reference_log_probs = reference.const_data_ptr<float>(), p.kl_weight = (float)o.kl_weight;
    p.denominator = (float)o.denominator;
    if (denominator.defined()) p.denominator_ptr = denominator.const_data_ptr<float>();
    // Row statistics (four floats a row), then the partial sums (doubles).
    p.stats = static_cast<float*>(workspace.data_ptr());
    p.partials = static_cast<double*>(workspace.data_ptr()) + 2 * p.rows;
    return p;
}

Tensor or_none(const OptTensor& t) { return has(t) ? *t : Tensor(); }

// (loss, log-probabilities, gradient, workspace).
std::tuple<Tensor, Tensor, Tensor, Tensor> loss_forward(const Tensor& logits, const Tensor& mask,
                                                        const Tensor& actions, const Tensor& old,
                                                        const Tensor& advantages, const Tensor& reference,
                                                        const Tensor& target, const Tensor& denominator,
                                                        const LossScalars& o, bool with_grad) {
    const int64_t n = logits.size(0);
    const auto floats = logits.options().dtype(at::kFloat).requires_grad(false);
    Tensor workspace = at::empty({2 * n + gk_policy_loss_parts(n, logits.size(1))}, floats.dtype(at::kDouble));
    Tensor loss = at::empty({}, floats), log_probs, grad;
    if (actions.defined()) log_probs = at::empty({n}, floats);
    if (with_grad) grad = at::empty(logits.sizes(), logits.options().requires_grad(false));
    gk_policy_loss_t p = loss_struct(logits, mask, actions, old, advantages, reference, target, denominator, o,
                                     workspace);
    p.loss = loss.data_ptr<float>();
    p.log_probs = log_probs.defined() ? log_probs.data_ptr<float>() : nullptr;
    p.grad = data(grad);
    const c10::cuda::CUDAGuard guard(logits.device());
    const auto stream = c10::cuda::getCurrentCUDAStream();
    for (const Tensor* t : {&logits, &mask, &actions, &old, &advantages, &reference, &target, &denominator})
        used(*t, stream);
    ran("gk_policy_loss_forward", gk_policy_loss_forward(&p, stream.stream()));
    return {loss, log_probs, grad, workspace};
}

struct PolicyLoss : torch::autograd::Function<PolicyLoss> {
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const OptTensor& mask,
                                 const OptTensor& actions, const OptTensor& old, const OptTensor& advantages,
                                 const OptTensor& reference, const OptTensor& target, const OptTensor& denominator,
                                 const std::vector<double>& o) {
        const LossScalars scalars{o[0], o[1], o[2], o[3], o[4]};
        // fp16 training scales its loss, so a gradient for an upstream of one
        // would be computed in vain; the other types get it in the same pass.
        auto [loss, log_probs, grad, workspace] =
            loss_forward(logits, or_none(mask), or_none(actions), or_none(old), or_none(advantages),
                         or_none(reference), or_none(target), or_none(denominator), scalars,
                         logits.scalar_type() != at::kHalf);
        ctx->save_for_backward({logits, or_none(mask), or_none(actions), or_none(old), or_none(advantages),
                                or_none(reference), or_none(target), or_none(denominator), workspace});
        ctx->saved_data["o"] = o;
        if (grad.defined()) ctx->saved_data["grad"] = grad;
        if (!log_probs.defined()) log_probs = at::empty({0}, loss.options());
        ctx->mark_non_differentiable({log_probs});
        return {loss, log_probs};
    }

    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const variable_list s = ctx->get_saved_variables();  // raises if an input was modified in place
        const auto o = ctx->saved_data["o"].toDoubleVector();
        Tensor grad;
        {
            const at::NoGradGuard no_grad;
            // The gradient of the forward pass is handed out once; a further pass makes its own.
            auto found = ctx->saved_data.find("grad");
            const bool written = found != ctx->saved_data.end();
            if (written) {
                grad = found->second.toTensor();
                ctx->saved_data.erase(found);
            } else {
                grad = at::empty(s[0].sizes(), s[0].options().requires_grad(false));
            }
            if (s[0].size(0) > 0) {
                const Tensor upstream = dense(grads[0]);
                gk_policy_loss_t p = loss_struct(s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7],
                                                 LossScalars{o[0], o[1], o[2], o[3], o[4]}, s[8]);
                p.loss = p.stats;  // not written by the backward pass
                p.grad = grad.data_ptr();
                const c10::cuda::CUDAGuard guard(s[0].device());
                const auto stream = c10::cuda::getCurrentCUDAStream();
                used(upstream, stream);
                ran("gk_policy_loss_backward",
                    gk_policy_loss_backward(&p, upstream.const_data_ptr<float>(), written ? 1 : 0, stream.stream()));
            }
        }
        variable_list out(9);
        out[0] = grad;
        return once(out, "policy_loss");
    }
};

constexpr const char* kNoGradient = " must not require a gradient: the loss differentiates by its logits alone";

OptTensor column(const char* name, const OptTensor& t, const Tensor& logits, at::ScalarType dtype) {
    if (!has(t)) return std::nullopt;
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == logits.size(0) && t->scalar_type() == dtype &&
                          t->device() == logits.device(),
                      std::string(name) + " must have shape (" + std::to_string(logits.size(0)) + ",), dtype " +
                          c10::toString(dtype) + " and the logits' device");
    TORCH_CHECK_VALUE(!t->requires_grad(), std::string(name) + kNoGradient);
    return dense(*t);
}

OptTensor matrix(const char* name, const OptTensor& t, const Tensor& logits, bool fits) {
    if (!has(t)) return std::nullopt;
    TORCH_CHECK_VALUE(t->sizes() == logits.sizes() && fits && t->device() == logits.device(),
                      std::string(name) + " must have the logits' shape and device; legal_mask is bool, a target "
                                          "fp32 or of the logits' dtype");
    TORCH_CHECK_VALUE(!t->requires_grad(), std::string(name) + kNoGradient);
    return rows_of(*t, logits.size(1));
}

std::tuple<Tensor, Tensor> policy_loss(const Tensor& logits, const OptTensor& legal_mask, const OptTensor& actions,
                                       const OptTensor& old, const OptTensor& advantages, const OptTensor& reference,
                                       const OptTensor& target, double clip_low, double clip_high, double kl_weight,
                                       double target_weight, double denominator, const OptTensor& denominator_tensor) {
    TORCH_CHECK_VALUE(logits.is_cuda(), "policy_loss requires CUDA logits");
    TORCH_CHECK_VALUE(logits.dim() == 2 && type_of(logits.scalar_type()) >= 0 && logits.size(1) >= 1 &&
                          logits.size(1) <= kMostColumns,
                      "logits must have shape [N, A] with A > 0 and dtype float32, bfloat16 or float16");
    if (!has(actions)) {
        TORCH_CHECK_VALUE(!has(old) && !has(advantages) && !has(reference),
                          "old_log_probs, advantages and reference_log_probs go with actions");
        TORCH_CHECK_VALUE(has(target), "policy_loss needs actions or a target");
    } else {
        TORCH_CHECK_VALUE(has(old) && has(advantages), "actions go with old_log_probs and advantages");
    }
    if (has(denominator_tensor)) {
        TORCH_CHECK_VALUE(denominator_tensor->numel() == 1 && denominator_tensor->scalar_type() == at::kFloat &&
                              denominator_tensor->device() == logits.device(),
                          "denominator must hold one float32 on the logits' device");
        TORCH_CHECK_VALUE(!denominator_tensor->requires_grad(), "denominator must not require a gradient");
    }
    no_tangent("policy_loss", logits, old, advantages, reference, target, denominator_tensor);
    const Tensor z = rows_of(logits, logits.size(1));
    const OptTensor mask = matrix("legal_mask", legal_mask, logits,
                                  has(legal_mask) && legal_mask->scalar_type() == at::kBool);
    const OptTensor t = matrix("target", target, logits,
                               has(target) && (target->scalar_type() == at::kFloat ||
                                               target->scalar_type() == logits.scalar_type()));
    const OptTensor a = column("actions", actions, logits, at::kLong);
    const OptTensor q = column("old_log_probs", old, logits, at::kFloat);
    const OptTensor adv = column("advantages", advantages, logits, at::kFloat);
    const OptTensor ref = column("reference_log_probs", reference, logits, at::kFloat);
    if (at::GradMode::is_enabled() && z.requires_grad()) {
        const auto out = PolicyLoss::apply(z, mask, a, q, adv, ref, t, denominator_tensor,
                                           std::vector<double>{clip_low, clip_high, kl_weight, target_weight,
                                                               denominator});
        return {out[0], out[1]};
    }
    auto [loss, log_probs, grad, workspace] =
        loss_forward(z, or_none(mask), or_none(a), or_none(q), or_none(adv), or_none(ref), or_none(t),
                     or_none(denominator_tensor),
                     LossScalars{clip_low, clip_high, kl_weight, target_weight, denominator}, false);
    if (!log_probs.defined()) log_probs = at::empty({0}, loss.options());
    return {loss, log_probs};
}

}  // namespace

TORCH_LIBRARY(gk, m) {
    m.def("pack(Tensor x) -> (Tensor, Tensor)", pack);
    m.def("unpack(Tensor codes, Tensor scales, int[] shape, ScalarType dtype) -> Tensor", unpack);
    m.def("linear(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, int activation, bool packed, "
          "Tensor status) -> Tensor",
          linear);
    m.def("policy_loss(Tensor logits, Tensor? legal_mask, Tensor? actions, Tensor? old_log_probs, "
          "Tensor? advantages, Tensor? reference_log_probs, Tensor? target, float clip_low, float clip_high, "
          "float kl_weight, float target_weight, float denominator, Tensor? denominator_tensor) -> (Tensor, Tensor)",
          policy_loss);
}
