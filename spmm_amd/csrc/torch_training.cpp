// torch_training.cpp -- the training operators (include/tca_train.h) as torch
// operators of namespace spmm_amd, autograd formulas included:
//
//   layer_norm, layer_norm_stats, layer_norm_backward
//   cross_entropy, cross_entropy_stats, cross_entropy_backward, cross_entropy_grad
//   adamw_step_, adamw_step_device_
//
// Host code only, in C++ because small calls are bound by the host: a forward and
// backward layer norm of 8 rows takes 73 us here and 124 us as a Python autograd
// function around ctypes calls, whose backward has to take the interpreter's
// lock on autograd's thread.  Checks raise ValueError or TypeError, errors of the
// library RuntimeError with its message.  Everything runs on the current stream
// of the tensors' device; workspaces come from torch's allocator.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <cmath>
#include <optional>
#include <tuple>
#include <vector>

#include "../../include/tca_train.h"

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The library's value type of a torch dtype, or -1.
int32_t value_type(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return TCA_F32;
        case at::kHalf: return TCA_F16;
        case at::kBFloat16: return TCA_BF16;
        default: return -1;
    }
}

const void* address(const optional<Tensor>& t) { return t ? t->const_data_ptr() : nullptr; }

// The device's current stream, with the device made current for the launch.
struct Launch {
    c10::DeviceGuard guard;
    void* stream;
    explicit Launch(const Tensor& t)
        : guard(t.device()), stream(t.is_cuda() ? c10::hip::getCurrentHIPStream(t.device().index()).stream() : nullptr) {}
};

void check(int status, const char* name) { TORCH_CHECK(status == TCA_OK, name, ": ", tca_last_error()); }

// t as a matrix of rows along its last axis, a view where t's strides allow one:
// any distance between rows, neighbouring columns side by side.
Tensor as_rows(const Tensor& t) {
    Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
    return r.size(1) == 1 || (r.stride(1) == 1 && r.stride(0) >= 0) ? r : r.contiguous();
}

optional<Tensor> dense(const optional<Tensor>& t) {
    return t && t->defined() ? optional<Tensor>(t->contiguous()) : std::nullopt;
}

bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
bool wants_grad(const optional<Tensor>& t) { return t && wants_grad(*t); }

// A tangent is refused: below autograd's keys it would be lost without a word.
void check_tangent(const char* name, const Tensor& t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), name,
                                ": forward-mode derivatives are not implemented");
}
void check_tangent(const char* name, const optional<Tensor>& t) {
    if (t) check_tangent(name, *t);
}

// ---------------------------------------------------------------- layer norm
void check_norm(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, double eps,
                at::ScalarType out) {
    TORCH_CHECK_VALUE(x.is_cuda(), "layer_norm: x must be a GPU tensor (no CPU fallback)");
    TORCH_CHECK_TYPE(value_type(x.scalar_type()) >= 0, "layer_norm: x must be float32, float16 or bfloat16, got ",
                     x.scalar_type());
    TORCH_CHECK_TYPE(value_type(out) >= 0 && (out == x.scalar_type() || x.scalar_type() == at::kFloat),
                     "layer_norm: the output has x's dtype, or any for float32 x; got ", x.scalar_type(), " -> ", out);
    TORCH_CHECK_VALUE(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= TCA_LAYER_NORM_MAX_WIDTH,
                      "layer_norm: the last axis must have 1 to ", TCA_LAYER_NORM_MAX_WIDTH, " entries, got ", x.sizes());
    TORCH_CHECK_VALUE(eps >= 0 && std::isfinite(eps), "layer_norm: eps must be at least 0, got ", eps);
    for (const auto* t : {&weight, &bias}) {
        if (!*t || !(*t)->defined()) continue;
        const char* name = t == &weight ? "weight" : "bias";
        TORCH_CHECK_VALUE((*t)->device() == x.device(), "layer_norm: ", name, " is on ", (*t)->device(), ", x on ",
                          x.device());
        TORCH_CHECK_VALUE((*t)->dim() == 1 && (*t)->size(0) == x.size(-1), "layer_norm: ", name, " must be 1-D with ",
                          x.size(-1), " entries, got ", (*t)->sizes());
        const auto type = (*t)->scalar_type();
        TORCH_CHECK_TYPE(type == x.scalar_type() || type == out || type == at::kFloat, "layer_norm: ", name,
                         " must have the dtype of x, of the output or float32, got ", type);
    }
    TORCH_CHECK_TYPE(!weight || !bias || weight->scalar_type() == bias->scalar_type(),
                     "layer_norm: weight and bias have different dtypes");
}

at::ScalarType weight_type(const optional<Tensor>& weight, const optional<Tensor>& bias) {
    return weight ? weight->scalar_type() : bias ? bias->scalar_type() : at::kFloat;
}

std::tuple<Tensor, Tensor> norm_forward(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias,
                                        double eps, optional<at::ScalarType> out_dtype, bool want_stats) {
    const auto out = out_dtype.value_or(x.scalar_type());
    check_norm(x, weight, bias, eps, out);
    const Tensor xr = as_rows(x);
    const auto w = dense(weight), b = dense(bias);
    const Launch launch(x);
    Tensor y = at::empty(x.sizes(), x.options().dtype(out));
    Tensor stats = want_stats ? at::empty({xr.size(0), 2}, x.options().dtype(at::kFloat)) : Tensor();
    check(tca_layer_norm(xr.const_data_ptr(), xr.size(0), static_cast<int32_t>(xr.size(1)), xr.stride(0),
                         value_type(x.scalar_type()), address(w), address(b), value_type(weight_type(weight, bias)),
                         static_cast<float>(eps), y.mutable_data_ptr(), value_type(out),
                         want_stats ? stats.mutable_data_ptr<float>() : nullptr, launch.stream),
          "layer_norm");
    return {std::move(y), std::move(stats)};
}

Tensor layer_norm(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, double eps,
                  optional<at::ScalarType> out_dtype) {
    return std::get<0>(norm_forward(x, weight, bias, eps, out_dtype, false));
}

std::tuple<Tensor, Tensor> layer_norm_stats(const Tensor& x, const optional<Tensor>& weight,
                                            const optional<Tensor>& bias, double eps,
                                            optional<at::ScalarType> out_dtype) {
    return norm_forward(x, weight, bias, eps, out_dtype, true);
}

// dx, dweight, dbias; an empty tensor for each that is not needed.
std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const Tensor& dy, const Tensor& x, const optional<Tensor>& weight,
                                                       const Tensor& stats, bool need_dx, bool need_dw, bool need_db,
                                                       at::ScalarType weight_dtype) {
    check_norm(x, weight, std::nullopt, 0.0, dy.scalar_type());
    const Tensor xr = as_rows(x);
    const int64_t rows = xr.size(0);
    const auto width = static_cast<int32_t>(xr.size(1));
    TORCH_CHECK_VALUE(dy.sizes() == x.sizes() && dy.device() == x.device(), "layer_norm_backward: dy must be like x");
    TORCH_CHECK_TYPE(!weight || weight->scalar_type() == weight_dtype,
                     "layer_norm_backward: weight_dtype must be the weight's");
    TORCH_CHECK_VALUE(stats.scalar_type() == at::kFloat && stats.numel() == 2 * rows && stats.is_contiguous() &&
                          stats.device() == x.device(),
                      "layer_norm_backward: stats must be what layer_norm_stats gave for x");
    const Tensor dyr = as_rows(dy);
    const auto w = dense(weight);
    const Launch launch(x);
    Tensor dx = at::empty(need_dx ? x.sizes() : at::IntArrayRef{0}, x.options());
    Tensor dw = at::empty({need_dw ? width : 0}, x.options().dtype(weight_dtype));
    Tensor db = at::empty({need_db ? width : 0}, x.options().dtype(weight_dtype));
    size_t size = 0;
    Tensor work;
    if (need_dw || need_db) {
        check(tca_layer_norm_backward_workspace(rows, width, &size), "layer_norm_backward");
        work = at::empty({static_cast<int64_t>(size)}, x.options().dtype(at::kByte));
    }
    check(tca_layer_norm_backward(dyr.const_data_ptr(), dyr.stride(0), value_type(dy.scalar_type()),
                                  xr.const_data_ptr(), xr.stride(0), value_type(x.scalar_type()), rows, width,
                                  address(w), value_type(weight_dtype), stats.const_data_ptr<float>(),
                                  need_dx ? dx.mutable_data_ptr() : nullptr, need_dw ? dw.mutable_data_ptr() : nullptr,
                                  need_db ? db.mutable_data_ptr() : nullptr,
                                  work.defined() ? work.mutable_data_ptr() : nullptr, size, launch.stream),
          "layer_norm_backward");
    return {std::move(dx), std::move(dw), std::move(db)};
}

template <typename F>
auto operation(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

// Where no second derivative can be asked for, a backward operation goes past
// autograd's keys; where one can, it meets the kernel there that refuses it.
struct BelowAutograd {
    optional<at::AutoDispatchBelowADInplaceOrView> below;
    BelowAutograd() {
        if (!at::GradMode::is_enabled()) below.emplace();
    }
};

struct LayerNorm : torch::autograd::Function<LayerNorm> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& weight,
                          const optional<Tensor>& bias, double eps, optional<at::ScalarType> out_dtype) {
        static const auto op = operation<decltype(layer_norm_stats)>("spmm_amd::layer_norm_stats");
        const at::AutoDispatchBelowADInplaceOrView below;
        auto [y, stats] = op.call(x, weight, bias, eps, out_dtype);
        ctx->save_for_backward({x, weight.value_or(Tensor()), stats});
        ctx->saved_data["type"] = static_cast<int64_t>(weight_type(weight, bias));
        ctx->saved_data["weight"] = weight.has_value();
        ctx->saved_data["bias"] = bias.has_value();
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list dy) {
        static const auto op = operation<decltype(layer_norm_backward)>("spmm_amd::layer_norm_backward");
        const auto saved = ctx->get_saved_variables();
        const bool weight = ctx->saved_data["weight"].toBool(), bias = ctx->saved_data["bias"].toBool();
        // gradients are asked for by position among the tensors that were given
        const bool dx = ctx->needs_input_grad(0), dw = weight && ctx->needs_input_grad(1);
        const bool db = bias && ctx->needs_input_grad(weight ? 2 : 1);
        const BelowAutograd below;
        auto [gx, gw, gb] =
            op.call(dy[0], saved[0], saved[1].defined() ? optional<Tensor>(saved[1]) : std::nullopt, saved[2], dx, dw, db,
                    static_cast<at::ScalarType>(ctx->saved_data["type"].toInt()));
        return {dx ? gx : Tensor(), dw ? gw : Tensor(), db ? gb : Tensor(), Tensor(), Tensor()};
    }
};

Tensor layer_norm_autograd(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, double eps,
                           optional<at::ScalarType> out_dtype) {
    check_tangent("layer_norm", x);
    check_tangent("layer_norm", weight);
    check_tangent("layer_norm", bias);
    if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(weight) || wants_grad(bias)))
        return LayerNorm::apply(x, weight, bias, eps, out_dtype);
    static const auto op = operation<decltype(layer_norm)>("spmm_amd::layer_norm");
    const at::AutoDispatchBelowADInplaceOrView below;
    return op.call(x, weight, bias, eps, out_dtype);
}

// -------------------------------------------------------------- cross entropy
struct LossInput {
    Tensor x, target;
    LossInput(const char* name, const Tensor& logits, const Tensor& t) {
        TORCH_CHECK_VALUE(logits.is_cuda() && t.device() == logits.device(), name,
                          ": logits and target must be tensors of one GPU (no CPU fallback)");
        TORCH_CHECK_TYPE(value_type(logits.scalar_type()) >= 0, name,
                         ": logits must be float32, float16 or bfloat16, got ", logits.scalar_type());
        TORCH_CHECK_TYPE(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, name,
                         ": target must be int64 or int32, got ", t.scalar_type());
        TORCH_CHECK_VALUE(logits.dim() == 2 && logits.size(1) >= 1 && logits.size(1) <= INT32_MAX, name,
                          ": logits must be rows x classes, got ", logits.sizes());
        TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == logits.size(0), name, ": target must be 1-D with ",
                          logits.size(0), " entries, got ", t.sizes());
        x = as_rows(logits);
        // rows further apart than the library takes: their copy holds the rows alone
        if (x.stride(0) > INT32_MAX) x = x.clone(at::MemoryFormat::Contiguous);
        target = t.contiguous();
    }
    int64_t rows() const { return x.size(0); }
    int32_t classes() const { return static_cast<int32_t>(x.size(1)); }
    int32_t type() const { return value_type(x.scalar_type()); }
    int32_t target_bytes() const { return static_cast<int32_t>(target.element_size()); }
    at::TensorOptions f32() const { return x.options().dtype(at::kFloat); }
};

struct Workspace {
    size_t size = 0;
    Tensor bytes;
    explicit Workspace(const LossInput& in) {
        check(tca_cross_entropy_workspace(in.rows(), in.classes(), &size), "cross_entropy");
        bytes = at::empty({static_cast<int64_t>(size)}, in.x.options().dtype(at::kByte));
    }
};

std::tuple<Tensor, Tensor, Tensor> loss_forward(const Tensor& logits, const Tensor& target, int64_t ignore_index,
                                                int64_t reduction, bool want_grad) {
    const LossInput in("cross_entropy", logits, target);
    const Launch launch(logits);
    const Workspace work(in);
    const bool mean = reduction == TCA_LOSS_MEAN;
    Tensor loss = reduction == TCA_LOSS_NONE ? at::empty({in.rows()}, in.f32()) : at::empty({}, in.f32());
    Tensor stats = want_grad ? at::empty({in.rows(), 2}, in.f32()) : Tensor();
    Tensor norm = want_grad ? (mean ? at::empty({}, in.f32()) : at::empty({0}, in.f32())) : Tensor();
    check(tca_cross_entropy(in.x.const_data_ptr(), in.rows(), in.classes(), in.x.stride(0), in.type(),
                            in.target.const_data_ptr(), in.target_bytes(), ignore_index,
                            static_cast<int32_t>(reduction), loss.mutable_data_ptr<float>(),
                            want_grad ? stats.mutable_data_ptr<float>() : nullptr,
                            want_grad && mean ? norm.mutable_data_ptr<float>() : nullptr, work.bytes.mutable_data_ptr(),
                            work.size, launch.stream),
          "cross_entropy");
    return {std::move(loss), std::move(stats), std::move(norm)};
}

Tensor cross_entropy(const Tensor& logits, const Tensor& target, int64_t ignore_index, int64_t reduction) {
    return std::get<0>(loss_forward(logits, target, ignore_index, reduction, false));
}

// The loss, the rows' {max, sum} and, for the mean, 1 / count (else empty).
std::tuple<Tensor, Tensor, Tensor> cross_entropy_stats(const Tensor& logits, const Tensor& target, int64_t ignore_index,
                                                       int64_t reduction) {
    return loss_forward(logits, target, ignore_index, reduction, true);
}

Tensor cross_entropy_backward(const Tensor& gloss, const Tensor& logits, const Tensor& target, int64_t ignore_index,
                              const Tensor& stats, const Tensor& norm) {
    const LossInput in("cross_entropy_backward", logits, target);
    const Tensor g = gloss.to(at::kFloat);
    TORCH_CHECK_VALUE((g.dim() == 0 || (g.dim() == 1 && g.size(0) == in.rows())) && g.device() == logits.device(),
                      "cross_entropy_backward: gloss must be a scalar or one value per row");
    TORCH_CHECK_VALUE(stats.scalar_type() == at::kFloat && stats.numel() == 2 * in.rows() && stats.is_contiguous() &&
                          stats.device() == logits.device() && norm.scalar_type() == at::kFloat &&
                          norm.device() == logits.device(),
                      "cross_entropy_backward: stats and norm must be what cross_entropy_stats gave");
    const Launch launch(logits);
    Tensor dx = at::empty(logits.sizes(), logits.options());
    check(tca_cross_entropy_backward(g.const_data_ptr<float>(), g.dim() ? g.stride(0) : 0, in.x.const_data_ptr(),
                                     in.rows(), in.classes(), in.x.stride(0), in.type(), in.target.const_data_ptr(),
                                     in.target_bytes(), ignore_index, stats.const_data_ptr<float>(),
                                     norm.numel() ? norm.const_data_ptr<float>() : nullptr, dx.mutable_data_ptr(),
                                     launch.stream),
          "cross_entropy_backward");
    return dx;
}

std::tuple<Tensor, Tensor> cross_entropy_grad(const Tensor& logits, const Tensor& target, int64_t ignore_index,
                                              int64_t reduction, double scale) {
    const LossInput in("cross_entropy_grad", logits, target);
    const Launch launch(logits);
    const Workspace work(in);
    Tensor loss = at::empty({}, in.f32());
    Tensor dx = at::empty(logits.sizes(), logits.options());
    check(tca_cross_entropy_grad(in.x.const_data_ptr(), in.rows(), in.classes(), in.x.stride(0), in.type(),
                                 in.target.const_data_ptr(), in.target_bytes(), ignore_index,
                                 static_cast<int32_t>(reduction), static_cast<float>(scale),
                                 loss.mutable_data_ptr<float>(), dx.mutable_data_ptr(), work.bytes.mutable_data_ptr(),
                                 work.size, launch.stream),
          "cross_entropy_grad");
    return {std::move(loss), std::move(dx)};
}

struct CrossEntropy : torch::autograd::Function<CrossEntropy> {
    static Tensor forward(AutogradContext* ctx, const Tensor& logits, const Tensor& target, int64_t ignore_index,
                          int64_t reduction) {
        static const auto op = operation<decltype(cross_entropy_stats)>("spmm_amd::cross_entropy_stats");
        const at::AutoDispatchBelowADInplaceOrView below;
        auto [loss, stats, norm] = op.call(logits, target, ignore_index, reduction);
        ctx->save_for_backward({logits, target, stats, norm});
        ctx->saved_data["ignore"] = ignore_index;
        return loss;
    }
    static variable_list backward(AutogradContext* ctx, variable_list g) {
        static const auto op = operation<decltype(cross_entropy_backward)>("spmm_amd::cross_entropy_backward");
        const auto saved = ctx->get_saved_variables();
        const BelowAutograd below;
        return {op.call(g[0], saved[0], saved[1], ctx->saved_data["ignore"].toInt(), saved[2], saved[3]), Tensor(),
                Tensor(), Tensor()};
    }
};

Tensor cross_entropy_autograd(const Tensor& logits, const Tensor& target, int64_t ignore_index, int64_t reduction) {
    check_tangent("cross_entropy", logits);
    if (at::GradMode::is_enabled() && wants_grad(logits))
        return CrossEntropy::apply(logits, target, ignore_index, reduction);
    static const auto op = operation<decltype(cross_entropy)>("spmm_amd::cross_entropy");
    const at::AutoDispatchBelowADInplaceOrView below;
    return op.call(logits, target, ignore_index, reduction);
}

// Its outputs are constants to autograd in either mode, the gradient among them.
std::tuple<Tensor, Tensor> cross_entropy_grad_autograd(const Tensor& logits, const Tensor& target, int64_t ignore_index,
                                                       int64_t reduction, double scale) {
    static const auto op = operation<decltype(cross_entropy_grad)>("spmm_amd::cross_entropy_grad");
    const at::AutoDispatchBelowADInplaceOrView below;
    return op.call(logits, target, ignore_index, reduction, scale);
}

// ---------------------------------------------------------------------- AdamW
// Address of a state tensor that has n contiguous values of `type` on `device`.
void* held(const Tensor& t, const char* name, at::ScalarType type, int64_t n, c10::Device device) {
    TORCH_CHECK_VALUE(t.scalar_type() == type && t.numel() == n && t.device() == device && t.is_contiguous(),
                      "AdamW: state '", name, "' must be contiguous ", type, " with ", n, " entries on ", device,
                      "; got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
    return t.data_ptr();
}

// The tensors of one step: parameters of one dtype and device.  `states` holds
// their state tensors one kind after the other: exp_avg and exp_avg_sq, or exp_avg,
// exp_avg_rms and their scales; then the masters of 16-bit parameters.
struct AdamTable {
    std::vector<tca_adamw_tensor> table;
    std::vector<Tensor> copies;  // of gradients with strides, until the launches are queued
    int32_t type = -1;

    AdamTable(at::TensorList params, at::TensorList grads, at::TensorList states, int64_t state_bits)
        : table(params.size()) {
        const auto count = params.size();
        const Tensor& lead = params[0];
        const auto dtype = lead.scalar_type();
        const auto device = lead.device();
        type = value_type(dtype);
        TORCH_CHECK_VALUE(lead.is_cuda() && type >= 0,
                          "AdamW: parameters must be float32, float16 or bfloat16 GPU tensors (no CPU fallback), got ",
                          dtype, " on ", device);
        const bool master = dtype != at::kFloat, bits8 = state_bits == 8;
        const size_t kinds = (bits8 ? 4 : 2) + (master ? 1 : 0);
        TORCH_CHECK_VALUE(grads.size() == count && states.size() == kinds * count, "AdamW: ", count, " parameters, ",
                          grads.size(), " gradients, ", states.size(), " states");
        const auto state = [&](size_t kind, size_t k) -> const Tensor& { return states[kind * count + k]; };
        for (size_t k = 0; k < count; ++k) {
            const Tensor &p = params[k], &g = grads[k];
            const int64_t n = p.numel(), blocks = (n + TCA_ADAMW_BLOCK - 1) / TCA_ADAMW_BLOCK;
            TORCH_CHECK_VALUE(p.scalar_type() == dtype && p.device() == device && p.is_contiguous(),
                              "AdamW: parameters must be contiguous");
            TORCH_CHECK_VALUE(g.layout() == at::kStrided, "AdamW: sparse gradients are not supported");
            TORCH_CHECK_TYPE(g.scalar_type() == dtype && g.device() == device && g.sizes() == p.sizes(),
                             "AdamW: a gradient must have its parameter's dtype, device and shape; got ",
                             g.scalar_type(), " ", g.sizes(), " on ", g.device(), " for ", dtype, " ", p.sizes(),
                             " on ", device);
            tca_adamw_tensor& t = table[k];
            t.n = n;
            t.param = p.mutable_data_ptr();
            if (g.is_contiguous()) {
                t.grad = g.const_data_ptr();
            } else {
                copies.push_back(g.contiguous());
                t.grad = copies.back().const_data_ptr();
            }
            if (bits8) {
                const int64_t size = blocks * TCA_ADAMW_BLOCK;
                t.m = held(state(0, k), "exp_avg", at::kFloat8_e4m3fn, size, device);
                t.v = held(state(1, k), "exp_avg_rms", at::kFloat8_e4m3fn, size, device);
                t.m_scale = static_cast<float*>(held(state(2, k), "exp_avg_scale", at::kFloat, blocks, device));
                t.v_scale = static_cast<float*>(held(state(3, k), "exp_avg_rms_scale", at::kFloat, blocks, device));
            } else {
                t.m = held(state(0, k), "exp_avg", at::kFloat, n, device);
                t.v = held(state(1, k), "exp_avg_sq", at::kFloat, n, device);
                t.m_scale = t.v_scale = nullptr;
            }
            t.master =
                master ? static_cast<float*>(held(state(kinds - 1, k), "master", at::kFloat, n, device)) : nullptr;
        }
    }
    int32_t count() const { return static_cast<int32_t>(table.size()); }
};

// A backward pass that saved a parameter notices that it has changed.
void bump(at::TensorList params) {
    for (const Tensor& p : params) p.unsafeGetTensorImpl()->bump_version();
}

// One step of parameters that have taken the same number of them.
void adamw_step_(at::TensorList params, at::TensorList grads, at::TensorList states, int64_t state_bits, int64_t step,
                 double lr, double beta1, double beta2, double eps, double weight_decay) {
    if (params.empty()) return;
    const Launch launch(params[0]);
    const AdamTable t(params, grads, states, state_bits);
    check(tca_adamw_step(t.table.data(), t.count(), t.type, static_cast<int32_t>(state_bits), step, lr, beta1, beta2, eps,
                         weight_decay, launch.stream),
          "AdamW");
    bump(params);
}

// The same with an int64 step count on the GPU for each parameter, raised here.
void adamw_step_device_(at::TensorList params, at::TensorList grads, at::TensorList states, at::TensorList steps,
                        int64_t state_bits, double lr, double beta1, double beta2, double eps, double weight_decay) {
    if (params.empty()) return;
    const Launch launch(params[0]);
    const AdamTable t(params, grads, states, state_bits);
    TORCH_CHECK_VALUE(steps.size() == params.size(), "AdamW: ", params.size(), " parameters, ", steps.size(), " steps");
    std::vector<int64_t*> counts;
    for (const Tensor& step : steps)
        counts.push_back(static_cast<int64_t*>(held(step, "step", at::kLong, 1, params[0].device())));
    Tensor factors = at::empty({2 * t.count()}, params[0].options().dtype(at::kFloat));
    check(tca_adamw_step_device(t.table.data(), counts.data(), t.count(), t.type, static_cast<int32_t>(state_bits), lr,
                                beta1, beta2, eps, weight_decay, factors.mutable_data_ptr<float>(), launch.stream),
          "AdamW");
    bump(params);
}

TORCH_LIBRARY_FRAGMENT(spmm_amd, m) {
    m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, ScalarType? out_dtype) -> Tensor");
    m.def("layer_norm_stats(Tensor x, Tensor? weight, Tensor? bias, float eps, ScalarType? out_dtype) -> (Tensor, Tensor)");
    m.def("layer_norm_backward(Tensor dy, Tensor x, Tensor? weight, Tensor stats, bool need_dx, bool need_dw, "
          "bool need_db, ScalarType weight_dtype) -> (Tensor, Tensor, Tensor)");
    m.def("cross_entropy(Tensor logits, Tensor target, int ignore_index, int reduction) -> Tensor");
    m.def("cross_entropy_stats(Tensor logits, Tensor target, int ignore_index, int reduction) "
          "-> (Tensor, Tensor, Tensor)");
    m.def("cross_entropy_backward(Tensor gloss, Tensor logits, Tensor target, int ignore_index, Tensor stats, "
          "Tensor norm) -> Tensor");
    m.def("cross_entropy_grad(Tensor logits, Tensor target, int ignore_index, int reduction, float scale) "
          "-> (Tensor, Tensor)");
    m.def("adamw_step_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] states, int state_bits, int step, float lr, "
          "float beta1, float beta2, float eps, float weight_decay) -> ()");
    m.def("adamw_step_device_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] states, Tensor(c!)[] steps, "
          "int state_bits, float lr, float beta1, float beta2, float eps, float weight_decay) -> ()");
}

// For every device: what is not a GPU tensor is refused by name.
TORCH_LIBRARY_IMPL(spmm_amd, CompositeExplicitAutograd, m) {
    m.impl("layer_norm", layer_norm);
    m.impl("layer_norm_stats", layer_norm_stats);
    m.impl("layer_norm_backward", layer_norm_backward);
    m.impl("cross_entropy", cross_entropy);
    m.impl("cross_entropy_stats", cross_entropy_stats);
    m.impl("cross_entropy_backward", cross_entropy_backward);
    m.impl("cross_entropy_grad", cross_entropy_grad);
    m.impl("adamw_step_", adamw_step_);
    m.impl("adamw_step_device_", adamw_step_device_);
}

TORCH_LIBRARY_IMPL(spmm_amd, Autograd, m) {
    m.impl("layer_norm", layer_norm_autograd);
    m.impl("cross_entropy", cross_entropy_autograd);
    m.impl("cross_entropy_grad", cross_entropy_grad_autograd);
    for (const char* name : {"layer_norm_stats", "layer_norm_backward", "cross_entropy_stats", "cross_entropy_backward"})
        m.impl(name, torch::autograd::autogradNotImplementedFallback());
}

}  // namespace
