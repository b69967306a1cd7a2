// PyTorch operators of the logits-level steps over the C ABI (include/trlk.h): log-probs and entropies, the GRPO and DPO
// losses and what they log.  A step of a small run consists of a dozen launches of a few microseconds, so what a call
// costs on the host counts: an operator registered from Python spends 10 to 15 us per call in Python layers (argument
// conversion, the autograd and aliasing wrappers, ctypes, one Python tensor object per temporary), one registered here 3
// to 5.  Their shapes for tracers are registered in ops.py.
//
// Each operator checks its shapes, allocates its outputs and hands raw device pointers, sizes, strides and the
// current stream of the tensors' device to the library.  GPU tensors only: other devices have no kernel registered.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_strided.h>
#include <ATen/ops/zeros.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/InferenceMode.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>
#include <torch/python.h>

#include <algorithm>
#include <limits>
#include <cstdlib>
#include <map>
#include <mutex>
#include <string>

#include "trlk.h"

namespace {
using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A status of the library as the exception class that the Python package raises for it.
void check(int status) {
    if (status == 0) return;
    const std::string what = (status < 0 ? "trlk status " : "trlk launch failed with hipError_t ") + std::to_string(status) +
                             ": " + trlk_last_error();
    pybind11::gil_scoped_acquire gil;
    const auto lib = pybind11::module_::import("trl_amd._lib");
    const auto cls = lib.attr(status < 0 ? "TrlkArgumentError" : "TrlkError");
    PyErr_SetString(cls.ptr(), what.c_str());
    throw pybind11::error_already_set();
}

int dtype_code(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return TRLK_F32;
        case at::kBFloat16: return TRLK_BF16;
        case at::kHalf: return TRLK_F16;
        default:
            TORCH_CHECK_TYPE(false, "trl_amd kernels take float32, bfloat16 or float16 logits, got ", t.scalar_type());
    }
}

trlk_stream_t stream_of(const Tensor& t) {
    return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}
Tensor f32(const Tensor& like, at::IntArrayRef sizes) { return at::empty(sizes, like.options().dtype(at::kFloat)); }
// fp32 and contiguous
Tensor f32c(const Tensor& t) { return t.contiguous().to(at::kFloat); }
optional<Tensor> f32c(const optional<Tensor>& t) { return t ? optional<Tensor>(f32c(*t)) : std::nullopt; }
// The data of an operand.  A call is dispatched here if ANY of its tensors is on a GPU: one in ordinary host memory among them
// is an error and must not reach a kernel (pinned memory can be read).
const void* operand(const Tensor& t) {
    TORCH_CHECK(t.is_cuda() || t.numel() == 0 || t.is_pinned(),
                "Expected all tensors to be on the same device, but found one of shape ", t.sizes(), " on ", t.device());
    return t.const_data_ptr();
}
const float* fptr(const Tensor& t) { return static_cast<const float*>(operand(t)); }
const float* fptr(const optional<Tensor>& t) { return t ? fptr(*t) : nullptr; }
float* out(const Tensor& t) { return static_cast<float*>(t.mutable_data_ptr()); }
const int64_t* iptr(const Tensor& t) { return static_cast<const int64_t*>(operand(t)); }

// The int32 word per device that the kernels OR error bits into.  It lives until the process ends.
struct ErrorFlags {
    std::mutex mutex;
    std::map<int64_t, Tensor> of_device;
};
ErrorFlags& error_flags() {
    static auto* flags = new ErrorFlags;  // (never destroyed: the runtime may be gone by then)
    return *flags;
}
Tensor error_flag(int64_t index) {
    ErrorFlags& flags = error_flags();
    std::lock_guard<std::mutex> lock(flags.mutex);
    auto it = flags.of_device.find(index);
    if (it == flags.of_device.end()) {
        const c10::InferenceMode off(false);  // (a word made in inference mode could not be cleared outside of it)
        it = flags.of_device.emplace(index, at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, index))).first;
    }
    return it->second;
}
std::vector<Tensor> all_error_flags() {
    ErrorFlags& flags = error_flags();
    std::lock_guard<std::mutex> lock(flags.mutex);
    std::vector<Tensor> all;
    for (const auto& f : flags.of_device) all.push_back(f.second);
    return all;
}
int32_t* error_word(const Tensor& t) { return static_cast<int32_t*>(error_flag(t.device().index()).mutable_data_ptr()); }

// With TRL_AMD_SYNC_CHECKS=1 the error words are looked at behind each launch that reads token ids (a synchronisation).
const bool kSyncChecks = [] {
    const char* value = std::getenv("TRL_AMD_SYNC_CHECKS");
    return value != nullptr && std::string(value) == "1";
}();
void check_ids() {
    if (!kSyncChecks) return;
    pybind11::gil_scoped_acquire gil;
    pybind11::module_::import("trl_amd.ops").attr("check_device_errors")();
}

void check_logits3d(const Tensor& logits) {
    TORCH_CHECK_VALUE(logits.dim() == 3, "expected [n_seq, rows, vocab] logits, got shape ", logits.sizes());
    TORCH_CHECK_VALUE(logits.size(2) <= 1 || logits.stride(2) == 1, "the vocabulary axis of the logits must be contiguous");
    (void)operand(logits);
}
// the rows from keep_start on of every sequence
const char* window(const Tensor& logits, int64_t keep_start) {
    return static_cast<const char*>(logits.const_data_ptr()) + keep_start * logits.stride(1) * logits.element_size();
}
void check_window(const Tensor& logits, int64_t keep_start, int64_t keep_len) {
    TORCH_CHECK_VALUE(keep_start >= 0 && keep_len >= 0 && keep_start + keep_len <= logits.size(1), "rows ", keep_start, " to ",
                      keep_start + keep_len, " of ", logits.size(1));
}

// ---- log-probs and entropies ----------------------------------------------------------------------------------------
typedef std::tuple<Tensor, Tensor, Tensor> Tensor3;
typedef std::tuple<Tensor, Tensor, Tensor, Tensor> Tensor4;

Tensor4 run_logp_entropy(const Tensor& logits, const Tensor& index_, double temperature, int64_t keep_start, int64_t keep_len,
                         const optional<Tensor>& row_mask, bool with_stats, bool sum_p2) {
    check_logits3d(logits);
    const int64_t n_seq = logits.size(0), vocab = logits.size(2), rows = n_seq * keep_len, k = index_.size(-1);
    const c10::DeviceGuard guard(logits.device());
    Tensor logp = f32(logits, {rows, k}), ent = f32(logits, {rows}), lse = f32(logits, {rows}), stats;
    if (with_stats) stats = f32(logits, {rows, 4});
    if (rows == 0) return {logp, ent, lse, stats};
    check_window(logits, keep_start, keep_len);
    const Tensor index = index_.contiguous();
    check(trlk_logp_entropy_fwd(window(logits, keep_start), dtype_code(logits), n_seq, keep_len, vocab, logits.stride(0),
                                logits.stride(1), iptr(index), k, float(temperature),
                                row_mask ? static_cast<const uint8_t*>(operand(*row_mask)) : nullptr, out(logp), out(ent),
                                out(lse), with_stats ? out(stats) : nullptr, sum_p2 ? 1 : 0, error_word(logits),
                                stream_of(logits)));
    check_ids();
    return {logp, ent, lse, stats};
}
Tensor3 logp_entropy_fwd(const Tensor& logits, const Tensor& index, double temperature, int64_t keep_start, int64_t keep_len,
                         const optional<Tensor>& row_mask) {
    auto [logp, ent, lse, stats] = run_logp_entropy(logits, index, temperature, keep_start, keep_len, row_mask, false, true);
    return {logp, ent, lse};
}
Tensor4 logp_entropy_stats_fwd(const Tensor& logits, const Tensor& index, double temperature, int64_t keep_start,
                               int64_t keep_len, const optional<Tensor>& row_mask, bool sum_p2) {
    return run_logp_entropy(logits, index, temperature, keep_start, keep_len, row_mask, true, sum_p2);
}

Tensor logp_entropy_bwd(const Tensor& logits, const Tensor& index_, double temperature, int64_t keep_start, int64_t keep_len,
                        const Tensor& lse, const optional<Tensor>& entropy, const optional<Tensor>& g_logp_,
                        const optional<Tensor>& g_entropy_) {
    check_logits3d(logits);
    const int64_t n_seq = logits.size(0), length = logits.size(1), vocab = logits.size(2);
    const c10::DeviceGuard guard(logits.device());
    const Tensor dlogits = at::empty({n_seq, length, vocab}, logits.options());
    if (dlogits.numel() == 0) return dlogits;
    check_window(logits, keep_start, keep_len);
    const int64_t k = g_logp_ ? index_.size(-1) : 0;
    const Tensor index = index_.contiguous();
    const optional<Tensor> g_logp = f32c(g_logp_), g_entropy = f32c(g_entropy_);
    check(trlk_logp_entropy_bwd(window(logits, keep_start), dtype_code(logits), n_seq, keep_len, vocab, logits.stride(0),
                                logits.stride(1), iptr(index), k, float(temperature), fptr(lse),
                                g_entropy ? fptr(entropy) : nullptr, fptr(g_logp), fptr(g_entropy), dlogits.mutable_data_ptr(),
                                length, keep_start, dlogits.stride(0), dlogits.stride(1), stream_of(logits)));
    return dlogits;
}

// (the row window may be symbolic while a program is traced, so everything above the device kernels takes c10::SymInt)
typedef Tensor3 LogpEntropySig(const Tensor&, const Tensor&, double, c10::SymInt, c10::SymInt, const optional<Tensor>&);
typedef Tensor4 LogpEntropyStatsSig(const Tensor&, const Tensor&, double, c10::SymInt, c10::SymInt, const optional<Tensor>&, bool);
typedef Tensor LogpEntropyBwdSig(const Tensor&, const Tensor&, double, c10::SymInt, c10::SymInt, const Tensor&,
                                 const optional<Tensor>&, const optional<Tensor>&, const optional<Tensor>&);
template <typename Signature>
c10::TypedOperatorHandle<Signature> handle(const char* name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}
// Whether a derivative of the call is wanted.  A tangent (forward mode, which needs neither grad mode nor a tensor that requires a gradient)
// counts: the autograd functions have no formula for it and raise, where the plain call would return outputs without one.
bool needs_grad(std::initializer_list<const Tensor*> tensors) {
    const bool forward_mode = c10::AutogradState::get_tls_state().get_fw_grad_mode();
    for (const Tensor* t : tensors)
        if (t->defined() && ((c10::GradMode::is_enabled() && t->requires_grad()) || (forward_mode && t->_fw_grad(0).defined()))) return true;
    return false;
}
bool needs_grad(const optional<Tensor>& t) { return t && needs_grad({&*t}); }

// The gradient of the log-prob operators: the backward kernel recomputes the softmax from the saved per-row logsumexp.
class LogpEntropy : public torch::autograd::Function<LogpEntropy> {
  public:
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& index, double temperature,
                                 c10::SymInt keep_start, c10::SymInt keep_len, const optional<Tensor>& row_mask, bool with_stats,
                                 bool sum_p2) {
        variable_list result;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            if (with_stats) {
                static const auto op = handle<LogpEntropyStatsSig>("trl_amd::logp_entropy_stats_fwd");
                auto [logp, ent, lse, stats] = op.call(logits, index, temperature, keep_start, keep_len, row_mask, sum_p2);
                result = {logp, ent, lse, stats};
            } else {
                static const auto op = handle<LogpEntropySig>("trl_amd::logp_entropy_fwd");
                auto [logp, ent, lse] = op.call(logits, index, temperature, keep_start, keep_len, row_mask);
                result = {logp, ent, lse};
            }
        }
        ctx->save_for_backward({logits, index, result[2], result[1]});
        ctx->saved_data["temperature"] = temperature;
        ctx->saved_data["keep_start"] = keep_start;
        ctx->saved_data["keep_len"] = keep_len;
        ctx->set_materialize_grads(false);
        return result;
    }
    // (the lse output only exists to be saved for this backward; a gradient arriving there is ignored)
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        variable_list result(8);
        Tensor g_logp = grads[0];
        const Tensor& g_ent = grads[1];
        if (!g_logp.defined() && !g_ent.defined()) return result;
        const auto saved = ctx->get_saved_variables();
        const Tensor &logits = saved[0], &index = saved[1];
        if (!g_logp.defined() && index.sym_size(-1) > 0)
            g_logp = at::zeros_symint(index.sym_sizes(), logits.options().dtype(at::kFloat));
        static const auto op = handle<LogpEntropyBwdSig>("trl_amd::logp_entropy_bwd");
        result[0] = op.call(logits, index, ctx->saved_data["temperature"].toDouble(), ctx->saved_data["keep_start"].toSymInt(),
                            ctx->saved_data["keep_len"].toSymInt(), saved[2], saved[3],
                            g_logp.defined() ? optional<Tensor>(g_logp) : std::nullopt,
                            g_ent.defined() ? optional<Tensor>(g_ent) : std::nullopt);
        return result;
    }
};
Tensor3 logp_entropy_fwd_autograd(const Tensor& logits, const Tensor& index, double temperature, c10::SymInt keep_start,
                                  c10::SymInt keep_len, const optional<Tensor>& row_mask) {
    if (needs_grad({&logits})) {
        const auto r = LogpEntropy::apply(logits, index, temperature, keep_start, keep_len, row_mask, false, true);
        return {r[0], r[1], r[2]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<LogpEntropySig>("trl_amd::logp_entropy_fwd");
    return op.call(logits, index, temperature, keep_start, keep_len, row_mask);
}
Tensor4 logp_entropy_stats_fwd_autograd(const Tensor& logits, const Tensor& index, double temperature, c10::SymInt keep_start,
                                        c10::SymInt keep_len, const optional<Tensor>& row_mask, bool sum_p2) {
    if (needs_grad({&logits})) {
        const auto r = LogpEntropy::apply(logits, index, temperature, keep_start, keep_len, row_mask, true, sum_p2);
        return {r[0], r[1], r[2], r[3]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<LogpEntropyStatsSig>("trl_amd::logp_entropy_stats_fwd");
    return op.call(logits, index, temperature, keep_start, keep_len, row_mask, sum_p2);
}

// ---- GRPO -----------------------------------------------------------------------------------------------------------
void check_token_shape(const char* op, const char* name, const optional<Tensor>& t, int64_t B, int64_t T) {
    TORCH_CHECK_VALUE(!t || (t->dim() == 2 && t->size(0) == B && t->size(1) == T), op, ": ", name, " has shape ",
                      t ? t->sizes() : at::IntArrayRef(), ", expected (", B, ", ", T, ")");
}
// strides of the advantages along (sequence, token): one per sequence, or one per token
std::pair<int64_t, int64_t> advantage_strides(const char* op, const Tensor& adv, int64_t B, int64_t T) {
    if (adv.dim() == 1 || (adv.dim() == 2 && adv.size(1) == 1)) {
        TORCH_CHECK_VALUE(adv.numel() == B, op, ": advantages must have one entry per sequence");
        return {1, 0};
    }
    TORCH_CHECK_VALUE(adv.dim() == 2 && adv.size(0) == B && adv.size(1) == T, op, ": advantages of shape ", adv.sizes(),
                      " do not match [B]=", B, " or [B,T]");
    return {T, 1};
}

Tensor4 grpo_loss(const Tensor& logp_, const optional<Tensor>& old_, const optional<Tensor>& ref_, const optional<Tensor>& ent_,
                  const Tensor& advantages_, const Tensor& mask_, const optional<Tensor>& weight_,
                  const optional<Tensor>& entropy_mask_, const optional<Tensor>& normalizer_, int64_t loss_type,
                  double epsilon_low, double epsilon_high, double delta, double beta, bool bias_correction_kl,
                  double grad_accum_steps, double dr_grpo_denominator, double num_processes, double entropy_coef,
                  int64_t policy_term, bool sequence_level, const optional<Tensor>& seq_coef_, double sapo_pos, double sapo_neg) {
    TORCH_CHECK_VALUE(logp_.dim() == 2, "grpo_loss: per-token log-probs must be [B, T]");
    const int64_t B = logp_.size(0), T = logp_.size(1);
    const c10::DeviceGuard guard(logp_.device());
    const Tensor logp = f32c(logp_), mask = f32c(mask_), advantages = f32c(advantages_);
    const optional<Tensor> old = f32c(old_), ref = f32c(ref_), ent = f32c(ent_), weight = f32c(weight_),
                           entropy_mask = f32c(entropy_mask_);
    const auto [sb, st] = advantage_strides("grpo_loss", advantages, B, T);
    check_token_shape("grpo_loss", "old_logp", old, B, T);
    check_token_shape("grpo_loss", "ref_logp", ref, B, T);
    check_token_shape("grpo_loss", "entropy", ent, B, T);
    check_token_shape("grpo_loss", "mask", mask, B, T);
    check_token_shape("grpo_loss", "token_weight", weight, B, T);
    check_token_shape("grpo_loss", "entropy_mask", entropy_mask, B, T);
    const optional<Tensor> normalizer = normalizer_ ? f32c(optional<Tensor>(normalizer_->reshape({1}))) : std::nullopt;
    TORCH_CHECK_VALUE(!seq_coef_ || seq_coef_->numel() == B, "grpo_loss: seq_coef must have one entry per sequence");
    const optional<Tensor> seq_coef = seq_coef_ ? f32c(optional<Tensor>(seq_coef_->reshape({B}))) : std::nullopt;
    const Tensor loss = f32(logp, {}), metrics = f32(logp, {TRLK_GRPO_NUM_METRICS}), dlogp = f32(logp, {B, T}),
                 dent = entropy_coef != 0.0 ? f32(logp, {B, T}) : f32(logp, {0});
    const size_t ws_bytes = trlk_grpo_workspace_bytes(B);
    const Tensor ws = at::empty({int64_t(ws_bytes)}, logp.options().dtype(at::kByte));
    check(trlk_grpo_loss(fptr(logp), fptr(old), fptr(ref), fptr(ent), fptr(advantages), sb, st, fptr(mask), fptr(weight),
                         fptr(entropy_mask), fptr(seq_coef), B, T, int(loss_type), int(policy_term), sequence_level ? 1 : 0,
                         float(epsilon_low), float(epsilon_high), float(delta), float(beta), bias_correction_kl ? 1 : 0,
                         float(grad_accum_steps), float(dr_grpo_denominator), fptr(normalizer), float(num_processes),
                         float(entropy_coef), float(sapo_pos), float(sapo_neg), out(loss), out(metrics), out(dlogp),
                         entropy_coef != 0.0 ? out(dent) : nullptr, ws.mutable_data_ptr(), ws_bytes, stream_of(logp)));
    return {loss, metrics, dlogp, dent};
}

class GrpoLoss : public torch::autograd::Function<GrpoLoss> {
  public:
    static variable_list forward(AutogradContext* ctx, const Tensor& logp, const optional<Tensor>& old, const optional<Tensor>& ref,
                                 const optional<Tensor>& ent, const Tensor& advantages, const Tensor& mask,
                                 const optional<Tensor>& weight, const optional<Tensor>& entropy_mask,
                                 const optional<Tensor>& normalizer, int64_t loss_type, double epsilon_low, double epsilon_high,
                                 double delta, double beta, bool bias_correction_kl, double grad_accum_steps,
                                 double dr_grpo_denominator, double num_processes, double entropy_coef, int64_t policy_term,
                                 bool sequence_level, const optional<Tensor>& seq_coef, double sapo_pos, double sapo_neg) {
        variable_list result;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            static const auto op = handle<decltype(grpo_loss)>("trl_amd::grpo_loss");
            auto [loss, metrics, dlogp, dent] =
                op.call(logp, old, ref, ent, advantages, mask, weight, entropy_mask, normalizer, loss_type, epsilon_low,
                        epsilon_high, delta, beta, bias_correction_kl, grad_accum_steps, dr_grpo_denominator, num_processes,
                        entropy_coef, policy_term, sequence_level, seq_coef, sapo_pos, sapo_neg);
            result = {loss, metrics, dlogp, dent};
        }
        ctx->save_for_backward({result[2], result[3]});
        ctx->saved_data["dtype"] = logp.scalar_type();
        ctx->saved_data["entropy"] = entropy_coef != 0.0 && ent.has_value();
        ctx->set_materialize_grads(false);
        return result;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        variable_list result(24);
        if (!grads[0].defined()) return result;
        const auto saved = ctx->get_saved_variables();
        result[0] = (grads[0] * saved[0]).to(ctx->saved_data["dtype"].toScalarType());
        if (ctx->saved_data["entropy"].toBool()) result[3] = grads[0] * saved[1];
        return result;
    }
};
Tensor4 grpo_loss_autograd(const Tensor& logp, const optional<Tensor>& old, const optional<Tensor>& ref, const optional<Tensor>& ent,
                           const Tensor& advantages, const Tensor& mask, const optional<Tensor>& weight,
                           const optional<Tensor>& entropy_mask, const optional<Tensor>& normalizer, int64_t loss_type,
                           double epsilon_low, double epsilon_high, double delta, double beta, bool bias_correction_kl,
                           double grad_accum_steps, double dr_grpo_denominator, double num_processes, double entropy_coef,
                           int64_t policy_term, bool sequence_level, const optional<Tensor>& seq_coef, double sapo_pos,
                           double sapo_neg) {
    const bool grad = needs_grad({&logp, &advantages, &mask}) || needs_grad(old) || needs_grad(ref) || needs_grad(ent) ||
                      needs_grad(weight) || needs_grad(entropy_mask) || needs_grad(normalizer) || needs_grad(seq_coef);
    if (grad) {
        const auto r = GrpoLoss::apply(logp, old, ref, ent, advantages, mask, weight, entropy_mask, normalizer, loss_type,
                                       epsilon_low, epsilon_high, delta, beta, bias_correction_kl, grad_accum_steps,
                                       dr_grpo_denominator, num_processes, entropy_coef, policy_term, sequence_level, seq_coef,
                                       sapo_pos, sapo_neg);
        return {r[0], r[1], r[2], r[3]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(grpo_loss)>("trl_amd::grpo_loss");
    return op.call(logp, old, ref, ent, advantages, mask, weight, entropy_mask, normalizer, loss_type, epsilon_low, epsilon_high,
                   delta, beta, bias_correction_kl, grad_accum_steps, dr_grpo_denominator, num_processes, entropy_coef,
                   policy_term, sequence_level, seq_coef, sapo_pos, sapo_neg);
}

Tensor4 grpo_fused(const Tensor& logits, const Tensor& index_, double temperature, int64_t keep_start, int64_t keep_len,
                   const Tensor& mask_, const Tensor& advantages_, const Tensor& row_scale_, const optional<Tensor>& old_,
                   const optional<Tensor>& ref_, const optional<Tensor>& weight_, const optional<Tensor>& seq_coef_,
                   int64_t policy_term, double epsilon_low, double epsilon_high, double delta, double beta,
                   bool bias_correction_kl, double sapo_pos, double sapo_neg, bool compute_masked_rows,
                   const optional<Tensor>& entropy_weight_) {
    check_logits3d(logits);
    const int64_t n_seq = logits.size(0), length = logits.size(1), vocab = logits.size(2);
    for (const Tensor* t : {&index_, &mask_})
        TORCH_CHECK_VALUE(t->dim() == 2 && t->size(0) == n_seq && t->size(1) == keep_len, "grpo_fused: index and mask must be [",
                          n_seq, ", ", keep_len, "]");
    const c10::DeviceGuard guard(logits.device());
    const Tensor index = index_.contiguous().to(at::kLong), mask = f32c(mask_), advantages = f32c(advantages_);
    const optional<Tensor> old = f32c(old_), ref = f32c(ref_), weight = f32c(weight_), entropy_weight = f32c(entropy_weight_);
    check_token_shape("grpo_fused", "old_logp", old, n_seq, keep_len);
    check_token_shape("grpo_fused", "ref_logp", ref, n_seq, keep_len);
    check_token_shape("grpo_fused", "token_weight", weight, n_seq, keep_len);
    check_token_shape("grpo_fused", "entropy_weight", entropy_weight, n_seq, keep_len);
    const auto [sb, st] = advantage_strides("grpo_fused", advantages, n_seq, keep_len);
    const Tensor row_scale = f32c(row_scale_.reshape({n_seq}));
    const optional<Tensor> seq_coef = seq_coef_ ? f32c(optional<Tensor>(seq_coef_->reshape({n_seq}))) : std::nullopt;
    const Tensor logp = f32(logits, {n_seq, keep_len}), ent = f32(logits, {n_seq, keep_len}),
                 lse = f32(logits, {n_seq, keep_len}), dlogits = at::empty({n_seq, length, vocab}, logits.options());
    if (dlogits.numel() == 0) return {logp, ent, lse, dlogits};
    check_window(logits, keep_start, keep_len);
    check(trlk_grpo_fused_fwd_bwd(
        window(logits, keep_start), dtype_code(logits), n_seq, keep_len, vocab, logits.stride(0), logits.stride(1), iptr(index),
        float(temperature), fptr(old), fptr(ref), fptr(advantages), sb, st, fptr(mask), fptr(weight), fptr(seq_coef),
        fptr(row_scale), fptr(entropy_weight), int(policy_term), float(epsilon_low), float(epsilon_high), float(delta),
        float(beta), bias_correction_kl ? 1 : 0, float(sapo_pos), float(sapo_neg), out(logp), out(ent), out(lse),
        dlogits.mutable_data_ptr(), length, keep_start, dlogits.stride(0), dlogits.stride(1), compute_masked_rows ? 1 : 0,
        error_word(logits), stream_of(logits)));
    check_ids();
    return {logp, ent, lse, dlogits};
}

void scale_unless_one_(const Tensor& data, const Tensor& scale_) {
    TORCH_CHECK_VALUE(data.is_contiguous() && (data.scalar_type() == at::kBFloat16 || data.scalar_type() == at::kHalf ||
                                               data.scalar_type() == at::kFloat),
                      "scale_unless_one_: contiguous bf16 / fp16 / fp32 data expected");
    const c10::DeviceGuard guard(data.device());
    const Tensor scale = scale_.reshape({1}).to(data.options().dtype(at::kFloat));
    (void)operand(data);
    check(trlk_scale_unless_one(data.mutable_data_ptr(), dtype_code(data), data.numel(), fptr(scale), stream_of(data)));
}

// The loss of a pass that has written its gradient already.  Backward hands `dlogits` on as d loss / d logits, times what is left
// of the upstream gradient behind the factor `upstream` that the pass has applied: 1 as a rule, and then nothing is touched.
// A node of C++ and not of Python: the host takes longer than the device over a step of a small batch, and the device is idle
// from the metrics' copy to the next step's first launch, where this backward lies.  GRPO step, Python node -> this one, in us:
// bf16 [4, 256, 32000] 178-181 -> 137-154, [16, 509, 50257] 401-405 -> 365-380, [32, 1024, 151936] 2872 -> 2850.
class GradientInHand : public torch::autograd::Function<GradientInHand> {
  public:
    static Tensor forward(AutogradContext* ctx, const Tensor& loss, const Tensor& logits, const Tensor& dlogits,
                          const optional<Tensor>& upstream) {
        ctx->save_for_backward({dlogits, upstream ? *upstream : Tensor()});
        ctx->saved_data["consumed"] = false;
        ctx->set_materialize_grads(false);
        return loss.variable_data();  // (a tensor of its own on the same number, not a view: it may be changed in place)
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        const auto saved = ctx->get_saved_variables();
        variable_list result(4);
        if (!grads[0].defined()) return result;
        // the gradient buffer is scaled in place and handed on: a second pass would scale it again
        TORCH_CHECK(!ctx->saved_data["consumed"].toBool(),
                    "grpo_loss_from_logits: its backward can run only once (the gradient written by the forward pass is handed to "
                    "the graph in place); call the function again instead of retain_graph=True");
        ctx->saved_data["consumed"] = true;
        {
            // in place: the buffer belongs to this node and is handed on once (the kernel returns at once for a scale of 1)
            const at::NoGradGuard no_grad;
            static const auto op = handle<decltype(scale_unless_one_)>("trl_amd::scale_unless_one_");
            op.call(saved[0], saved[1].defined() ? grads[0].to(at::kFloat) / saved[1] : grads[0]);
        }
        result[1] = saved[0];
        if (c10::GradMode::is_enabled() && grads[0].requires_grad()) {  // its own gradient is refused, not dropped
            const auto refuse = std::make_shared<torch::autograd::DelayedError>(
                "trying to differentiate twice: the gradient of grpo_loss_from_logits has no gradient of its own", 1);
            result[1] = (*refuse)({saved[0].detach().requires_grad_(true)})[0];
        }
        return result;
    }
};
Tensor gradient_in_hand(const Tensor& loss, const Tensor& logits, const Tensor& dlogits, const optional<Tensor>& upstream) {
    return GradientInHand::apply(loss, logits, dlogits, upstream);
}

Tensor grpo_log_values(const Tensor& metrics) {
    const c10::DeviceGuard guard(metrics.device());
    const Tensor values = f32(metrics, {TRLK_GRPO_LOG_VALUES});
    check(trlk_grpo_log_values(fptr(metrics), error_word(metrics), out(values), stream_of(metrics)));
    return values;
}

std::tuple<Tensor, Tensor> grpo_row_scale(const Tensor& mask, int64_t loss_type, double numerator, const optional<Tensor>& n_items,
                                          const optional<Tensor>& upstream, bool with_mask) {
    const int64_t B = mask.size(0), T = mask.size(1);
    for (const auto* t : {&n_items, &upstream})
        TORCH_CHECK_VALUE(!*t || (*t)->device() == mask.device(), "grpo_row_scale: the mask and the scalars must be on one GPU");
    int type = 0;
    switch (mask.scalar_type()) {
        case at::kBool:
        case at::kByte: type = 0; break;
        case at::kInt: type = 1; break;
        case at::kLong: type = 2; break;
        case at::kFloat: type = 3; break;
        default: TORCH_CHECK_TYPE(false, "grpo_row_scale: masks are bool, uint8, int32, int64 or float32");
    }
    const c10::DeviceGuard guard(mask.device());
    const Tensor mask_f = with_mask ? f32(mask, {B, T}) : f32(mask, {0}), scale = f32(mask, {B});
    check(trlk_grpo_row_scale(operand(mask), type, B, T, mask.stride(0), mask.stride(1), int(loss_type), float(numerator),
                              fptr(n_items), fptr(upstream), with_mask ? out(mask_f) : nullptr, out(scale), stream_of(mask)));
    return {mask_f, scale};
}

// ---- DPO ------------------------------------------------------------------------------------------------------------
Tensor4 dpo_loss(const Tensor& logp_, const Tensor& mask_, const Tensor& ref_chosen_, const Tensor& ref_rejected_, double beta) {
    TORCH_CHECK_VALUE(logp_.dim() == 2, "dpo_loss: per-token log-probs must be [B, T]");
    const int64_t B = logp_.size(0), T = logp_.size(1);
    TORCH_CHECK_VALUE(B % 2 == 0 && B >= 2, "dpo_loss: the batch must be [chosen; rejected], i.e. an even number of sequences");
    const c10::DeviceGuard guard(logp_.device());
    const Tensor logp = f32c(logp_), mask = f32c(mask_), ref_chosen = f32c(ref_chosen_), ref_rejected = f32c(ref_rejected_);
    TORCH_CHECK_VALUE(mask.dim() == 2 && mask.size(0) == B && mask.size(1) == T && ref_chosen.numel() == B / 2 &&
                          ref_rejected.numel() == B / 2,
                      "dpo_loss: mask must be [B, T] and the reference log-probs [B/2] each");
    const Tensor loss = f32(logp, {}), seq = f32(logp, {B}), metrics = f32(logp, {TRLK_DPO_NUM_METRICS}), dlogp = f32(logp, {B, T});
    check(trlk_dpo_loss(fptr(logp), fptr(mask), fptr(ref_chosen), fptr(ref_rejected), B, T, float(beta), out(seq), out(loss),
                        out(metrics), out(dlogp), stream_of(logp)));
    return {loss, seq, metrics, dlogp};
}
class DpoLoss : public torch::autograd::Function<DpoLoss> {
  public:
    static variable_list forward(AutogradContext* ctx, const Tensor& logp, const Tensor& mask, const Tensor& ref_chosen,
                                 const Tensor& ref_rejected, double beta) {
        variable_list result;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            static const auto op = handle<decltype(dpo_loss)>("trl_amd::dpo_loss");
            auto [loss, seq, metrics, dlogp] = op.call(logp, mask, ref_chosen, ref_rejected, beta);
            result = {loss, seq, metrics, dlogp};
        }
        ctx->save_for_backward({result[3], mask});
        ctx->saved_data["dtype"] = logp.scalar_type();
        ctx->set_materialize_grads(false);
        return result;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        variable_list result(5);
        const auto saved = ctx->get_saved_variables();
        Tensor g;
        if (grads[0].defined()) g = grads[0] * saved[0];
        if (grads[1].defined()) {
            const Tensor extra = grads[1].unsqueeze(1) * saved[1].ne(0).to(at::kFloat);
            g = g.defined() ? g + extra : extra;
        }
        if (g.defined()) result[0] = g.to(ctx->saved_data["dtype"].toScalarType());
        return result;
    }
};
Tensor4 dpo_loss_autograd(const Tensor& logp, const Tensor& mask, const Tensor& ref_chosen, const Tensor& ref_rejected, double beta) {
    if (needs_grad({&logp, &mask, &ref_chosen, &ref_rejected})) {
        const auto r = DpoLoss::apply(logp, mask, ref_chosen, ref_rejected, beta);
        return {r[0], r[1], r[2], r[3]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(dpo_loss)>("trl_amd::dpo_loss");
    return op.call(logp, mask, ref_chosen, ref_rejected, beta);
}

Tensor dpo_log_values(const Tensor& entropy_, const Tensor& row_stats_, const Tensor& mask_, const Tensor& seq_logps_,
                      const Tensor& ref_chosen_, const Tensor& ref_rejected_, double beta) {
    const int64_t B = mask_.size(0), T = mask_.size(1), P = B / 2;
    TORCH_CHECK_VALUE(B % 2 == 0 && entropy_.numel() == B * T && row_stats_.numel() == 4 * B * T && seq_logps_.numel() == B,
                      "dpo_log_values: the shapes do not match");
    (void)operand(mask_);
    const c10::DeviceGuard guard(mask_.device());
    const Tensor entropy = f32c(entropy_), row_stats = f32c(row_stats_), mask = f32c(mask_), seq_logps = f32c(seq_logps_);
    const Tensor ref_chosen = f32c(ref_chosen_.expand({P})), ref_rejected = f32c(ref_rejected_.expand({P}));
    const Tensor values = f32(mask, {8 + 2 * B});
    if (B == 0) return values.zero_();
    const Tensor ws = f32(mask, {4 * B});
    check(trlk_dpo_log_values(fptr(entropy), fptr(row_stats), fptr(mask), B, T, fptr(seq_logps), fptr(ref_chosen),
                              fptr(ref_rejected), float(beta), error_word(mask), out(values), out(ws), stream_of(mask)));
    return values;
}

// ---- tokens drawn from, and scored under, a filtered distribution ------------------------------------------------------
// an operand is where the logits are
void beside(const char* op, const Tensor& logits, const Tensor& t) {
    TORCH_CHECK(t.device() == logits.device(), op, ": an operand is on ", t.device(), ", the logits are on ", logits.device());
}
// The sampling settings: a number for all rows, or a tensor with a value for each.
struct Settings {
    double temperature, top_p, min_p;
    int64_t top_k;
    optional<Tensor> temperatures, top_ks, top_ps, min_ps;
    const float* t() const { return fptr(temperatures); }
    const float* p() const { return fptr(top_ps); }
    const float* m() const { return fptr(min_ps); }
    const int32_t* k() const { return top_ks ? static_cast<const int32_t*>(operand(*top_ks)) : nullptr; }
};
// int32, and what lies beyond it (all tokens, or no filter) at its ends
Tensor int32_values(const Tensor& t) {
    constexpr int64_t most = std::numeric_limits<int32_t>::max();
    return t.scalar_type() == at::kInt ? t.contiguous() : t.to(at::kLong).clamp(-most, most).to(at::kInt).contiguous();
}
Settings settings(const char* op, const Tensor& logits, int64_t rows, double temperature, int64_t top_k, double top_p, double min_p,
                  const optional<Tensor>& temperatures, const optional<Tensor>& top_ks, const optional<Tensor>& top_ps,
                  const optional<Tensor>& min_ps) {
    for (const optional<Tensor>* t : {&temperatures, &top_ks, &top_ps, &min_ps}) {
        if (!*t) continue;
        TORCH_CHECK_VALUE((*t)->numel() == rows, op, ": a setting has ", (*t)->numel(), " values for ", rows, " rows");
        beside(op, logits, **t);
    }
    return {temperature, top_p, min_p, top_k, f32c(temperatures), top_ks ? optional<Tensor>(int32_values(*top_ks)) : std::nullopt, f32c(top_ps),
            f32c(min_ps)};
}
// Logits [..., V] as rows [n_seq, rows_per_seq] with strides: where they lie if the strides say so, else a copy.
struct Rows {
    Tensor x;  // as in memory, or the copy
    int64_t n_seq = 1, length = 1, vocab, seq_stride = 0, row_stride = 0, count;
    int dtype;
    explicit Rows(const Tensor& logits) : x(logits) {
        TORCH_CHECK_VALUE(x.dim() > 0, "logits must have at least one dimension");
        (void)operand(x);
        dtype = dtype_code(x);
        vocab = x.size(-1);
        if (x.dim() > 3) {  // (the product by itself: without rows in the last but one dimension a reshape could not tell it)
            int64_t leading = 1;
            for (int64_t i = 0; i < x.dim() - 2; ++i) leading *= x.size(i);
            x = x.reshape({leading, x.size(-2), vocab});
        }
        if ((vocab > 1 && x.stride(-1) != 1) || (x.dim() > 1 && x.size(-2) > 1 && x.stride(-2) < vocab)) x = x.contiguous();
        if (x.dim() > 1) length = x.size(-2), row_stride = x.stride(-2);
        if (x.dim() > 2) n_seq = x.size(0), seq_stride = x.stride(0);
        count = n_seq * length;
    }
    const void* data() const { return x.const_data_ptr(); }
};
// one byte for each row
optional<Tensor> byte_mask(const char* op, const Tensor& logits, const optional<Tensor>& mask, int64_t rows) {
    if (!mask) return std::nullopt;
    beside(op, logits, *mask);
    TORCH_CHECK_VALUE(mask->numel() == rows, op, ": the row mask has ", mask->numel(), " entries for ", rows, " rows");
    return mask->scalar_type() == at::kBool ? mask->contiguous() : mask->ne(0).contiguous();
}
const uint8_t* mask_ptr(const optional<Tensor>& mask) { return mask ? static_cast<const uint8_t*>(operand(*mask)) : nullptr; }
Tensor bytes(const Tensor& like, size_t n) { return at::empty({int64_t(n)}, like.options().dtype(at::kByte)); }

std::tuple<Tensor, Tensor> sample_tokens(const Tensor& logits, const Tensor& uniforms_, double temperature, int64_t top_k, double top_p,
                                         double min_p, const optional<Tensor>& temperatures, const optional<Tensor>& top_ks,
                                         const optional<Tensor>& top_ps, const optional<Tensor>& min_ps,
                                         const optional<Tensor>& row_mask, int64_t fill_id) {
    const c10::DeviceGuard guard(logits.device());
    const Rows r(logits);
    TORCH_CHECK_VALUE(uniforms_.numel() == r.count, "sample_tokens: ", uniforms_.numel(), " uniform numbers for ", r.count, " rows");
    beside("sample_tokens", logits, uniforms_);
    const Tensor ids = at::empty(uniforms_.sizes(), logits.options().dtype(at::kLong)), logp = f32(logits, uniforms_.sizes());
    const Settings s = settings("sample_tokens", logits, r.count, temperature, top_k, top_p, min_p, temperatures, top_ks, top_ps, min_ps);
    const optional<Tensor> mask = byte_mask("sample_tokens", logits, row_mask, r.count);
    const bool f64 = uniforms_.scalar_type() == at::kDouble;
    const Tensor uniforms = f64 ? uniforms_.contiguous() : f32c(uniforms_);
    const size_t ws_bytes = trlk_token_filter_workspace_bytes(r.count, r.vocab, r.dtype);
    const Tensor ws = bytes(logits, ws_bytes);
    check(trlk_sample_tokens(r.data(), r.dtype, r.n_seq, r.length, r.vocab, r.seq_stride, r.row_stride, operand(uniforms), f64 ? 1 : 0,
                             s.temperature, s.t(), s.top_k, s.k(), s.top_p, s.p(), s.min_p, s.m(), mask_ptr(mask), fill_id,
                             static_cast<int64_t*>(ids.mutable_data_ptr()), out(logp), error_word(logits), ws.mutable_data_ptr(), ws_bytes,
                             stream_of(logits)));
    check_ids();
    return {ids, logp};
}

Tensor3 filtered_logps_fwd(const Tensor& logits, const Tensor& index_, double temperature, int64_t top_k, double top_p, double min_p,
                           const optional<Tensor>& temperatures, const optional<Tensor>& top_ks, const optional<Tensor>& top_ps,
                           const optional<Tensor>& min_ps, const optional<Tensor>& row_mask) {
    const c10::DeviceGuard guard(logits.device());
    const Rows r(logits);
    TORCH_CHECK_VALUE(index_.numel() == r.count && index_.scalar_type() == at::kLong, "filtered_logps: ", index_.numel(), " ",
                      index_.scalar_type(), " token ids for ", r.count, " rows of int64");
    beside("filtered_logps", logits, index_);
    const Settings s = settings("filtered_logps", logits, r.count, temperature, top_k, top_p, min_p, temperatures, top_ks, top_ps, min_ps);
    const optional<Tensor> mask = byte_mask("filtered_logps", logits, row_mask, r.count);
    const bool blocks = trlk_token_filter_has_blocks(s.temperature, s.t(), s.top_k, s.k(), s.top_p, s.p(), s.min_p, s.m()) != 0;
    const Tensor logp = f32(logits, index_.sizes()), state = f32(logits, {r.count, 4});
    const Tensor block_max = at::empty({blocks ? r.count : 0, trlk_token_filter_blocks(r.vocab)}, logits.options());
    const Tensor index = index_.contiguous();
    const size_t ws_bytes = trlk_token_filter_workspace_bytes(r.count, r.vocab, r.dtype);
    const Tensor ws = bytes(logits, ws_bytes);
    check(trlk_filtered_logps_fwd(r.data(), r.dtype, r.n_seq, r.length, r.vocab, r.seq_stride, r.row_stride, iptr(index), s.temperature,
                                  s.t(), s.top_k, s.k(), s.top_p, s.p(), s.min_p, s.m(), mask_ptr(mask), out(logp), out(state),
                                  blocks ? block_max.mutable_data_ptr() : nullptr, error_word(logits), ws.mutable_data_ptr(), ws_bytes,
                                  stream_of(logits)));
    check_ids();
    return {logp, state, block_max};
}

Tensor filtered_logps_bwd(const Tensor& logits, const Tensor& index_, double temperature, const optional<Tensor>& temperatures_,
                          const Tensor& state, const Tensor& block_max, const Tensor& g_logp_) {
    const c10::DeviceGuard guard(logits.device());
    const Tensor dlogits = at::empty(logits.sizes(), logits.options());
    if (dlogits.numel() == 0) return dlogits;
    const Rows r(logits);
    TORCH_CHECK_VALUE(index_.numel() == r.count && g_logp_.numel() == r.count && state.numel() == 4 * r.count && state.is_contiguous() &&
                          (!temperatures_ || temperatures_->numel() == r.count) &&
                          (block_max.numel() == 0 || block_max.numel() == r.count * trlk_token_filter_blocks(r.vocab)),
                      "filtered_logps: the backward's operands do not match");
    const Tensor index = index_.contiguous(), g_logp = f32c(g_logp_);
    const optional<Tensor> temperatures = f32c(temperatures_);
    check(trlk_filtered_logps_bwd(r.data(), r.dtype, r.n_seq, r.length, r.vocab, r.seq_stride, r.row_stride, iptr(index), temperature,
                                  fptr(temperatures), fptr(state), block_max.numel() ? operand(block_max) : nullptr, fptr(g_logp),
                                  dlogits.mutable_data_ptr(), stream_of(logits)));
    return dlogits;
}

class FilteredLogps : public torch::autograd::Function<FilteredLogps> {
  public:
    static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& index, double temperature, int64_t top_k,
                                 double top_p, double min_p, const optional<Tensor>& temperatures, const optional<Tensor>& top_ks,
                                 const optional<Tensor>& top_ps, const optional<Tensor>& min_ps, const optional<Tensor>& row_mask) {
        variable_list result;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            static const auto op = handle<decltype(filtered_logps_fwd)>("trl_amd::filtered_logps_fwd");
            auto [logp, state, block_max] =
                op.call(logits, index, temperature, top_k, top_p, min_p, temperatures, top_ks, top_ps, min_ps, row_mask);
            result = {logp, state, block_max};
        }
        ctx->save_for_backward({logits, index, result[1], result[2], temperatures ? *temperatures : Tensor()});
        ctx->saved_data["temperature"] = temperature;
        ctx->mark_non_differentiable({result[1], result[2]});
        ctx->set_materialize_grads(false);
        return result;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        variable_list result(11);
        if (!grads[0].defined()) return result;
        const auto saved = ctx->get_saved_variables();
        static const auto op = handle<decltype(filtered_logps_bwd)>("trl_amd::filtered_logps_bwd");
        result[0] = op.call(saved[0], saved[1], ctx->saved_data["temperature"].toDouble(),
                            saved[4].defined() ? optional<Tensor>(saved[4]) : std::nullopt, saved[2], saved[3], grads[0]);
        return result;
    }
};
Tensor3 filtered_logps_fwd_autograd(const Tensor& logits, const Tensor& index, double temperature, int64_t top_k, double top_p,
                                    double min_p, const optional<Tensor>& temperatures, const optional<Tensor>& top_ks,
                                    const optional<Tensor>& top_ps, const optional<Tensor>& min_ps, const optional<Tensor>& row_mask) {
    TORCH_CHECK(!needs_grad(temperatures) && !needs_grad(top_ps) && !needs_grad(min_ps),
                "filtered_logps is differentiable with respect to the logits alone: detach the settings");
    if (needs_grad({&logits})) {
        const auto r = FilteredLogps::apply(logits, index, temperature, top_k, top_p, min_p, temperatures, top_ks, top_ps, min_ps, row_mask);
        return {r[0], r[1], r[2]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<decltype(filtered_logps_fwd)>("trl_amd::filtered_logps_fwd");
    return op.call(logits, index, temperature, top_k, top_p, min_p, temperatures, top_ks, top_ps, min_ps, row_mask);
}

// ---- embeddings -------------------------------------------------------------------------------------------------------
// Ids of 32 or 64 bits, contiguous.
Tensor token_ids(const char* op, const Tensor& ids) {
    TORCH_CHECK_TYPE(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, op, ": ids are int64 or int32, not ", ids.scalar_type());
    return ids.contiguous();
}
int id_bits(const Tensor& ids) { return ids.scalar_type() == at::kLong ? 64 : 32; }
// Matrices whose rows are apart but whose entries are not.
Tensor with_rows(const Tensor& t) { return (t.size(1) <= 1 || t.stride(1) == 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)) ? t : t.contiguous(); }

Tensor embedding_fwd(const Tensor& ids_, const Tensor& weight_, double scale) {
    TORCH_CHECK_VALUE(weight_.dim() == 2, "embedding: the table is [tokens, width], got shape ", weight_.sizes());
    TORCH_CHECK(ids_.device() == weight_.device(), "embedding: ids are on ", ids_.device(), ", the table on ", weight_.device());
    const c10::DeviceGuard guard(weight_.device());
    const Tensor ids = token_ids("embedding", ids_), weight = with_rows(weight_);
    std::vector<int64_t> sizes = ids.sizes().vec();
    sizes.push_back(weight.size(1));
    const Tensor rows = at::empty(sizes, weight.options());
    check(trlk_embedding_fwd(weight.const_data_ptr(), dtype_code(weight), weight.size(0), weight.size(1), weight.stride(0), ids.const_data_ptr(),
                             id_bits(ids), ids.numel(), float(scale), rows.mutable_data_ptr(), error_word(weight), stream_of(weight)));
    if (rows.numel()) check_ids();
    return rows;
}

void embedding_into(const Tensor& into, const Tensor& grad_, const Tensor& ids_, double scale, int64_t padding_idx, bool accumulate) {
    TORCH_CHECK_VALUE(grad_.dim() == ids_.dim() + 1 && grad_.sizes().slice(0, ids_.dim()) == ids_.sizes() && grad_.size(-1) == into.size(1),
                      "embedding's gradient: ids of shape ", ids_.sizes(), ", gradients of shape ", grad_.sizes(), ", table of shape ", into.sizes());
    TORCH_CHECK(grad_.device() == into.device() && ids_.device() == into.device(), "embedding's gradient: the table is on ", into.device(),
                ", gradients on ", grad_.device(), ", ids on ", ids_.device());
    const Tensor ids = token_ids("embedding's gradient", ids_);
    const Tensor grad = with_rows(grad_.reshape({ids.numel(), into.size(1)}));
    const size_t ws_bytes = trlk_embedding_bwd_workspace_bytes(ids.numel(), into.size(0), into.size(1));
    const Tensor ws = bytes(into, ws_bytes);
    check(trlk_embedding_bwd(grad.const_data_ptr(), dtype_code(grad), ids.numel(), into.size(1), grad.stride(0), ids.const_data_ptr(), id_bits(ids),
                             into.size(0), float(scale), padding_idx, accumulate ? 1 : 0, into.mutable_data_ptr(), dtype_code(into), into.stride(0),
                             error_word(into), ws.mutable_data_ptr(), ws_bytes, stream_of(into)));
}

Tensor embedding_bwd(const Tensor& grad, const Tensor& ids, int64_t vocab, double scale, int64_t padding_idx) {
    const c10::DeviceGuard guard(grad.device());
    TORCH_CHECK_VALUE(grad.dim() > 0, "embedding_bwd: gradients have a width");
    const Tensor dweight = at::empty({vocab, grad.size(-1)}, grad.options());
    embedding_into(dweight, grad, ids, scale, padding_idx, false);
    return dweight;
}

void embedding_grad_(const Tensor& grad_weight, const Tensor& grad, const Tensor& ids, double scale, int64_t padding_idx) {
    TORCH_CHECK_VALUE(grad_weight.dim() == 2, "embedding_grad_: the table's gradient is [tokens, width], got shape ", grad_weight.sizes());
    TORCH_CHECK_TYPE(grad_weight.scalar_type() == grad.scalar_type() || grad_weight.scalar_type() == at::kFloat, "embedding_grad_: gradients in ",
                     grad.scalar_type(), " add to a table's gradient of that type or fp32, not ", grad_weight.scalar_type());
    const c10::DeviceGuard guard(grad_weight.device());
    TORCH_CHECK_VALUE((grad_weight.size(1) <= 1 || grad_weight.stride(1) == 1) && (grad_weight.size(0) <= 1 || grad_weight.stride(0) >= grad_weight.size(1)),
                      "embedding_grad_: the table's gradient has gaps between the entries of a row, or rows that overlap");
    TORCH_CHECK_VALUE(grad.numel() == 0 || !grad_weight.is_alias_of(grad) || at::get_overlap_status(grad_weight, grad) == at::MemOverlapStatus::No,
                      "embedding_grad_: the table's gradient shares memory with the tokens' gradients");
    embedding_into(grad_weight, grad, ids, scale, padding_idx, true);
    if (!grad_weight.is_inference()) grad_weight.unsafeGetTensorImpl()->bump_version();
    if (grad.numel()) check_ids();
}

class Embedding : public torch::autograd::Function<Embedding> {
  public:
    static Tensor forward(AutogradContext* ctx, const Tensor& ids, const Tensor& weight, double scale, int64_t padding_idx) {
        ctx->save_for_backward({ids});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["padding_idx"] = padding_idx;
        ctx->saved_data["vocab"] = weight.sym_size(0);
        at::AutoDispatchBelowADInplaceOrView below;
        static const auto op = handle<Tensor(const Tensor&, const Tensor&, double, int64_t)>("trl_amd::embedding");
        return op.call(ids, weight, scale, padding_idx);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        variable_list result(4);
        if (!grads[0].defined()) return result;
        const auto saved = ctx->get_saved_variables();
        static const auto op = handle<Tensor(const Tensor&, const Tensor&, c10::SymInt, double, int64_t)>("trl_amd::embedding_bwd");
        result[1] = op.call(grads[0], saved[0], ctx->saved_data["vocab"].toSymInt(), ctx->saved_data["scale"].toDouble(),
                            ctx->saved_data["padding_idx"].toInt());
        return result;
    }
};
// (padding_idx is the backward's alone)
Tensor embedding(const Tensor& ids, const Tensor& weight, double scale, int64_t) { return embedding_fwd(ids, weight, scale); }
Tensor embedding_autograd(const Tensor& ids, const Tensor& weight, double scale, int64_t padding_idx) {
    if (needs_grad({&weight})) return Embedding::apply(ids, weight, scale, padding_idx);
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = handle<Tensor(const Tensor&, const Tensor&, double, int64_t)>("trl_amd::embedding");
    return op.call(ids, weight, scale, padding_idx);
}

// ---- AdamW ------------------------------------------------------------------------------------------------------------
constexpr int64_t kStateBlock = 256;  // entries of 8-bit moments that share a scale

// Whether memory that a call writes is listed twice, or read as something else: lists of ranges, some of them written.  Lists in ascending
// order, the pieces of one buffer for instance, are told apart by where they begin and end, others by their storages, which share nothing;
// only where a storage comes twice all ranges are sorted.  (2 us of the 40 that a call with 224 tensors takes the host.)
class Ranges {
  public:
    Ranges(size_t n_lists, size_t per_list) : lists_(n_lists, Range{~uintptr_t(0), 0, nullptr, false}) { all_.reserve(n_lists * per_list); }
    void add(size_t list, bool is_written, const Tensor& t, const void* data, size_t bytes) {  // (dense: so many bytes from the first entry)
        if (bytes == 0) return;
        const uintptr_t begin = reinterpret_cast<uintptr_t>(data), end = begin + bytes;
        Range& l = lists_[list];
        ascending_ &= !is_written || begin >= l.end;
        l = {std::min(l.begin, begin), std::max(l.end, end), nullptr, is_written};
        all_.push_back({begin, end, t.storage().unsafeGetStorageImpl(), is_written});
    }
    bool shared() {
        return !(ascending_ && !overlap(lists_)) && storage_twice() && overlap(all_);
    }

  private:
    struct Range {
        uintptr_t begin, end;
        const void* storage;
        bool is_written;
    };
    static bool overlap(std::vector<Range>& ranges) {
        std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
        uintptr_t end = 0, end_written = 0;  // of what lies before
        for (const Range& r : ranges) {
            if (r.begin < (r.is_written ? end : end_written)) return true;
            end = std::max(end, r.end);
            if (r.is_written) end_written = std::max(end_written, r.end);
        }
        return false;
    }
    bool storage_twice() const {
        size_t size = 64;
        while (size < 2 * all_.size()) size *= 2;
        std::vector<const void*> table(size, nullptr);
        for (const bool written : {true, false})  // (storages may be read twice)
            for (const Range& r : all_) {
                if (r.is_written != written) continue;
                size_t at = (reinterpret_cast<uintptr_t>(r.storage) >> 4) * 0x9E3779B97F4A7C15ull >> 32;
                while (table[at & (size - 1)] != nullptr && table[at & (size - 1)] != r.storage) ++at;
                if (table[at & (size - 1)] != nullptr) return true;
                if (written) table[at & (size - 1)] = r.storage;
            }
        return false;
    }
    std::vector<Range> lists_, all_;
    bool ascending_ = true;
};

// (List: at::TensorList, or the tensors of a Python list where they are)
template <typename List>
Tensor adamw_step(const List& params, const List& grads_, const List& exp_avgs, const List& exp_avg_sqs, const List& steps,
                  const List& exp_avg_scales, const List& exp_avg_sq_scales, at::IntArrayRef group_of, at::ArrayRef<double> hyper,
                  const List& lrs, double max_grad_norm, int64_t seed) {
    const size_t n = params.size(), n_groups = hyper.size() / 5;
    TORCH_CHECK_VALUE(grads_.size() == n && exp_avgs.size() == n && exp_avg_sqs.size() == n && steps.size() == n &&
                          (group_of.empty() || group_of.size() == n) && (exp_avg_scales.empty() || exp_avg_scales.size() == n) &&
                          exp_avg_scales.size() == exp_avg_sq_scales.size(),
                      "adamw_step_: the lists differ in length");
    TORCH_CHECK_VALUE(hyper.size() == 5 * n_groups && n_groups > 0 && (lrs.empty() || lrs.size() == n_groups),
                      "adamw_step_: five numbers and one learning rate for each group are expected");
    TORCH_CHECK_VALUE(n > 0, "adamw_step_: no parameters");
    const at::Device device = params[0].device();
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard guard(device);
    std::vector<trlk_adamw_tensor> table(n);
    std::vector<trlk_adamw_group> groups(n_groups);
    std::vector<Tensor> copies;  // of gradients in another order than their parameters
    Ranges ranges(7, n);
    const auto here = [&](const Tensor& t, size_t i, const char* what) {
        TORCH_CHECK(t.device() == device, "adamw_step_: ", what, " ", i, " is on ", t.device(), ", the first parameter on ", device);
    };
    for (size_t g = 0; g < n_groups; ++g) {
        groups[g] = {hyper[5 * g], hyper[5 * g + 1], hyper[5 * g + 2], hyper[5 * g + 3], hyper[5 * g + 4], nullptr};
        if (lrs.empty() || lrs[g].numel() == 0) continue;
        here(lrs[g], g, "learning rate");
        TORCH_CHECK_VALUE(lrs[g].numel() == 1 && lrs[g].scalar_type() == at::kFloat, "adamw_step_: a learning rate on the GPU is one fp32 number");
        groups[g].d_lr = static_cast<const float*>(lrs[g].const_data_ptr());
    }
    for (size_t i = 0; i < n; ++i) {
        const Tensor &p = params[i], &m = exp_avgs[i], &v = exp_avg_sqs[i], &step = steps[i];
        here(p, i, "parameter");
        here(grads_[i], i, "gradient");
        here(m, i, "exp_avg");
        here(v, i, "exp_avg_sq");
        here(step, i, "step");
        const bool eight = m.scalar_type() == at::kFloat8_e4m3fn;
        TORCH_CHECK_VALUE(grads_[i].sizes() == p.sizes() && m.sizes() == p.sizes() && v.sizes() == p.sizes(),
                          "adamw_step_: parameter ", i, " of shape ", p.sizes(), " and its gradient or moments differ in shape");
        TORCH_CHECK_TYPE(grads_[i].scalar_type() == p.scalar_type(), "adamw_step_: parameter ", i, " is ", p.scalar_type(), ", its gradient ",
                         grads_[i].scalar_type());
        TORCH_CHECK_TYPE(eight ? v.scalar_type() == at::kByte : m.scalar_type() == at::kFloat && v.scalar_type() == at::kFloat,
                         "adamw_step_: moments are fp32 both, or float8_e4m3fn and uint8");
        TORCH_CHECK_VALUE(step.numel() == 1 && step.scalar_type() == at::kFloat, "adamw_step_: a step is one fp32 number");
        const bool plain = p.is_contiguous() && m.is_contiguous() && v.is_contiguous();
        TORCH_CHECK_VALUE(plain || (p.is_non_overlapping_and_dense() && m.strides() == p.strides() && v.strides() == p.strides()),
                          "adamw_step_: parameter ", i, " has gaps or its moments another order of entries");
        Tensor g = grads_[i];
        if (!(plain && g.is_contiguous()) && g.strides() != p.strides()) {
            g = at::empty_strided(p.sizes(), p.strides(), p.options()).copy_(g);
            copies.push_back(g);
        }
        trlk_adamw_tensor& t = table[i];
        t = {};
        t.numel = p.numel();
        t.d_param = p.mutable_data_ptr();
        t.d_grad = g.const_data_ptr();
        t.d_exp_avg = m.mutable_data_ptr();
        t.d_exp_avg_sq = v.mutable_data_ptr();
        t.d_step = out(step);
        t.dtype = dtype_code(p);
        t.state_bits = eight ? 8 : 32;
        t.group = group_of.empty() ? 0 : int32_t(group_of[i]);
        const size_t bytes = size_t(t.numel) * p.element_size(), moment_bytes = size_t(t.numel) * (eight ? 1 : sizeof(float));
        ranges.add(0, true, p, t.d_param, bytes);
        ranges.add(1, false, g, t.d_grad, bytes);
        ranges.add(2, true, m, t.d_exp_avg, moment_bytes);
        ranges.add(3, true, v, t.d_exp_avg_sq, moment_bytes);
        ranges.add(4, true, step, t.d_step, sizeof(float));
        if (eight) {
            TORCH_CHECK_VALUE(!exp_avg_scales.empty(), "adamw_step_: 8-bit moments need their scales");
            const int64_t blocks = (t.numel + kStateBlock - 1) / kStateBlock;
            for (const Tensor* s : {&exp_avg_scales[i], &exp_avg_sq_scales[i]}) {
                here(*s, i, "scales");
                TORCH_CHECK_VALUE(s->numel() == blocks && s->scalar_type() == at::kFloat && s->is_contiguous(), "adamw_step_: parameter ", i,
                                  " needs ", blocks, " contiguous fp32 scales for each moment");
            }
            t.d_exp_avg_scale = out(exp_avg_scales[i]);
            t.d_exp_avg_sq_scale = out(exp_avg_sq_scales[i]);
            ranges.add(5, true, exp_avg_scales[i], t.d_exp_avg_scale, size_t(blocks) * sizeof(float));
            ranges.add(6, true, exp_avg_sq_scales[i], t.d_exp_avg_sq_scale, size_t(blocks) * sizeof(float));
        }
    }
    TORCH_CHECK_VALUE(!ranges.shared(), "adamw_step_: parameters, moments, scales or steps are listed twice or share memory, with each other or with a gradient");
    TORCH_CHECK(device.is_cuda(), "adamw_step_: the parameters are on ", device, ", not on a GPU");
    const Tensor norm = at::empty(max_grad_norm < 0 ? at::IntArrayRef({0}) : at::IntArrayRef(), params[0].options().dtype(at::kFloat));
    const size_t ws_bytes = trlk_adamw_workspace_bytes(table.data(), int32_t(n));
    const Tensor ws = bytes(params[0], ws_bytes);
    check(trlk_adamw_step(table.data(), int32_t(n), groups.data(), int32_t(n_groups), max_grad_norm, uint32_t(seed),
                          max_grad_norm < 0 ? nullptr : out(norm), ws.mutable_data_ptr(), ws_bytes, stream_of(params[0])));
    for (const List* list : {&params, &exp_avgs, &exp_avg_sqs, &steps, &exp_avg_scales, &exp_avg_sq_scales})
        for (size_t i = 0; i < list->size(); ++i)
            if (!(*list)[i].is_inference()) (*list)[i].unsafeGetTensorImpl()->bump_version();  // (graphs that saved it learn that it has changed)
    return norm;
}
Tensor adamw_step_(at::TensorList params, at::TensorList grads, at::TensorList exp_avgs, at::TensorList exp_avg_sqs, at::TensorList steps,
                   at::TensorList exp_avg_scales, at::TensorList exp_avg_sq_scales, at::IntArrayRef group_of, at::ArrayRef<double> hyper,
                   at::TensorList lrs, double max_grad_norm, int64_t seed) {
    return adamw_step(params, grads, exp_avgs, exp_avg_sqs, steps, exp_avg_scales, exp_avg_sq_scales, group_of, hyper, lrs, max_grad_norm, seed);
}

// The tensors of a Python list or tuple, held by it.
struct PyTensors {
    PyObject** items = nullptr;
    size_t n = 0;
    size_t size() const { return n; }
    bool empty() const { return n == 0; }
    const Tensor& operator[](size_t i) const { return THPVariable_Unpack(items[i]); }
    // false if something else than plain tensors and parameters is in it
    bool take(PyObject* object) {
        if (!PyList_Check(object) && !PyTuple_Check(object)) return false;
        n = size_t(PySequence_Fast_GET_SIZE(object));
        items = PySequence_Fast_ITEMS(object);
        return std::all_of(items, items + n, [](PyObject* o) { return THPVariable_CheckExact(o); });
    }
};

Tensor adamw_state_values(const Tensor& codes, const Tensor& scales) {
    const bool has_sign = codes.scalar_type() == at::kFloat8_e4m3fn;
    TORCH_CHECK_TYPE(has_sign || codes.scalar_type() == at::kByte, "adamw_state_values: codes are float8_e4m3fn (exp_avg) or uint8 (exp_avg_sq)");
    TORCH_CHECK_VALUE(codes.is_non_overlapping_and_dense() && scales.is_contiguous() && scales.scalar_type() == at::kFloat &&
                          scales.numel() == (codes.numel() + kStateBlock - 1) / kStateBlock,
                      "adamw_state_values: one contiguous fp32 scale for each ", kStateBlock, " codes is expected");
    TORCH_CHECK(codes.device() == scales.device(), "adamw_state_values: codes are on ", codes.device(), ", scales on ", scales.device());
    const c10::DeviceGuard guard(codes.device());
    const Tensor values = at::empty_strided(codes.sizes(), codes.strides(), codes.options().dtype(at::kBFloat16));
    check(trlk_adamw_state_values(static_cast<const uint8_t*>(codes.const_data_ptr()), fptr(scales), codes.numel(), has_sign ? 1 : 0,
                                  values.mutable_data_ptr(), stream_of(codes)));
    return values;
}
// ---- Muon -------------------------------------------------------------------------------------------------------------
// The matrices of tensors [..., m, n], one entry of the table each.  `momenta` null: no step, params are the outputs.
template <typename List>
class MatrixTable {
  public:
    std::vector<trlk_muon_matrix> table;
    MatrixTable(const char* op, const at::Device& device) : op_(op), device_(device) {}
    void add(size_t i, const Tensor& p, const Tensor& g, const Tensor* momentum, int32_t group) {
        TORCH_CHECK(p.device() == device_ && g.device() == device_ && (momentum == nullptr || momentum->device() == device_), op_, ": matrix ", i,
                    " or what belongs to it is not on ", device_, " as the first one");
        TORCH_CHECK_VALUE(p.dim() >= 2, op_, ": matrices are expected, entry ", i, " has shape ", p.sizes());
        const int64_t rows = p.size(-2), cols = p.size(-1), count = p.numel() == 0 ? 0 : p.numel() / (rows * cols);
        for (int64_t k = 0; k < count; ++k) {
            trlk_muon_matrix x{};
            const int64_t at = k * rows * cols;
            x.d_param = static_cast<char*>(p.mutable_data_ptr()) + at * p.element_size();
            x.d_grad = static_cast<const char*>(g.const_data_ptr()) + at * g.element_size();
            x.d_momentum = momentum ? out(*momentum) + at : nullptr;
            x.rows = rows, x.cols = cols, x.dtype = dtype_code(p), x.group = group;
            table.push_back(x);
        }
    }

  private:
    const char* op_;
    at::Device device_;
};
void check_iteration(const char* op, at::ArrayRef<double> c, int64_t steps) {
    TORCH_CHECK_VALUE(c.size() == 3, op, ": three coefficients are expected, got ", c.size());
    TORCH_CHECK_VALUE(steps >= 1 && steps <= 100, op, ": 1 to 100 steps, not ", steps);
}

template <typename List>
void muon_step(const List& params, const List& grads_, const List& momenta, at::IntArrayRef group_of, at::ArrayRef<double> hyper, const List& lrs,
               at::ArrayRef<double> coefficients, int64_t steps, double eps) {
    const size_t n = params.size(), n_groups = hyper.size() / 5;
    TORCH_CHECK_VALUE(grads_.size() == n && momenta.size() == n && (group_of.empty() || group_of.size() == n), "muon_step_: the lists differ in length");
    TORCH_CHECK_VALUE(hyper.size() == 5 * n_groups && n_groups > 0 && (lrs.empty() || lrs.size() == n_groups),
                      "muon_step_: five numbers and one learning rate for each group are expected");
    TORCH_CHECK_VALUE(n > 0, "muon_step_: no parameters");
    check_iteration("muon_step_", coefficients, steps);
    const at::Device device = params[0].device();
    const at::NoGradGuard no_grad;
    const c10::DeviceGuard guard(device);
    std::vector<trlk_muon_group> groups(n_groups);
    for (size_t g = 0; g < n_groups; ++g) {
        const double* h = hyper.data() + 5 * g;
        groups[g] = {h[0], h[1], h[2], nullptr, h[3] != 0.0, int32_t(h[4])};
        if (lrs.empty() || lrs[g].numel() == 0) continue;
        TORCH_CHECK(lrs[g].device() == device, "muon_step_: learning rate ", g, " is on ", lrs[g].device(), ", the first parameter on ", device);
        TORCH_CHECK_VALUE(lrs[g].numel() == 1 && lrs[g].scalar_type() == at::kFloat, "muon_step_: a learning rate on the GPU is one fp32 number");
        groups[g].d_lr = static_cast<const float*>(lrs[g].const_data_ptr());
    }
    MatrixTable<List> matrices("muon_step_", device);
    std::vector<Tensor> copies;  // of gradients that are not contiguous
    Ranges ranges(4, n);
    for (size_t i = 0; i < n; ++i) {
        const Tensor &p = params[i], &m = momenta[i];
        TORCH_CHECK_VALUE(grads_[i].sizes() == p.sizes() && m.sizes() == p.sizes(), "muon_step_: parameter ", i, " of shape ", p.sizes(),
                          " and its gradient or momentum differ in shape");
        TORCH_CHECK_TYPE(grads_[i].scalar_type() == p.scalar_type(), "muon_step_: parameter ", i, " is ", p.scalar_type(), ", its gradient ",
                         grads_[i].scalar_type());
        TORCH_CHECK_TYPE(m.scalar_type() == at::kFloat, "muon_step_: momentum is fp32, not ", m.scalar_type());
        TORCH_CHECK_VALUE(p.is_contiguous() && m.is_contiguous(), "muon_step_: parameter ", i, " or its momentum is not contiguous");
        Tensor g = grads_[i];
        if (!g.is_contiguous()) copies.push_back(g = g.contiguous());
        const int64_t group = group_of.empty() ? 0 : group_of[i];
        TORCH_CHECK_VALUE(group >= 0 && size_t(group) < n_groups, "muon_step_: parameter ", i, " is in no group");
        matrices.add(i, p, g, &m, int32_t(group));
        if (p.numel() == 0) continue;
        const size_t numel = size_t(p.numel());
        ranges.add(0, true, p, p.const_data_ptr(), numel * p.element_size());
        ranges.add(1, false, g, g.const_data_ptr(), numel * g.element_size());
        ranges.add(2, true, m, m.const_data_ptr(), numel * sizeof(float));
    }
    for (size_t g = 0; g < lrs.size(); ++g) {
        if (lrs[g].numel()) ranges.add(3, false, lrs[g], lrs[g].const_data_ptr(), sizeof(float));
    }
    TORCH_CHECK_VALUE(!ranges.shared(), "muon_step_: parameters or momenta are listed twice or share memory, with each other, a gradient or a learning rate");
    TORCH_CHECK(device.is_cuda(), "muon_step_: the parameters are on ", device, ", not on a GPU");
    const int32_t count = int32_t(matrices.table.size());
    const size_t ws_bytes = trlk_muon_workspace_bytes(matrices.table.data(), count);
    const Tensor ws = bytes(params[0], ws_bytes);
    check(trlk_muon_step(matrices.table.data(), count, groups.data(), int32_t(n_groups), int32_t(steps), coefficients[0], coefficients[1],
                         coefficients[2], eps, ws.mutable_data_ptr(), ws_bytes, stream_of(params[0])));
    for (const List* list : {&params, &momenta})
        for (size_t i = 0; i < list->size(); ++i)
            if (!(*list)[i].is_inference()) (*list)[i].unsafeGetTensorImpl()->bump_version();  // (graphs that saved it learn that it has changed)
}
void muon_step_(at::TensorList params, at::TensorList grads, at::TensorList momenta, at::IntArrayRef group_of, at::ArrayRef<double> hyper,
                at::TensorList lrs, at::ArrayRef<double> coefficients, int64_t steps, double eps) {
    muon_step(params, grads, momenta, group_of, hyper, lrs, coefficients, steps, eps);
}

std::vector<Tensor> orthogonalize(at::TensorList matrices, at::ArrayRef<double> coefficients, int64_t steps, double eps) {
    TORCH_CHECK_VALUE(!matrices.empty(), "orthogonalize: no matrices");
    check_iteration("orthogonalize", coefficients, steps);
    const at::Device device = matrices[0].device();
    const c10::DeviceGuard guard(device);
    MatrixTable<at::TensorList> list("orthogonalize", device);
    std::vector<Tensor> inputs, results;
    for (size_t i = 0; i < matrices.size(); ++i) {
        inputs.push_back(matrices[i].contiguous());
        results.push_back(at::empty(matrices[i].sizes(), matrices[i].options()));
        list.add(i, results[i], inputs[i], nullptr, 0);
    }
    TORCH_CHECK(device.is_cuda(), "orthogonalize: the matrices are on ", device, ", not on a GPU");
    const int32_t count = int32_t(list.table.size());
    const size_t ws_bytes = trlk_muon_workspace_bytes(list.table.data(), count);
    const Tensor ws = bytes(matrices[0], ws_bytes);
    check(trlk_orthogonalize(list.table.data(), count, int32_t(steps), coefficients[0], coefficients[1], coefficients[2], eps, ws.mutable_data_ptr(),
                             ws_bytes, stream_of(matrices[0])));
    return results;
}
}  // namespace

// The AdamW step for lists of plain tensors, called with the arguments of the operator in one tuple and the GIL held.  The
// dispatcher takes 80 ns for each entry of a list that comes from Python, 90 us for the five lists of 224 tensors: this takes a fifth.
// Returns None where the operator has to be called (a subclass of tensor, another kind of list), null with a Python error set.
extern "C" __attribute__((visibility("default"))) PyObject* trlk_py_adamw_step(PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject* lists[7];
    PyObject *groups, *hyper, *lrs;
    double max_grad_norm;
    long long seed;
    if (!PyArg_ParseTuple(args, "OOOOOOOOOOdL", &lists[0], &lists[1], &lists[2], &lists[3], &lists[4], &lists[5], &lists[6], &groups, &hyper,
                          &lrs, &max_grad_norm, &seed))
        return nullptr;
    PyTensors tensors[8];
    for (int i = 0; i < 7; ++i)
        if (!tensors[i].take(lists[i])) Py_RETURN_NONE;
    if (!tensors[7].take(lrs) || !PyList_Check(groups) || !PyList_Check(hyper)) Py_RETURN_NONE;
    std::vector<int64_t> group_of;
    std::vector<double> numbers;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(groups); ++i) group_of.push_back(PyLong_AsLongLong(PyList_GET_ITEM(groups, i)));
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(hyper); ++i) numbers.push_back(PyFloat_AsDouble(PyList_GET_ITEM(hyper, i)));
    if (PyErr_Occurred()) return nullptr;
    return THPVariable_Wrap(adamw_step(tensors[0], tensors[1], tensors[2], tensors[3], tensors[4], tensors[5], tensors[6], group_of, numbers,
                                       tensors[7], max_grad_norm, seed));
    END_HANDLE_TH_ERRORS
}

// The same for the orthogonalised updates' step; True where it has been done.
extern "C" __attribute__((visibility("default"))) PyObject* trlk_py_muon_step(PyObject* args) {
    HANDLE_TH_ERRORS
    PyObject *lists[4], *groups, *numbers[2];
    long long steps;
    double eps;
    if (!PyArg_ParseTuple(args, "OOOOOOOLd", &lists[0], &lists[1], &lists[2], &groups, &numbers[0], &lists[3], &numbers[1], &steps, &eps)) return nullptr;
    PyTensors tensors[4];
    for (int i = 0; i < 4; ++i)
        if (!tensors[i].take(lists[i])) Py_RETURN_NONE;
    if (!PyList_Check(groups) || !PyList_Check(numbers[0]) || !PyList_Check(numbers[1])) Py_RETURN_NONE;
    if (tensors[0].size() == 0 || !tensors[0][0].is_cuda()) Py_RETURN_NONE;
    std::vector<int64_t> group_of;
    std::vector<double> hyper, coefficients;
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(groups); ++i) group_of.push_back(PyLong_AsLongLong(PyList_GET_ITEM(groups, i)));
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(numbers[0]); ++i) hyper.push_back(PyFloat_AsDouble(PyList_GET_ITEM(numbers[0], i)));
    for (Py_ssize_t i = 0; i < PyList_GET_SIZE(numbers[1]); ++i) coefficients.push_back(PyFloat_AsDouble(PyList_GET_ITEM(numbers[1], i)));
    if (PyErr_Occurred()) return nullptr;
    muon_step(tensors[0], tensors[1], tensors[2], group_of, hyper, tensors[3], coefficients, steps, eps);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

TORCH_LIBRARY_FRAGMENT(trl_amd, m) {
    m.def("error_flag(int device_index) -> Tensor", error_flag);
    m.def("error_flags() -> Tensor[]", all_error_flags);
    m.def("logp_entropy_fwd(Tensor logits, Tensor index, float temperature, SymInt keep_start, SymInt keep_len, Tensor? row_mask) "
          "-> (Tensor, Tensor, Tensor)");
    m.def("logp_entropy_stats_fwd(Tensor logits, Tensor index, float temperature, SymInt keep_start, SymInt keep_len, "
          "Tensor? row_mask, bool sum_p2=True) -> (Tensor, Tensor, Tensor, Tensor)");
    m.def("logp_entropy_bwd(Tensor logits, Tensor index, float temperature, SymInt keep_start, SymInt keep_len, Tensor lse, "
          "Tensor? entropy, Tensor? g_logp, Tensor? g_entropy) -> Tensor");
    m.def("grpo_loss(Tensor logp, Tensor? old_logp, Tensor? ref_logp, Tensor? entropy, Tensor advantages, Tensor mask, "
          "Tensor? token_weight, Tensor? entropy_mask, Tensor? dapo_normalizer, int loss_type, float epsilon_low, "
          "float epsilon_high, float delta, float beta, bool use_bias_correction_kl, float grad_accum_steps, "
          "float dr_grpo_denominator, float num_processes, float entropy_coef, int policy_term=0, bool sequence_level=False, "
          "Tensor? seq_coef=None, float sapo_temperature_pos=1.0, float sapo_temperature_neg=1.05) "
          "-> (Tensor, Tensor, Tensor, Tensor)");
    m.def("grpo_fused(Tensor logits, Tensor index, float temperature, SymInt keep_start, SymInt keep_len, Tensor mask, "
          "Tensor advantages, Tensor row_scale, Tensor? old_logp, Tensor? ref_logp, Tensor? token_weight, Tensor? seq_coef, "
          "int policy_term, float epsilon_low, float epsilon_high, float delta, float beta, bool use_bias_correction_kl, "
          "float sapo_temperature_pos, float sapo_temperature_neg, bool compute_masked_rows=False, Tensor? entropy_weight=None) "
          "-> (Tensor, Tensor, Tensor, Tensor)");
    m.def("scale_unless_one_(Tensor(a!) data, Tensor scale) -> ()");
    m.def("gradient_in_hand(Tensor(a) loss, Tensor logits, Tensor dlogits, Tensor? upstream) -> Tensor(a)", gradient_in_hand);
    m.def("grpo_log_values(Tensor metrics) -> Tensor");
    m.def("grpo_row_scale(Tensor mask, int loss_type, float numerator, Tensor? n_items, Tensor? upstream, bool with_mask) "
          "-> (Tensor, Tensor)");
    m.def("dpo_loss(Tensor token_logp, Tensor mask, Tensor ref_chosen, Tensor ref_rejected, float beta) "
          "-> (Tensor, Tensor, Tensor, Tensor)");
    m.def("dpo_log_values(Tensor entropy, Tensor row_stats, Tensor mask, Tensor seq_logps, Tensor ref_chosen, "
          "Tensor ref_rejected, float beta) -> Tensor");
    m.def("sample_tokens(Tensor logits, Tensor uniforms, float temperature, int top_k, float top_p, float min_p, "
          "Tensor? temperatures, Tensor? top_ks, Tensor? top_ps, Tensor? min_ps, Tensor? row_mask, int fill_id) -> (Tensor, Tensor)");
    m.def("filtered_logps_fwd(Tensor logits, Tensor index, float temperature, int top_k, float top_p, float min_p, "
          "Tensor? temperatures, Tensor? top_ks, Tensor? top_ps, Tensor? min_ps, Tensor? row_mask) -> (Tensor, Tensor, Tensor)");
    m.def("filtered_logps_bwd(Tensor logits, Tensor index, float temperature, Tensor? temperatures, Tensor state, Tensor block_max, "
          "Tensor g_logp) -> Tensor");
    m.def("adamw_step_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] exp_avgs, Tensor(c!)[] exp_avg_sqs, Tensor(d!)[] steps, "
          "Tensor(e!)[] exp_avg_scales, Tensor(f!)[] exp_avg_sq_scales, int[] group_of, float[] hyper, Tensor[] lrs, "
          "float max_grad_norm, int seed) -> Tensor");
    m.def("adamw_state_values(Tensor codes, Tensor scales) -> Tensor");
    m.def("muon_step_(Tensor(a!)[] params, Tensor[] grads, Tensor(b!)[] momentum_buffers, int[] group_of, float[] hyper, Tensor[] lrs, "
          "float[] coefficients, int steps, float eps) -> ()");
    m.def("orthogonalize(Tensor[] matrices, float[] coefficients, int steps, float eps) -> Tensor[]");
    m.def("embedding(Tensor ids, Tensor weight, float scale, int padding_idx) -> Tensor");
    m.def("embedding_bwd(Tensor grad, Tensor ids, SymInt vocab, float scale, int padding_idx) -> Tensor");
    m.def("embedding_grad_(Tensor(a!) grad_weight, Tensor grad, Tensor ids, float scale, int padding_idx) -> ()");
}
TORCH_LIBRARY_IMPL(trl_amd, CUDA, m) {
    m.impl("logp_entropy_fwd", logp_entropy_fwd);
    m.impl("logp_entropy_stats_fwd", logp_entropy_stats_fwd);
    m.impl("logp_entropy_bwd", logp_entropy_bwd);
    m.impl("grpo_loss", grpo_loss);
    m.impl("grpo_fused", grpo_fused);
    m.impl("scale_unless_one_", scale_unless_one_);
    m.impl("grpo_log_values", grpo_log_values);
    m.impl("grpo_row_scale", grpo_row_scale);
    m.impl("dpo_loss", dpo_loss);
    m.impl("dpo_log_values", dpo_log_values);
    m.impl("sample_tokens", sample_tokens);
    m.impl("filtered_logps_fwd", filtered_logps_fwd);
    m.impl("filtered_logps_bwd", filtered_logps_bwd);
    m.impl("adamw_step_", adamw_step_);
    m.impl("adamw_state_values", adamw_state_values);
    m.impl("muon_step_", muon_step_);
    m.impl("orthogonalize", orthogonalize);
    m.impl("embedding", embedding);
    m.impl("embedding_bwd", embedding_bwd);
    m.impl("embedding_grad_", embedding_grad_);
}
TORCH_LIBRARY_IMPL(trl_amd, Autograd, m) {
    m.impl("logp_entropy_fwd", logp_entropy_fwd_autograd);
    m.impl("logp_entropy_stats_fwd", logp_entropy_stats_fwd_autograd);
    m.impl("grpo_loss", grpo_loss_autograd);
    m.impl("dpo_loss", dpo_loss_autograd);
    m.impl("filtered_logps_fwd", filtered_logps_fwd_autograd);
    m.impl("embedding", embedding_autograd);
    for (const char* name : {"logp_entropy_bwd", "grpo_row_scale", "dpo_log_values", "filtered_logps_bwd", "embedding_bwd", "orthogonalize"})
        m.impl(name, torch::autograd::autogradNotImplementedFallback());
    // (these hand out a gradient, scale one in place, draw or step: their results belong to no graph, whatever the operands require)
    for (const char* name : {"grpo_fused", "scale_unless_one_", "sample_tokens", "adamw_step_", "adamw_state_values", "muon_step_", "embedding_grad_"})
        m.impl(name, torch::CppFunction::makeFallthrough());
}
