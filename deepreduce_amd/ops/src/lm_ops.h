// Entry points of the language-model operators (attention.hip, rotary.hip,
// grad_norm.hip), bound in hip_ops.hip.
#pragma once
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <ATen/hip/HIPContext.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <optional>
#include <string>
#include <vector>

torch::Tensor grad_norm(std::vector<torch::Tensor> grads);
std::pair<std::vector<torch::Tensor>, torch::Tensor> clip_grad_norm(
    std::vector<torch::Tensor> grads, double max_norm,
    std::optional<std::vector<torch::Tensor>> out, std::optional<torch::ScalarType> dtype);

std::vector<torch::Tensor> rotary(torch::Tensor q, torch::Tensor k, torch::Tensor positions,
                                  torch::Tensor frequencies, bool interleaved);

torch::Tensor attention(torch::Tensor q, torch::Tensor k, torch::Tensor v,
                        std::optional<torch::Tensor> documents,
                        std::optional<torch::Tensor> slopes, bool causal,
                        std::optional<double> scale);

// A leaf keeps the node that takes its gradient, and that node's stream, as
// long as any graph holds it.  A backward pass that is captured on another
// stream would leave the capture through it, which ends the process: the
// functions note such leaves and refuse that backward.
inline bool held_elsewhere(std::initializer_list<torch::Tensor> leaves) {
    for (auto& t : leaves) {
        if (!t.requires_grad() || !t.is_leaf()) continue;
        auto node = torch::autograd::impl::try_get_grad_accumulator(t);
        if (!node) continue;
        const c10::impl::VirtualGuardImpl device(t.device().type());
        const auto stream = node->stream();
        if (stream && *stream != device.getStream(t.device())) return true;
    }
    return false;
}
inline void check_capture(bool elsewhere, const char* name) {
    if (!elsewhere) return;
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    C10_HIP_CHECK(hipStreamIsCapturing(at::hip::getCurrentHIPStream(), &status));
    TORCH_CHECK(status == hipStreamCaptureStatusNone, name,
                ": an eager graph of the same leaves is alive on another stream; let it go before "
                "a backward pass is captured");
}

// A kernel's launch is no operation that torch sees: forward-mode derivatives
// would end at it, and a tracer would record its empty results.
inline void check_seen(std::initializer_list<torch::Tensor> inputs, const char* name) {
    using c10::impl::TorchDispatchModeTLS;
    TORCH_CHECK(!torch::jit::tracer::isTracing() &&
                    !TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY),
                name, ": cannot be traced on a GPU");
    if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
    for (auto& t : inputs)
        TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), name,
                                    ": has no forward-mode derivative");
}

// gradients that may be used in a graph of their own but not through it
inline torch::autograd::variable_list once_differentiable(torch::autograd::variable_list grads,
                                                          const char* name) {
    if (!at::GradMode::is_enabled()) return grads;
    auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string(name) + " is differentiable once", (int64_t)grads.size());
    for (auto& g : grads)
        if (g.defined()) g = g.detach().requires_grad_();
    return (*error)(std::move(grads));
}
