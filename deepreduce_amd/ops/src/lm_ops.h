// Entry points of the language-model operators (attention.hip, rotary.hip,
// grad_norm.hip), bound in hip_ops.hip.
#pragma once
#include <torch/extension.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
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
