// Entry points of the language-model operators (attention.hip, rotary.hip,
// grad_norm.hip), bound in hip_ops.hip.
#pragma once
#include <torch/extension.h>
#include <optional>
#include <tuple>
#include <vector>

torch::Tensor grad_norm(std::vector<torch::Tensor> grads);
torch::Tensor clip_grad_norm(std::vector<torch::Tensor> grads, std::vector<torch::Tensor> outs,
                             double max_norm);

std::vector<torch::Tensor> rotary(std::vector<torch::Tensor> xs, torch::Tensor positions,
                                  torch::Tensor frequencies, bool interleaved, bool inverse);

std::vector<torch::Tensor> attention_forward(torch::Tensor q, torch::Tensor k, torch::Tensor v,
                                             std::optional<torch::Tensor> documents,
                                             std::optional<torch::Tensor> slopes, bool causal,
                                             double scale, bool want_lse);
std::vector<torch::Tensor> attention_backward(torch::Tensor dout, torch::Tensor q,
                                              torch::Tensor k, torch::Tensor v, torch::Tensor out,
                                              torch::Tensor lse,
                                              std::vector<torch::Tensor> ranges,
                                              std::optional<torch::Tensor> documents,
                                              std::optional<torch::Tensor> slopes, bool causal,
                                              double scale);
