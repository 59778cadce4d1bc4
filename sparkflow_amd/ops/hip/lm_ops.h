// The language-model operators' launchers (dropout.hip, logprobs.hip,
// adapter.hip), for the bindings and the autograd nodes.
#pragma once

#include <torch/extension.h>

#include <vector>

// dropout.hip — mask drawn from a counter, never stored
torch::Tensor dropout(torch::Tensor x, torch::Tensor state, int64_t keep,
                      double scale);
torch::Tensor dropout_next(torch::Tensor state);

// logprobs.hip — scores of given tokens, entropy, best alternatives
std::vector<torch::Tensor> logprobs_fwd(torch::Tensor logits,
                                        torch::Tensor tokens, int64_t k,
                                        int64_t ignore);
torch::Tensor logprobs_bwd(torch::Tensor logits, torch::Tensor tokens,
                           torch::Tensor stat, torch::Tensor entropy,
                           torch::Tensor ids,
                           c10::optional<torch::Tensor> g_logp,
                           c10::optional<torch::Tensor> g_entropy,
                           c10::optional<torch::Tensor> g_top,
                           int64_t ignore);

// adapter.hip — low-rank adapters of many requests
torch::Tensor adapter_plan(torch::Tensor ids, int64_t E);
torch::Tensor adapter_shrink(torch::Tensor x, torch::Tensor w,
                             torch::Tensor ids, torch::Tensor plan,
                             c10::optional<torch::Tensor> scales,
                             double scale, bool kmajor, bool split);
torch::Tensor adapter_expand(c10::optional<torch::Tensor> base,
                             torch::Tensor z, torch::Tensor w,
                             torch::Tensor ids, torch::Tensor plan,
                             int64_t act, bool rmajor);
std::vector<torch::Tensor> adapter_outer(c10::optional<torch::Tensor> x,
                                         c10::optional<torch::Tensor> dz,
                                         c10::optional<torch::Tensor> dy,
                                         c10::optional<torch::Tensor> z,
                                         torch::Tensor ids,
                                         torch::Tensor plan, int64_t E,
                                         int64_t R);
torch::Tensor adapter_act_bwd(torch::Tensor y, torch::Tensor dy,
                              int64_t act);

// lm_autograd.cpp — the same with their gradients
torch::Tensor dropout_apply(torch::Tensor x, torch::Tensor state,
                            int64_t keep, double scale);
std::vector<torch::Tensor> logprobs_apply(torch::Tensor logits,
                                          torch::Tensor tokens, int64_t k,
                                          int64_t ignore);
torch::Tensor adapter_add_apply(torch::Tensor base, torch::Tensor x,
                                torch::Tensor a, torch::Tensor b,
                                c10::optional<torch::Tensor> scales,
                                double scale, torch::Tensor ids,
                                c10::optional<torch::Tensor> plan,
                                int64_t act);
