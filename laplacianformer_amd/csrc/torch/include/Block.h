// The transformer-block operators' host functions (torch adapters of the C ABI).
#pragma once

#include <torch/types.h>

#include <optional>
#include <vector>

namespace laplace {

std::vector<at::Tensor> AddRmsNorm_forward(const at::Tensor x, const at::Tensor weight,
                                           const std::optional<at::Tensor> residual, double eps, bool need_rstd);
std::vector<at::Tensor> AddRmsNorm_forward_fp8(const at::Tensor x, const at::Tensor weight,
                                               const std::optional<at::Tensor> residual, double eps);
std::vector<at::Tensor> AddRmsNorm_backward(const at::Tensor grad_y, const std::optional<at::Tensor> grad_sum,
                                            const at::Tensor x, const at::Tensor weight,
                                            const std::optional<at::Tensor> residual, const at::Tensor rstd,
                                            bool need_weight);
std::vector<at::Tensor> Rotary(const at::Tensor q, const std::optional<at::Tensor> k, const at::Tensor positions,
                               const std::vector<int64_t> sections, double base, bool interleaved, bool inverse);
std::vector<at::Tensor> SoftmaxAttention_forward(const at::Tensor q, const at::Tensor k, const at::Tensor v,
                                                 const std::optional<at::Tensor> mask, bool causal,
                                                 const std::optional<at::Tensor> k_lengths,
                                                 const std::optional<at::Tensor> q_lengths,
                                                 const std::optional<at::Tensor> q_starts, double scale,
                                                 bool need_stats);
std::vector<at::Tensor> SoftmaxAttention_backward(const at::Tensor grad_out, const at::Tensor q, const at::Tensor k,
                                                  const at::Tensor v, const at::Tensor out, const at::Tensor stats,
                                                  const std::optional<at::Tensor> mask, bool causal,
                                                  const std::optional<at::Tensor> k_lengths,
                                                  const std::optional<at::Tensor> q_lengths,
                                                  const std::optional<at::Tensor> q_starts, double scale, bool need_q,
                                                  bool need_kv);

// [y, sum, rstd, post_rstd]; [dx, dresidual, dweight, dpost_weight, dgate], undefined where not asked for.
std::vector<at::Tensor> GatedAddRmsNorm_forward(const at::Tensor x, const at::Tensor weight, const at::Tensor residual,
                                                const std::optional<at::Tensor> post_weight,
                                                const std::optional<at::Tensor> gate, double scale, double eps, bool need_rstd);
std::vector<at::Tensor> GatedAddRmsNorm_backward(const at::Tensor grad_y, const std::optional<at::Tensor> grad_sum,
                                                 const at::Tensor x, const at::Tensor weight, const at::Tensor residual,
                                                 const std::optional<at::Tensor> post_weight,
                                                 const std::optional<at::Tensor> gate, const at::Tensor rstd,
                                                 const std::optional<at::Tensor> post_rstd, double scale, double eps,
                                                 bool need_weight, bool need_post_weight, bool need_gate);
// state, last and their gradients: fp32 [batch, heads, key channels, value channels]; undefined where not asked for.
std::vector<at::Tensor> DecayAttention_forward(const at::Tensor q, const at::Tensor k, const at::Tensor v,
                                               const at::Tensor log_decay, const std::optional<at::Tensor> state,
                                               const std::optional<at::Tensor> lengths, double scale, bool need_last);
std::vector<at::Tensor> DecayAttention_backward(const std::optional<at::Tensor> grad_out,
                                                const std::optional<at::Tensor> grad_last, const at::Tensor q,
                                                const at::Tensor k, const at::Tensor v, const at::Tensor log_decay,
                                                const std::optional<at::Tensor> state,
                                                const std::optional<at::Tensor> lengths, double scale, bool need_q,
                                                bool need_kv, bool need_state);
at::Tensor DecayAttentionStep(const at::Tensor q, const at::Tensor k, const at::Tensor v, const at::Tensor log_decay,
                              const at::Tensor state, double scale);

// Those with autograd: [y] or [y, sum]; [q', k' or undefined]; out.
std::vector<at::Tensor> AddRmsNorm(const at::Tensor x, const at::Tensor weight, const std::optional<at::Tensor> residual,
                                   double eps);
std::vector<at::Tensor> RotaryPositions(const at::Tensor q, const std::optional<at::Tensor> k, const at::Tensor positions,
                                        const std::vector<int64_t> sections, double base, bool interleaved);
at::Tensor SoftmaxAttention(const at::Tensor q, const at::Tensor k, const at::Tensor v, const std::optional<at::Tensor> mask,
                            bool causal, const std::optional<at::Tensor> k_lengths,
                            const std::optional<at::Tensor> q_lengths, const std::optional<at::Tensor> q_starts,
                            double scale);
std::vector<at::Tensor> GatedAddRmsNorm(const at::Tensor x, const at::Tensor weight, const at::Tensor residual,
                                        const std::optional<at::Tensor> post_weight, const std::optional<at::Tensor> gate,
                                        double scale, double eps);
// [out] or [out, last].
std::vector<at::Tensor> DecayAttention(const at::Tensor q, const at::Tensor k, const at::Tensor v, const at::Tensor log_decay,
                                       const std::optional<at::Tensor> state, const std::optional<at::Tensor> lengths,
                                       double scale, bool return_state);

}  // namespace laplace
