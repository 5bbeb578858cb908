// Launchers of the per-token losses over a vocabulary, called by their
// bindings and by the differentiable entry points in token_losses_api.cpp.
#pragma once

#include <ATen/core/Tensor.h>
#include <c10/util/Optional.h>

namespace kb {

using OptTensor = c10::optional<at::Tensor>;

// Floats per row that a forward pass keeps for the backward pass.
constexpr int kTokenLogprobsStats = 2;
constexpr int kTopkDistillationStats = 8;
constexpr int kMaxTopK = 128;            // alternatives, or teacher slots, per row
constexpr int kMaxListVocab = 1 << 19;

// logits [rows, >= vocab] with unit inner stride; tokens with logprobs, and top_logprobs with top_ids, may be left out,
// and so may stats where no backward pass follows.
void token_logprobs_forward(const at::Tensor& logits, const OptTensor& tokens, const OptTensor& logprobs,
                            const at::Tensor& entropy, const OptTensor& stats, const OptTensor& top_logprobs,
                            const OptTensor& top_ids, int64_t vocab, double temperature, int64_t ignore_index);

// Row gradients are fp32, contiguous or expanded from one value.
void token_logprobs_backward(const at::Tensor& logits, const OptTensor& tokens, const at::Tensor& stats,
                             const at::Tensor& entropy, const OptTensor& dlogprobs, const OptTensor& dentropy,
                             const at::Tensor& out, int64_t vocab, double temperature, int64_t ignore_index);

// loss = weight * KL per row. With `out`, the gradient of the sum of the losses is written too (over the logits if they
// are the same).
void topk_distillation_forward(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& teacher,
                               const OptTensor& weight, const at::Tensor& loss, const OptTensor& stats,
                               const OptTensor& out, int64_t vocab, double temperature, bool tail);

// Gradient of sum(row_scale * loss) * scale; with `unless_one`, `out` stays as it is where the scale is one.
void topk_distillation_backward(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& teacher,
                                const at::Tensor& stats, const OptTensor& row_scale, const OptTensor& scale,
                                const at::Tensor& out, int64_t vocab, double temperature, bool tail, bool unless_one);

}  // namespace kb
