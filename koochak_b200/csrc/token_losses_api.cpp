// Differentiable entry points of the per-token losses, in C++: for the few
// rows of a decoding step or a short batch the host's work (checks,
// allocations, autograd nodes) outweighs the kernels'.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <stdexcept>
#include <string>
#include <tuple>
#include <vector>

#include "token_losses.h"

namespace kb {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// ValueError and TypeError, with their message put together from the parts. Not by a stream: formatting numbers through
// std::ostringstream (and so through TORCH_CHECK) from this library crashed inside Python processes.
std::string text(const char* t) { return t; }
std::string text(int64_t n) { return std::to_string(n); }
std::string text(int n) { return std::to_string(n); }
std::string text(double x) { return std::to_string(x); }
std::string text(at::IntArrayRef sizes) {
  std::string t = "[";
  for (size_t i = 0; i < sizes.size(); ++i) t += (i ? ", " : "") + std::to_string(sizes[i]);
  return t + "]";
}
template <typename Error, typename... P>
void require(bool ok, const P&... parts) {
  if (!ok) throw Error((std::string() + ... + text(parts)));
}
template <typename... P>
void check_value(bool ok, const P&... parts) {
  require<pybind11::value_error>(ok, parts...);
}

// logits [..., vocab] as [rows, vocab] with unit inner stride, without a copy where the strides allow it.
at::Tensor vocab_rows(const at::Tensor& logits, const char* name) {
  check_value(logits.dim() >= 1 && logits.size(-1) >= 1, name,
                    ": logits must be [..., vocab] with at least one column");
  check_value(logits.size(-1) <= kMaxListVocab, name, ": vocabularies of more than ", kMaxListVocab,
                    " entries are not supported");
  require<pybind11::type_error>(logits.scalar_type() == at::kBFloat16 || logits.scalar_type() == at::kHalf ||
                       logits.scalar_type() == at::kFloat,
                   name, ": logits must be bf16, fp16 or fp32, got ", at::toString(logits.scalar_type()));
  const int64_t vocab = logits.size(-1);
  at::Tensor z = logits.dim() == 2 ? logits : logits.reshape({logits.numel() / vocab, vocab});
  return z.stride(1) == 1 || vocab == 1 ? z : z.contiguous();
}

// Rows that start where z's do modulo 16 bytes, if z's rows do not overlap.
at::Tensor like_rows(const at::Tensor& z) {
  const int64_t rows = z.size(0), vocab = z.size(1);
  if (rows <= 1 || z.stride(0) < vocab || z.stride(0) > vocab + 1024 || z.stride(0) == vocab)
    return at::empty({rows, vocab}, z.options());
  return at::empty({rows, z.stride(0)}, z.options()).narrow(1, 0, vocab);
}

void check_temperature(double t, const char* name) {
  check_value(t >= 1e-4 && t <= 1e4, name, ": temperature must lie in [1e-4, 1e4], got ", t);
}

// fp32 rows, contiguous or expanded from one value.
OptTensor row_gradient(const at::Tensor& g) {
  if (!g.defined()) return c10::nullopt;
  const at::Tensor f = g.scalar_type() == at::kFloat ? g : g.to(at::kFloat);
  bool one = f.numel() > 0;
  for (int64_t s : f.strides()) one &= s == 0;
  if (f.dim() > 0 && one) return f.as_strided({f.numel()}, {0});
  return f.reshape({-1}).contiguous();
}

// The backward passes are kernels without a derivative of their own: differentiating their result raises, with respect to
// the upstream gradient or to the logits, which it always depends on.
at::Tensor once_differentiable(const at::Tensor& dz, bool recorded) {
  if (!recorded) return dz;
  at::AutoGradMode on(true);
  auto err = std::make_shared<torch::autograd::DelayedError>("this backward pass cannot be differentiated", 1);
  return (*err)(variable_list{dz.detach().requires_grad_()})[0];
}

// A tangent of the logits would not reach the results: the kernels have no forward mode.
void refuse_tangent(const at::Tensor& logits, const char* name) {
  require<std::runtime_error>(!logits._fw_grad(/*level=*/0).defined(), name,
                              ": forward-mode differentiation is not supported on CUDA");
}

using Logprobs = std::tuple<OptTensor, at::Tensor, OptTensor, OptTensor>;

struct LogprobsOut {
  at::Tensor logprobs, entropy, stats, top_logprobs, top_ids;
};

LogprobsOut logprobs_rows(const at::Tensor& logits, const at::Tensor& z, const OptTensor& tokens, int64_t top_k,
                          double temperature, int64_t ignore_index, bool keep) {
  const auto f32 = z.options().dtype(at::kFloat);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  LogprobsOut r;
  r.entropy = at::empty(lead, f32);
  if (tokens) r.logprobs = at::empty(lead, f32);
  if (keep) r.stats = at::empty({z.size(0), kTokenLogprobsStats}, f32);
  OptTensor top_logprobs, top_ids;
  if (top_k > 0) {
    std::vector<int64_t> shape(lead.begin(), lead.end());
    shape.push_back(top_k);
    r.top_logprobs = at::empty(shape, f32);
    r.top_ids = at::empty(shape, z.options().dtype(at::kLong));
    top_logprobs = r.top_logprobs;
    top_ids = r.top_ids;
  }
  token_logprobs_forward(z, tokens, tokens ? OptTensor(r.logprobs) : OptTensor(), r.entropy,
                         keep ? OptTensor(r.stats) : OptTensor(), top_logprobs, top_ids, z.size(1), temperature,
                         ignore_index);
  return r;
}

struct LogprobsFn : torch::autograd::Function<LogprobsFn> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& logits, const OptTensor& tokens, int64_t top_k,
                               double temperature, int64_t ignore_index) {
    const LogprobsOut r = logprobs_rows(logits, vocab_rows(logits, "token_logprobs"), tokens, top_k, temperature,
                                        ignore_index, true);
    ctx->save_for_backward({logits, tokens ? *tokens : at::Tensor(), r.stats, r.entropy.detach()});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["ignore_index"] = ignore_index;
    ctx->set_materialize_grads(false);
    variable_list out{r.entropy};
    if (tokens) out.push_back(r.logprobs);
    if (top_k > 0) {
      out.push_back(r.top_logprobs);
      out.push_back(r.top_ids);
      ctx->mark_non_differentiable({r.top_logprobs, r.top_ids});
    }
    return out;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor& logits = saved[0];
    const bool recorded = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    const OptTensor tokens = saved[1].defined() ? OptTensor(saved[1]) : OptTensor();
    const at::Tensor z = vocab_rows(logits, "token_logprobs");
    const at::Tensor dz = like_rows(z);
    token_logprobs_backward(z, tokens, saved[2], saved[3], tokens ? row_gradient(grads[1]) : OptTensor(),
                            row_gradient(grads[0]), dz, z.size(1), ctx->saved_data["temperature"].toDouble(),
                            ctx->saved_data["ignore_index"].toInt());
    const at::Tensor shaped = logits.dim() == 2 ? dz : dz.view(logits.sizes());
    return {once_differentiable(shaped, recorded), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

Logprobs token_logprobs(const at::Tensor& logits, const OptTensor& given, int64_t top_k, double temperature,
                        int64_t ignore_index) {
  const char* name = "token_logprobs";
  refuse_tangent(logits, name);
  at::Tensor z;
  {
    at::NoGradGuard no_grad;
    z = vocab_rows(logits, name);
  }
  check_temperature(temperature, name);
  check_value(top_k >= 0 && top_k <= std::min<int64_t>(kMaxTopK, z.size(1)), name, ": top_k must lie in [0, ",
                    std::min<int64_t>(kMaxTopK, z.size(1)), "], got ", top_k);
  OptTensor tokens;
  if (given) {
    check_value(given->sizes() == logits.sizes().slice(0, logits.dim() - 1) && given->scalar_type() == at::kLong &&
                          given->device() == logits.device(),
                      name, ": tokens must be int64 of shape ", logits.sizes().slice(0, logits.dim() - 1), " on the logits' device");
    tokens = given->reshape({-1}).contiguous();
  }
  const auto some = [](const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
  if (!at::GradMode::is_enabled() || !logits.requires_grad()) {
    const LogprobsOut r = logprobs_rows(logits, z, tokens, top_k, temperature, ignore_index, false);
    return {some(r.logprobs), r.entropy, some(r.top_logprobs), some(r.top_ids)};
  }
  const variable_list out = LogprobsFn::apply(logits, tokens, top_k, temperature, ignore_index);
  const size_t top = tokens ? 2 : 1;
  return {tokens ? OptTensor(out[1]) : OptTensor(), out[0], top_k > 0 ? OptTensor(out[top]) : OptTensor(),
          top_k > 0 ? OptTensor(out[top + 1]) : OptTensor()};
}

// Names the graph capture that the current stream of a device is in; 0 outside of any.
int64_t capture_id(const at::Tensor& t) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  C10_CUDA_CHECK(cudaStreamGetCaptureInfo(c10::cuda::getCurrentCUDAStream(t.get_device()).stream(), &status, &id));
  return status == cudaStreamCaptureStatusActive ? (int64_t)id : 0;
}

// Loss rows, or with a weight their weighted sum.
//
// The sum's gradient is written by the forward kernel, for an upstream
// gradient of one, while the row is on the chip; the backward pass leaves it
// where the upstream gradient is one (told on the device) and computes it anew
// otherwise, so it is rounded once in either case. fp16 logits, whose loss
// goes through a gradient scaler, take the two passes at once. A backward pass
// captured without its forward pass runs many times on one forward pass, with
// other upstream gradients and on what was made of its last result, so it
// computes its own.
struct DistillationFn : torch::autograd::Function<DistillationFn> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& logits, const at::Tensor& ids,
                            const at::Tensor& teacher, const OptTensor& weight, double temperature, bool tail) {
    const at::Tensor z = vocab_rows(logits, "topk_distillation");
    const auto f32 = z.options().dtype(at::kFloat);
    const at::Tensor loss = weight ? at::empty({z.size(0)}, f32) : at::empty(logits.sizes().slice(0, logits.dim() - 1), f32);
    const at::Tensor stats = at::empty({z.size(0), kTopkDistillationStats}, f32);
    OptTensor dz;
    if (weight && logits.scalar_type() != at::kHalf) dz = like_rows(z);
    topk_distillation_forward(z, ids, teacher, weight, loss, stats, dz, z.size(1), temperature, tail);
    ctx->save_for_backward({logits, ids, teacher, weight ? *weight : at::Tensor(), stats});
    ctx->saved_data["temperature"] = temperature;
    ctx->saved_data["tail"] = tail;
    if (dz) {
      ctx->saved_data["dz"] = *dz;
      ctx->saved_data["capture"] = capture_id(z);
    }
    return weight ? loss.sum() : loss;
  }

  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor& logits = saved[0];
    const bool recorded = at::GradMode::is_enabled();
    at::NoGradGuard no_grad;
    const at::Tensor z = vocab_rows(logits, "topk_distillation");
    const bool summed = saved[3].defined();
    // A gradient that is there is handed out once; a second backward pass computes its own.
    const auto found = ctx->saved_data.find("dz");
    const bool ready = found != ctx->saved_data.end() && ctx->saved_data["capture"].toInt() == capture_id(z);
    at::Tensor dz;
    if (ready) {
      dz = found->second.toTensor();
      ctx->saved_data.erase("dz");
    } else {
      dz = like_rows(z);
    }
    const OptTensor g = row_gradient(grads[0]);
    topk_distillation_backward(z, saved[1], saved[2], saved[4], summed ? OptTensor(saved[3]) : g,
                               summed ? g : OptTensor(), dz, z.size(1), ctx->saved_data["temperature"].toDouble(),
                               ctx->saved_data["tail"].toBool(), ready);
    const at::Tensor shaped = logits.dim() == 2 ? dz : dz.view(logits.sizes());
    return {once_differentiable(shaped, recorded), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

at::Tensor topk_distillation(const at::Tensor& logits, const at::Tensor& teacher_ids, const at::Tensor& teacher_logits,
                             double temperature, bool tail, const OptTensor& given_weight, bool summed) {
  const char* name = "topk_distillation";
  refuse_tangent(logits, name);
  const bool differentiable = at::GradMode::is_enabled() && logits.requires_grad();
  at::NoGradGuard no_grad;
  const at::Tensor z = vocab_rows(logits, name);
  check_temperature(temperature, name);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  check_value(teacher_ids.dim() == logits.dim() && teacher_ids.sizes().slice(0, logits.dim() - 1) == lead &&
                        teacher_ids.scalar_type() == at::kLong,
                    name, ": teacher_ids must be int64 of shape [*", lead, ", k]");
  check_value(teacher_logits.sizes() == teacher_ids.sizes() && at::isFloatingType(teacher_logits.scalar_type()),
                    name, ": teacher_logits must be floating, of teacher_ids' shape");
  const int64_t k = teacher_ids.size(-1);
  check_value(k >= 1 && k <= kMaxTopK, name, ": 1 to ", kMaxTopK, " teacher slots per row, got ", k);
  check_value(!given_weight || (summed && given_weight->sizes() == lead), name,
                    ": weight goes with reduction='sum' and has shape ", lead);
  check_value(teacher_ids.device() == logits.device() && teacher_logits.device() == logits.device() &&
                        (!given_weight || given_weight->device() == logits.device()),
                    name, ": all tensors must be on the logits' device");
  const int64_t rows = z.size(0);
  const at::Tensor ids = teacher_ids.reshape({rows, k}).contiguous();
  const at::Tensor teacher = teacher_logits.detach().reshape({rows, k}).to(at::kFloat).contiguous();
  OptTensor weight;
  if (summed)
    weight = given_weight ? given_weight->detach().reshape({-1}).to(at::kFloat).contiguous()
                          : at::ones({rows}, z.options().dtype(at::kFloat));
  if (differentiable) {
    at::AutoGradMode on(true);
    return DistillationFn::apply(logits, ids, teacher, weight, temperature, tail);
  }
  const auto f32 = z.options().dtype(at::kFloat);
  const at::Tensor loss = summed ? at::empty({rows}, f32) : at::empty(lead, f32);
  topk_distillation_forward(z, ids, teacher, weight, loss, c10::nullopt, c10::nullopt, z.size(1), temperature, tail);
  return summed ? loss.sum() : loss;
}

}  // namespace

void register_token_loss_api(pybind11::module& m) {
  m.def("token_logprobs", torch::wrap_pybind_function(token_logprobs), "differentiable log probabilities, entropies and alternatives");
  m.def("topk_distillation", torch::wrap_pybind_function(topk_distillation), "differentiable KL divergence from a teacher's top logits");
}

}  // namespace kb
