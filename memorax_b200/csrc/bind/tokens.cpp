// Both ends of a network over discrete symbols: rows of a table by token, and log probabilities of tokens.
#include <ATen/cuda/CUDAGraphsUtils.cuh>

#include "common.h"

namespace mxk_host {

int type_of(const Tensor& t, const char* name) {
  switch (t.scalar_type()) {
    case at::kFloat: return MXK_F32;
    case at::kBFloat16: return MXK_BF16;
    case at::kHalf: return MXK_F16;
    default: TORCH_CHECK_VALUE(false, name, " must be float32, bfloat16 or float16, got ", t.scalar_type());
  }
}
// Tangents and traces end at a native call: both are refused, here or by the autograd node.
void not_traced(const char* name) { TORCH_CHECK_VALUE(!torch::jit::tracer::isTracing(), name, " cannot be traced"); }
bool with_node(const char* name, std::initializer_list<Tensor> inputs) {
  bool any = false;
  for (const Tensor& t : inputs)
    if (t.defined() && ((at::GradMode::is_enabled() && t.requires_grad()) || (torch::autograd::ForwardADLevel::try_get_by_idx(0) && followed(t)))) any = true;
  if (any && at::cuda::currentStreamCaptureStatusMayInitCtx() != at::cuda::CaptureStatus::None) {
    // Where an eager graph of a leaf lives, its gradient is accumulated on that graph's stream, here too; a backward pass would
    // pull that stream into the capture, which the default one does not let happen: the process ends.
    for (const Tensor& t : inputs) {
      if (!t.defined() || !t.requires_grad() || !t.is_leaf()) continue;
      const auto accumulator = torch::autograd::impl::try_get_grad_accumulator(t);
      const auto home = accumulator ? accumulator->stream() : std::nullopt;
      TORCH_CHECK(!home || c10::cuda::CUDAStream(*home).stream() != nullptr, name,
                  ": a graph of the same parameter that was built on the default stream lives; release it before a capture");
    }
  }
  return any;
}
void once(const char* name) { TORCH_CHECK(!at::GradMode::is_enabled(), name, ": the gradient itself has none (create_graph)"); }

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// int32 or int64 on the device of `like`, dense
Tensor tokens_of(const Tensor& t, const Tensor& like, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == like.device(), name, " must be on ", like.device(), ", got ", t.device());
  TORCH_CHECK_VALUE(t.scalar_type() == at::kLong || t.scalar_type() == at::kInt, name, " must be int32 or int64, got ", t.scalar_type());
  return t.contiguous();
}
int width_of(const Tensor& t) { return t.scalar_type() == at::kLong ? 8 : 4; }

// ---------------------------------------------------------------------------------------------------------- embedding
Tensor lookup(const Tensor& ids, const Tensor& table, double scale, const Tensor& sorted = Tensor()) {
  auto sizes = ids.sizes().vec();
  sizes.push_back(table.size(1));
  const Tensor out = empty_like_of(table, sizes, table.scalar_type());
  if (ids.numel())
    check("mxk_embedding_fwd", mxk_embedding_fwd(ids.data_ptr(), width_of(ids), table.data_ptr(), out.data_ptr(), ptr<void>(sorted), sorted.defined() ? sorted.numel() : 0,
                                                 ids.numel(), table.size(0), table.size(1), type_of(table, "weight"), scale, stream()));
  return out;
}

struct Embedding : torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& table, const Tensor& ids, double scale) {
    const Tensor sorted = scratch(table, mxk_embedding_sorted_bytes(ids.numel(), table.size(0)));
    ctx->save_for_backward({sorted});
    ctx->saved_data["rows"] = ids.numel();
    ctx->saved_data["vocab"] = table.size(0);
    ctx->saved_data["type"] = static_cast<int64_t>(table.scalar_type());
    ctx->saved_data["scale"] = scale;
    return lookup(ids, dense(table), scale, sorted);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& gout) {
    once("embedding");
    const Tensor sorted = ctx->get_saved_variables()[0];
    const c10::cuda::CUDAGuard guard(sorted.device());
    const auto type = static_cast<at::ScalarType>(ctx->saved_data["type"].toInt());
    const Tensor dy = dense(gout[0].scalar_type() == type ? gout[0] : gout[0].to(type));
    const int64_t rows = ctx->saved_data["rows"].toInt(), vocab = ctx->saved_data["vocab"].toInt(), dim = gout[0].size(-1);
    const Tensor dw = empty_like_of(dy, {vocab, dim}, type);
    const size_t ws_bytes = mxk_embedding_bwd_workspace_bytes(rows, dim);
    const Tensor ws = scratch(dy, ws_bytes);
    check("mxk_embedding_bwd", mxk_embedding_bwd(sorted.data_ptr(), sorted.numel(), dy.data_ptr(), dw.data_ptr(), ws.data_ptr(), ws_bytes, rows, vocab, dim, type_of(dy, "dy"),
                                                 ctx->saved_data["scale"].toDouble(), stream()));
    return {dw, Tensor(), Tensor()};
  }
};

Tensor embedding(const Tensor& ids_in, const Tensor& table, double scale) {
  not_traced("embedding");
  TORCH_CHECK_VALUE(table.is_cuda(), "weight must be a CUDA tensor (memorax_b200 has no CPU path)");
  TORCH_CHECK_VALUE(table.dim() == 2 && table.numel() > 0 && table.size(1) <= 1 << 24, "weight must be (vocabulary, features), at most 2^24 of these, got ", table.sizes());
  type_of(table, "weight");
  const c10::cuda::CUDAGuard guard(table.device());
  const Tensor ids = tokens_of(ids_in, table, "ids");
  if (with_node("embedding", {table})) return Embedding::apply(table, ids, scale);
  return lookup(ids, dense(table), scale);
}

// -------------------------------------------------------------------------------------------------- log probabilities
// (rows, n) with neighbours in a row and rows a fixed step apart; copied where the memory is not laid out like that
struct Rows {
  Tensor t;
  int64_t ld;
};
Rows rows_of(const Tensor& in) {
  const Tensor t = in.is_neg() ? in.resolve_neg() : in;
  const int64_t d = t.dim();
  bool fits = t.size(-1) == 1 || t.stride(-1) == 1;
  int64_t ld = 0, inner = 1;     // of the extents over one: from the last to the first
  bool first = true;
  for (int64_t i = d - 2; i >= 0 && fits; --i) {
    if (t.size(i) == 1) continue;
    if (first) ld = t.stride(i), first = false;
    else fits = t.stride(i) == ld * inner;
    inner *= t.size(i);
  }
  if (fits) return {t, first ? t.size(-1) : ld};
  return {t.contiguous(), t.size(-1)};
}
// per-row cotangents; one value for all rows (an expanded one) is read as it is
struct PerRow {
  Tensor t;
  int64_t ld = 0;
};
PerRow per_row(const Tensor& in) {
  if (!in.defined()) return {};
  const Tensor t = in.scalar_type() == at::kFloat && !in.is_neg() ? in : dense(in.to(at::kFloat));
  bool same = true;
  for (int64_t i = 0; i < t.dim(); ++i) same &= t.size(i) == 1 || t.stride(i) == 0;
  if (same) return {t, 0};
  return {t.contiguous(), 1};
}

struct Logprobs {
  Tensor log_prob, entropy, top_value, top_index, stats;
};
Logprobs measure(const Tensor& logits, const Tensor& tokens, const Tensor& mask, double temperature, int64_t top, bool keep) {
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  const int64_t vocab = logits.size(-1), rows = logits.numel() / vocab;
  const Rows x = rows_of(logits), m = mask.defined() ? rows_of(mask) : Rows{};
  Logprobs out;
  if (tokens.defined()) out.log_prob = empty_like_of(logits, lead, at::kFloat);
  out.entropy = empty_like_of(logits, lead, at::kFloat);
  auto sizes = lead.vec();
  sizes.push_back(top);
  if (top) {
    out.top_value = empty_like_of(logits, sizes, at::kFloat);
    out.top_index = empty_like_of(logits, sizes, at::kLong);
  }
  if (keep) out.stats = empty_like_of(logits, {rows, 4}, at::kFloat);
  if (rows)
    check("mxk_token_logprob_fwd",
          mxk_token_logprob_fwd(x.t.data_ptr(), x.ld, bytes(m.t), m.ld, ptr<void>(tokens), tokens.defined() ? width_of(tokens) : 0, ptr(out.log_prob), ptr(out.entropy),
                                ptr(out.top_value), ptr<long long>(out.top_index), ptr(out.stats), rows, vocab, top, type_of(logits, "logits"), temperature, stream()));
  return out;
}

struct TokenLogProbs : torch::autograd::Function<TokenLogProbs> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const OptTensor& tokens_in, const OptTensor& mask_in, double temperature, int64_t top) {
    const Tensor tokens = tokens_in.value_or(Tensor()), mask = mask_in.value_or(Tensor());
    const Logprobs r = measure(logits, tokens, mask, temperature, top, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({logits, tokens, mask, r.stats});
    ctx->saved_data["temperature"] = temperature;
    variable_list out{r.entropy};
    if (tokens.defined()) out.push_back(r.log_prob);
    if (top) {
      out.push_back(r.top_value);
      out.push_back(r.top_index);
      ctx->mark_non_differentiable({r.top_value, r.top_index});
    }
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& gout) {
    once("token_log_probs");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &tokens = saved[1], &mask = saved[2], &stats = saved[3];
    const c10::cuda::CUDAGuard guard(logits.device());
    const int64_t vocab = logits.size(-1), rows = logits.numel() / vocab;
    const Rows x = rows_of(logits), m = mask.defined() ? rows_of(mask) : Rows{};
    const PerRow h = per_row(gout[0]), lp = tokens.defined() ? per_row(gout[1]) : PerRow{};
    const Tensor dx = empty_like_of(logits, logits.sizes(), logits.scalar_type());
    if (rows)
      check("mxk_token_logprob_bwd",
            mxk_token_logprob_bwd(x.t.data_ptr(), x.ld, bytes(m.t), m.ld, ptr<void>(tokens), tokens.defined() ? width_of(tokens) : 0, ptr(stats), ptr(lp.t), lp.ld, ptr(h.t),
                                  h.ld, dx.data_ptr(), rows, vocab, type_of(logits, "logits"), ctx->saved_data["temperature"].toDouble(), stream()));
    return {dx, Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

// -> (log_prob, entropy, top values, top indices), what was not asked for None
std::tuple<OptTensor, Tensor, OptTensor, OptTensor> token_log_probs(const Tensor& logits, const OptTensor& tokens_in, const OptTensor& mask_in, double temperature,
                                                                    int64_t top) {
  not_traced("token_log_probs");
  TORCH_CHECK_VALUE(logits.is_cuda(), "logits must be a CUDA tensor (memorax_b200 has no CPU path)");
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) > 0 && logits.size(-1) < 1 << 30, "logits must be (..., vocabulary), this below 2^30, got ", logits.sizes());
  type_of(logits, "logits");
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  TORCH_CHECK_VALUE(temperature >= 1e-30 && temperature <= 1e27, "temperature must be positive, from 1e-30 to 1e27, got ", temperature);
  TORCH_CHECK_VALUE(top >= 0 && top <= 32 && top <= logits.size(-1), "top must be between 0 and 32 and at most the vocabulary of ", logits.size(-1), ", got ", top);
  const c10::cuda::CUDAGuard guard(logits.device());
  Tensor tokens, mask;
  if (tokens_in && tokens_in->defined()) {
    TORCH_CHECK_VALUE(tokens_in->sizes() == lead, "tokens must be ", lead, " for logits of ", logits.sizes(), ", got ", tokens_in->sizes());
    tokens = tokens_of(*tokens_in, logits, "tokens");
  }
  if (mask_in && mask_in->defined()) {
    TORCH_CHECK_VALUE(mask_in->device() == logits.device(), "mask must be on ", logits.device());
    TORCH_CHECK_VALUE(mask_in->scalar_type() == at::kBool || mask_in->scalar_type() == at::kByte, "mask must be bool or uint8, got ", mask_in->scalar_type());
    mask = mask_in->expand(logits.sizes());      // raises where the shapes do not fit
  }
  if (with_node("token_log_probs", {logits})) {
    const variable_list out = TokenLogProbs::apply(logits, opt(tokens), opt(mask), temperature, top);
    const size_t t = tokens.defined() ? 2 : 1;
    return {tokens.defined() ? OptTensor(out[1]) : std::nullopt, out[0], top ? OptTensor(out[t]) : std::nullopt, top ? OptTensor(out[t + 1]) : std::nullopt};
  }
  const Logprobs r = measure(logits, tokens, mask, temperature, top, false);
  return {opt(r.log_prob), r.entropy, opt(r.top_value), opt(r.top_index)};
}

}  // namespace

void bind_tokens(pybind11::module_& m) {
  m.def("embedding", &embedding);
  m.def("token_log_probs", &token_log_probs);
}

}  // namespace mxk_host
