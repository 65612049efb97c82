// Norms of query and key heads with the position rotation.
#include "common.h"

namespace mxk_host {
namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// heads whose elements are neighbours
Tensor heads_of(const Tensor& t) {
  if (t.is_neg()) return t.resolve_neg().contiguous();
  return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous();
}
struct Setting {
  int64_t rot, interleaved, norm;
  double eps;
};
mxk_rotate arguments(const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const Tensor& positions, const Tensor& turns, const Setting& s) {
  mxk_rotate a{};
  const Tensor* x[2] = {&q, &k};
  const Tensor* w[2] = {&wq, &wk};
  for (int i = 0; i < 2; ++i) {
    a.side[i].x = x[i]->data_ptr();
    a.side[i].sb = x[i]->stride(0); a.side[i].st = x[i]->stride(1); a.side[i].sh = x[i]->stride(2);
    a.side[i].w = ptr<void>(*w[i]);
    a.side[i].heads = x[i]->size(2);
  }
  if (positions.defined()) {
    a.positions = positions.data_ptr();
    a.positions_bytes = positions.scalar_type() == at::kLong ? 8 : 4;
    // broadcast to (batch, steps), without a trip through the dispatcher
    const int64_t d = positions.dim();
    a.pt = d >= 1 && positions.size(d - 1) > 1 ? positions.stride(d - 1) : 0;
    a.pb = d == 2 && positions.size(0) > 1 ? positions.stride(0) : 0;
  }
  a.turns = ptr<unsigned long long>(turns);
  a.batch = q.size(0); a.steps = q.size(1);
  a.dim = q.size(3); a.rot = s.rot; a.interleaved = s.interleaved; a.norm = s.norm;
  a.type = type_of(q, "q");
  a.eps = s.eps;
  return a;
}
variable_list turn(const Tensor& q_in, const Tensor& k_in, const Tensor& wq, const Tensor& wk, const Tensor& positions, const Tensor& turns, const Setting& s) {
  const Tensor q = heads_of(q_in), k = heads_of(k_in);
  const Tensor yq = empty_like_of(q, q.sizes(), q.scalar_type()), yk = empty_like_of(k, k.sizes(), k.scalar_type());
  if (q.size(0) * q.size(1)) {
    mxk_rotate a = arguments(q, k, wq, wk, positions, turns, s);
    a.side[0].out = yq.data_ptr();
    a.side[1].out = yk.data_ptr();
    check("mxk_norm_rotate_fwd", mxk_norm_rotate_fwd(&a, stream()));
  }
  return {yq, yk};
}

struct NormRotate : torch::autograd::Function<NormRotate> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const OptTensor& wq, const OptTensor& wk, const OptTensor& positions,
                               const Tensor& turns, int64_t rot, bool interleaved, int64_t norm, double eps) {
    ctx->set_materialize_grads(false);
    const Setting s{rot, interleaved, norm, eps};
    const Tensor w0 = wq ? dense(*wq) : Tensor(), w1 = wk ? dense(*wk) : Tensor(), p = positions.value_or(Tensor());
    ctx->save_for_backward({q, k, w0, w1, p, turns});
    ctx->saved_data["rot"] = rot;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["norm"] = norm;
    ctx->saved_data["eps"] = eps;
    return turn(q, k, w0, w1, p, turns, s);
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& gout) {
    once("norm_rotate");
    const variable_list saved = ctx->get_saved_variables();
    const Tensor q = heads_of(saved[0]), k = heads_of(saved[1]);
    const Tensor &wq = saved[2], &wk = saved[3];
    const c10::cuda::CUDAGuard guard(q.device());
    const Setting s{ctx->saved_data["rot"].toInt(), ctx->saved_data["interleaved"].toBool(), ctx->saved_data["norm"].toInt(), ctx->saved_data["eps"].toDouble()};
    const auto cotangent = [](const Tensor& g, const Tensor& x) {
      if (!g.defined()) return empty_like_of(x, x.sizes(), x.scalar_type()).zero_();
      return heads_of(g.scalar_type() == x.scalar_type() ? g : g.to(x.scalar_type()));
    };
    const Tensor gq = cotangent(gout[0], q), gk = cotangent(gout[1], k);
    variable_list grads(10);
    grads[0] = empty_like_of(q, q.sizes(), q.scalar_type());
    grads[1] = empty_like_of(k, k.sizes(), k.scalar_type());
    const bool weights = wq.defined();
    if (weights) {
      grads[2] = empty_like_of(wq, wq.sizes(), wq.scalar_type());
      grads[3] = empty_like_of(wk, wk.sizes(), wk.scalar_type());
    }
    if (q.size(0) * q.size(1) == 0) {
      if (weights) grads[2].zero_(), grads[3].zero_();
      return grads;
    }
    mxk_rotate a = arguments(q, k, wq, wk, saved[4], saved[5], s);
    const Tensor* g[2] = {&gq, &gk};
    for (int i = 0; i < 2; ++i) {
      a.side[i].dy = g[i]->data_ptr();
      a.side[i].db = g[i]->stride(0); a.side[i].dt = g[i]->stride(1); a.side[i].dh = g[i]->stride(2);
      a.side[i].out = grads[i].data_ptr();
    }
    const size_t ws_bytes = weights ? mxk_norm_rotate_bwd_workspace_bytes(a.dim) : 0;
    const Tensor ws = weights ? scratch(q, ws_bytes) : Tensor();
    check("mxk_norm_rotate_bwd", mxk_norm_rotate_bwd(&a, ptr<void>(grads[2]), ptr<void>(grads[3]), ptr<void>(ws), ws_bytes, stream()));
    return grads;
  }
};

std::tuple<Tensor, Tensor> norm_rotate(const Tensor& q, const Tensor& k, const Tensor& turns, const OptTensor& positions_in, const OptTensor& wq, const OptTensor& wk,
                                       bool interleaved, int64_t norm, double eps) {
  not_traced("norm_rotate");
  TORCH_CHECK_VALUE(q.is_cuda() && k.is_cuda(), "q and k must be CUDA tensors (memorax_b200 has no CPU path)");
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3) && q.size(2) > 0 && k.size(2) > 0,
                    "q and k must be (batch, steps, heads, head_dim) of the same batch, steps and head_dim, got ", q.sizes(), " and ", k.sizes());
  TORCH_CHECK_VALUE(q.scalar_type() == k.scalar_type() && q.device() == k.device(), "q and k must be of one type and device");
  type_of(q, "q");
  const int64_t dim = q.size(3), rot = 2 * turns.numel();
  TORCH_CHECK_VALUE(dim % 2 == 0 && dim >= 2 && dim <= 512, "head_dim must be even and at most 512, got ", dim);
  TORCH_CHECK_VALUE(q.size(2) <= 65535 && k.size(2) <= 65535, "at most 65535 heads, got ", q.size(2), " and ", k.size(2));
  TORCH_CHECK_VALUE(eps >= 0, "eps must not be negative, got ", eps);
  TORCH_CHECK_VALUE(turns.device() == q.device(), "the plan is on ", turns.device(), ", q on ", q.device());
  TORCH_CHECK_VALUE(rot >= 2 && rot <= dim, "the plan rotates ", rot, " elements of heads of ", dim);
  TORCH_CHECK_VALUE(turns.scalar_type() == at::kLong && turns.is_contiguous(), "the plan's turns must be int64");
  const bool weights = wq && wq->defined();
  TORCH_CHECK_VALUE(weights == (wk && wk->defined()), "weights are given for both queries and keys, or for none");
  TORCH_CHECK_VALUE(!weights || norm == MXK_NORM_RMS, "weights belong to the rms norm");
  if (weights)
    for (const Tensor& w : {*wq, *wk})
      TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == dim && w.scalar_type() == q.scalar_type() && w.device() == q.device(), "weights must be (", dim,
                        ") of q's type and device, got ", w.sizes(), " ", w.scalar_type());
  const c10::cuda::CUDAGuard guard(q.device());
  Tensor positions;
  if (positions_in && positions_in->defined()) {
    positions = *positions_in;
    TORCH_CHECK_VALUE(positions.device() == q.device() && (positions.scalar_type() == at::kLong || positions.scalar_type() == at::kInt),
                      "positions must be int32 or int64 on ", q.device(), ", got ", positions.scalar_type(), " on ", positions.device());
    const int64_t d = positions.dim(), last = d >= 1 ? positions.size(d - 1) : 1, first = d == 2 ? positions.size(0) : 1;
    TORCH_CHECK_VALUE(d <= 2 && (last == 1 || last == q.size(1)) && (first == 1 || first == q.size(0)), "positions must broadcast to (", q.size(0), ", ", q.size(1), "), got ",
                      positions.sizes());
  }
  if (with_node("norm_rotate", {q, k, weights ? *wq : Tensor(), weights ? *wk : Tensor()})) {
    const variable_list out = NormRotate::apply(q, k, weights ? wq : std::nullopt, weights ? wk : std::nullopt, opt(positions), turns, rot, interleaved, norm, eps);
    return {out[0], out[1]};
  }
  const variable_list out = turn(q, k, weights ? dense(*wq) : Tensor(), weights ? dense(*wk) : Tensor(), positions, turns, {rot, interleaved, norm, eps});
  return {out[0], out[1]};
}

}  // namespace

void bind_rotate(pybind11::module_& m) { m.def("norm_rotate", &norm_rotate); }

}  // namespace mxk_host
