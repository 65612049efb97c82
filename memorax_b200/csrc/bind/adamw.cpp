// AdamW over a list of tensors: their moments, and a step.
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <torch/csrc/autograd/python_variable.h>

#include "common.h"

namespace mxk_host {
namespace {

constexpr int64_t kBlock = 256;   // elements of a block of 8-bit moments; every tensor's moments begin at a multiple

class AdamW {
 public:
  // master: a float32 copy of each 16-bit parameter, None for a float32 one, which takes the update itself
  AdamW(std::vector<Tensor> params, const std::optional<std::vector<OptTensor>>& master, int64_t bits) : params_(std::move(params)), bits_(bits) {
    TORCH_CHECK_VALUE(!params_.empty(), "params must not be empty");
    TORCH_CHECK_VALUE(bits == 8 || bits == 32, "state_bits must be 8 or 32, got ", bits);
    if (master) {
      TORCH_CHECK_VALUE(master->size() == params_.size(), "master has ", master->size(), " tensors for ", params_.size(), " parameters");
      for (const OptTensor& t : *master) master_.push_back(t.value_or(Tensor()));
    }
    device_ = params_[0].device();
    int64_t at = 0;
    std::vector<std::pair<uintptr_t, uintptr_t>> spans;
    for (size_t i = 0; i < params_.size(); ++i) {
      fits(params_[i], "a parameter");
      types_.push_back(type_of(params_[i], "a parameter"));
      dtypes_.push_back(params_[i].dtype());
      sizes_.push_back(params_[i].numel());
      span(spans, params_[i]);
      if (!master_.empty()) {
        TORCH_CHECK_VALUE(master_[i].defined() == (types_[i] != MXK_F32), "parameter ", i, " is ", params_[i].scalar_type(),
                          ": the 16-bit ones take a float32 copy each, float32 ones none");
      }
      if (!master_.empty() && master_[i].defined()) {
        fits(master_[i], "a float32 copy");
        TORCH_CHECK_VALUE(master_[i].scalar_type() == at::kFloat && master_[i].numel() == sizes_[i], "master must be float32 of the parameters' sizes");
        span(spans, master_[i]);
      }
      starts_.push_back(at);
      at += (sizes_[i] + kBlock - 1) / kBlock * kBlock;
    }
    std::sort(spans.begin(), spans.end());
    for (size_t i = 1; i < spans.size(); ++i) TORCH_CHECK_VALUE(spans[i - 1].second <= spans[i].first, "the same memory appears twice among the parameters");
    const c10::cuda::CUDAGuard guard(device_);
    const auto zeros = [&](int64_t n, at::ScalarType type) { return at::zeros({n}, at::TensorOptions().dtype(type).device(device_)); };
    m_ = zeros(at, bits == 8 ? at::kByte : at::kFloat);
    v_ = zeros(at, bits == 8 ? at::kByte : at::kFloat);
    if (bits == 8) {
      m_ = m_.view(at::kFloat8_e4m3fn);
      v_ = v_.view(at::kFloat8_e4m3fn);
      m_scale_ = zeros(at / kBlock, at::kFloat);
      v_scale_ = zeros(at / kBlock, at::kFloat);
    }
  }

  // grads: a list or tuple of tensors and None, or None for the parameters' own
  void step(const pybind11::object& grads, double lr, double b1, double b2, double eps, double weight_decay, double grad_scale, int64_t step, const OptTensor& count,
            const OptTensor& rate, const OptTensor& now) {
    const bool given_list = !grads.is_none();
    const pybind11::object list = given_list ? pybind11::reinterpret_steal<pybind11::object>(PySequence_Fast(grads.ptr(), "grads must be a list of tensors")) : pybind11::object();
    if (given_list && !list) throw pybind11::error_already_set();
    const Py_ssize_t many = given_list ? PySequence_Fast_GET_SIZE(list.ptr()) : 0;
    TORCH_CHECK_VALUE(!given_list || many == static_cast<Py_ssize_t>(params_.size()), "grads has ", many, " tensors for ", params_.size(), " parameters");
    const c10::cuda::CUDAGuard guard(device_);
    TORCH_CHECK(count || at::cuda::currentStreamCaptureStatusMayInitCtx() == at::cuda::CaptureStatus::None,
                "a captured step would replay its own number: build the optimiser with capturable=True");
    TORCH_CHECK_VALUE(!rate || (rate->scalar_type() == at::kFloat && rate->device() == device_ && rate->numel() == 1), "lr must be one float32 on ", device_);
    std::vector<Tensor> kept;                               // gradients that had to be laid out anew
    std::vector<size_t> changed;
    changed.reserve(params_.size());
    for (auto& group : groups_) group.clear();
    for (size_t i = 0; i < params_.size(); ++i) {
      const Tensor& p = params_[i];
      const Tensor* g = nullptr;
      if (given_list) {
        PyObject* const item = PySequence_Fast_GET_ITEM(list.ptr(), static_cast<Py_ssize_t>(i));
        if (item == Py_None) continue;
        TORCH_CHECK_TYPE(THPVariable_CheckExact(item) || THPVariable_Check(item), "gradient ", i, " is no tensor");
        g = &THPVariable_Unpack(item);
      } else {
        g = &p.grad();
      }
      if (!g->defined() || sizes_[i] == 0) continue;
      c10::TensorImpl &pi = *p.unsafeGetTensorImpl(), &gi = *g->unsafeGetTensorImpl();
      const auto type = pi.dtype();
      TORCH_CHECK_VALUE(pi.numel() == sizes_[i] && pi.is_contiguous() && pi.device() == device_ && type == dtypes_[i], "parameter ", i,
                        " has another size, type, layout or device than it had");
      TORCH_CHECK_VALUE(gi.layout() == at::kStrided, "gradient ", i, " is not dense");
      TORCH_CHECK_VALUE(gi.device() == device_ && gi.sizes() == pi.sizes(), "gradient ", i, " is ", g->sizes(), " on ", g->device(), " for a parameter of ", p.sizes(), " on ", device_);
      const bool own = gi.dtype() == type;
      TORCH_CHECK_VALUE(own || gi.dtype() == caffe2::TypeMeta::Make<float>(), "gradient ", i, " is ", g->scalar_type(), " for a parameter of ", p.scalar_type());
      if (!gi.is_contiguous() || g->is_neg()) {
        kept.push_back(dense(*g));
        g = &kept.back();
      }
      changed.push_back(i);
      groups_[2 * types_[i] + !own].push_back({pi.mutable_data(), g->unsafeGetTensorImpl()->data(), master_.empty() ? nullptr : ptr(master_[i]), sizes_[i], starts_[i]});
    }
    mxk_adamw_state state{m_.data_ptr(), v_.data_ptr(), ptr(m_scale_), ptr(v_scale_), now ? ptr(*now) : nullptr, static_cast<int>(bits_)};
    if (count) check("mxk_adamw_tick", mxk_adamw_tick(ptr<long long>(*count), ptr(*rate), b1, b2, weight_decay, ptr(*now), stream()));
    for (int k = 0; k < 6; ++k)
      if (!groups_[k].empty())
        check("mxk_adamw", mxk_adamw(groups_[k].data(), static_cast<int>(groups_[k].size()), k / 2, k % 2 ? MXK_F32 : k / 2, &state, lr, b1, b2, eps, weight_decay, grad_scale,
                                     step, stream()));
    const auto moved = [](const Tensor& t) {                 // what autograd has saved of it is not what it holds now
      if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
    };
    for (const size_t i : changed) {
      moved(params_[i]);
      if (!master_.empty() && master_[i].defined()) moved(master_[i]);
    }
  }

  // the tensors' pieces of a buffer laid out like the moments
  std::vector<Tensor> cut(const Tensor& flat) const {
    TORCH_CHECK_VALUE(flat.dim() == 1 && flat.is_contiguous() && flat.numel() == m_.numel(), "not a buffer of the moments' size");
    std::vector<Tensor> out;
    for (size_t i = 0; i < params_.size(); ++i) out.push_back(piece(flat, starts_[i], params_[i].sizes()));
    return out;
  }

  Tensor m_, v_, m_scale_, v_scale_;
  std::vector<int64_t> starts_;

 private:
  void fits(const Tensor& t, const char* name) const {
    TORCH_CHECK_VALUE(t.is_cuda() && t.device() == device_, name, " is on ", t.device(), ": all must be on one CUDA device (memorax_b200 has no CPU path)");
    TORCH_CHECK_VALUE(t.layout() == at::kStrided && t.is_contiguous() && !t.is_neg(), name, " of ", t.sizes(), " is not contiguous");
  }
  static void span(std::vector<std::pair<uintptr_t, uintptr_t>>& spans, const Tensor& t) {
    const uintptr_t from = reinterpret_cast<uintptr_t>(t.data_ptr());
    if (t.numel()) spans.emplace_back(from, from + t.nbytes());
  }

  std::vector<Tensor> params_, master_;
  std::vector<int64_t> sizes_;
  std::vector<int> types_;
  std::vector<caffe2::TypeMeta> dtypes_;
  std::vector<mxk_adamw_tensor> groups_[6];                 // of the step at hand: [parameter type][gradient type: its own, float32]
  int64_t bits_;
  c10::Device device_ = c10::Device(c10::kCUDA, 0);
};

}  // namespace

void bind_adamw(pybind11::module_& m) {
  pybind11::class_<AdamW>(m, "AdamW")
      .def(pybind11::init<std::vector<Tensor>, const std::optional<std::vector<OptTensor>>&, int64_t>())
      .def("step", &AdamW::step)
      .def("cut", &AdamW::cut)
      .def_readonly("m", &AdamW::m_)
      .def_readonly("v", &AdamW::v_)
      .def_property_readonly("m_scale", [](const AdamW& a) { return opt(a.m_scale_); })
      .def_property_readonly("v_scale", [](const AdamW& a) { return opt(a.v_scale_); })
      .def_readonly("starts", &AdamW::starts_);
}

}  // namespace mxk_host
