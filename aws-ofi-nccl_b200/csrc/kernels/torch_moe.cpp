// The operators of a mixture-of-experts block on one GPU as native layers: the norm with its output in 8 bits, tokens sorted by expert and back,
// and the optimizer's step over many tensors. They run on the tensors' device, whichever is current, and on its current stream.
#include <algorithm>
#include <climits>
#include <functional>
#include <map>
#include <utility>
#include <vector>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>

#include "torch_layer.h"

namespace {

using namespace b200torch;
using c10::cuda::CUDAGuard;

void launched(int kernels = 1) { g_launches.fetch_add(kernels, std::memory_order_relaxed); }
// A new tensor beside `like`, without the dispatcher, which takes as long again as the allocation
Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt);
}
bool same_device(const Tensor& a, const Tensor& b) { return a.is_cuda() && a.device() == b.device(); }
// A dual tensor may require no gradient: its tangent would be lost without a word, and what is lost counts as zero.
void refuse_tangents(std::initializer_list<const Tensor*> inputs, const char* what) {
  for (const Tensor* t : inputs)   // torch has one level of them
    if (t && t->defined() && t->_fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode()) raise(PyExc_RuntimeError, what);
}
void refuse_gradients(std::initializer_list<const Tensor*> inputs, const char* what) {
  refuse_tangents(inputs, "8-bit outputs have no forward-mode derivative");
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor* t : inputs) require(!t || !t->requires_grad(), what);
}
// A matrix of rows that the kernels can step through: as it is where its rows are contiguous, else a copy
Tensor rows_with_pitch(const Tensor& t) { return t.stride(1) == 1 || t.size(1) == 1 ? t : t.contiguous(); }
int64_t pitch_of(const Tensor& t) { return t.size(0) <= 1 ? t.size(1) : t.stride(0); }

// ------------------------------------------------------------------ RMSNorm with its output in 8 bits
variable_list rmsnorm_fp8(const Tensor& x, const c10::optional<Tensor>& res, const Tensor& weight, double eps, int64_t group) {
  require(bf16_cuda(x) && x.dim() >= 1, "x is a bfloat16 CUDA tensor with a last dimension");
  const int64_t H = x.size(-1);
  const int64_t T = rows_of(x, H);
  require(!res || (bf16_cuda(*res) && same_device(*res, x) && res->sizes() == x.sizes()), "the residual is a bfloat16 CUDA tensor like x");
  require(bf16_cuda(weight) && same_device(weight, x) && weight.is_contiguous() && weight.numel() == H, "the weight is a bfloat16 CUDA tensor of one row");
  require(H % 8 == 0 && H <= 16384, "rows are of a multiple of 8 elements, at most 16384");
  require(group == 0 || (group == 128 && H % 128 == 0), "a scale is one row's (group 0) or 128 columns' (group 128) of rows that are a multiple of them");
  refuse_gradients({&x, res ? &*res : nullptr, &weight}, "rmsnorm_fp8 has no gradient: call it under torch.no_grad()");
  auto matrix = [&](const Tensor& t) {   // rows of a pitch that the kernel's vectors fit
    const Tensor m = rows_with_pitch(t.dim() == 2 ? t : t.reshape({T, H}));
    return reinterpret_cast<uintptr_t>(m.data_ptr()) % 16 || pitch_of(m) % 8 ? m.clone(at::MemoryFormat::Contiguous) : m;
  };
  const CUDAGuard guard(x.device());
  const Tensor xm = matrix(x), rm = res ? matrix(*res) : Tensor(), w = rows16(weight);
  auto shape = x.sizes().vec();
  Tensor q = fresh(shape, at::kFloat8_e4m3fn, x), h = res ? fresh(shape, at::kBFloat16, x) : x;
  if (group)
    shape.back() = H / group;
  else
    shape.pop_back();
  Tensor scale = fresh(shape, at::kFloat, x);
  if (T) launched();
  check(b200_rmsnorm_fp8(xm.data_ptr(), pitch_of(xm), res ? rm.data_ptr() : nullptr, res ? pitch_of(rm) : 0, res ? h.data_ptr() : nullptr, w.data_ptr(),
                         q.data_ptr(), scale.data_ptr<float>(), T, static_cast<int>(H), static_cast<float>(eps), static_cast<int>(group), stream()),
        "b200_rmsnorm_fp8");
  return {q, scale, h};
}

// ------------------------------------------------------------------ tokens sorted by expert and back
variable_list expert_order(const Tensor& idx, int64_t experts) {
  require(idx.is_cuda() && idx.dim() == 2 && idx.is_contiguous() && (idx.scalar_type() == at::kInt || idx.scalar_type() == at::kLong),
          "the choices are a contiguous [tokens, k] CUDA matrix of 32-bit or 64-bit integers");
  require(idx.size(1) > 0, "a token has at least one choice");
  require(experts >= 1 && experts <= 1024, "there are 1 to 1024 experts");
  require(idx.numel() <= INT_MAX, "rows are numbers of 32 bits");
  const CUDAGuard guard(idx.device());
  Tensor row_of = fresh(idx.sizes(), at::kInt, idx), offsets = fresh({experts + 1}, at::kInt, idx);
  launched();
  check(b200_expert_order(idx.data_ptr(), idx.scalar_type() == at::kLong, idx.numel(), static_cast<int>(experts), row_of.data_ptr<int>(),
                          offsets.data_ptr<int>(), stream()),
        "b200_expert_order");
  return {row_of, offsets};
}

void check_rows(const Tensor& row_of, const Tensor& like) {
  require(row_of.scalar_type() == at::kInt && same_device(row_of, like) && row_of.dim() == 2 && row_of.is_contiguous() && row_of.size(1) > 0 &&
              row_of.numel() <= INT_MAX,
          "row_of is the contiguous [tokens, k] matrix that expert_order made, on the rows' device");
}

Tensor gather(const Tensor& x, const Tensor& row_of, const Tensor& scale, Tensor* row_scale) {
  const CUDAGuard guard(x.device());
  const int64_t T = row_of.size(0), k = row_of.size(1), H = x.size(1), elem = x.element_size();
  const Tensor m = rows_with_pitch(x);
  Tensor rows = fresh({T * k, H}, x.scalar_type(), x);
  int groups = 0;
  if (scale.defined()) {
    groups = static_cast<int>(scale.dim() == 1 ? 1 : scale.size(1));
    auto shape = scale.sizes().vec();
    shape[0] = T * k;
    *row_scale = fresh(shape, at::kFloat, scale);
  }
  if (T) launched();
  check(b200_permute_rows(m.data_ptr(), pitch_of(m) * elem, rows.data_ptr(), row_of.data_ptr<int>(), groups ? scale.data_ptr<float>() : nullptr,
                          groups ? row_scale->data_ptr<float>() : nullptr, groups, T, static_cast<int>(k), H * elem, static_cast<int>(elem), stream()),
        "b200_permute_rows");
  return rows;
}
Tensor weighted_sum(const Tensor& rows, const Tensor& row_of, const float* w) {
  const CUDAGuard guard(rows.device());
  const int64_t T = row_of.size(0), k = row_of.size(1), H = rows.size(1);
  const Tensor m = rows_with_pitch(rows);
  Tensor out = fresh({T, H}, rows.scalar_type(), rows);
  if (T) launched();
  check(b200_unpermute_rows(m.data_ptr(), pitch_of(m), w, row_of.data_ptr<int>(), out.data_ptr(), T, static_cast<int>(k), static_cast<int>(H),
                            rows.scalar_type() == at::kFloat, stream()),
        "b200_unpermute_rows");
  return out;
}

// Each one's gradient is the other one, so that both have derivatives of any order (a backward pass that is to be differentiated runs with gradients on).
constexpr const char* NO_TANGENTS_THERE = "permute_tokens has no forward-mode derivative";
constexpr const char* NO_TANGENTS_BACK = "unpermute_tokens has no forward-mode derivative";
Tensor permute(const Tensor& x, const Tensor& row_of);
Tensor unpermute(const Tensor& rows, const Tensor& row_of, const c10::optional<Tensor>& w);

// rows[row_of[t][j]] = x[t]; its gradient is the sum over a token's rows
struct Permute : public Function<Permute> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& row_of) {
    ctx->save_for_backward({row_of});
    return gather(x, row_of, Tensor(), nullptr);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return on_engine_thread([&]() -> variable_list { return {unpermute(grads[0], ctx->get_saved_variables()[0], c10::nullopt), Tensor()}; });
  }
};

// out[t] = sum over j of w[t][j] * rows[row_of[t][j]]; rows are kept for the weights' gradient alone
struct Unpermute : public Function<Unpermute> {
  static Tensor forward(AutogradContext* ctx, const Tensor& rows, const Tensor& row_of, const c10::optional<Tensor>& w) {
    const Tensor weights = w ? w->contiguous() : Tensor();
    ctx->save_for_backward({row_of, weights, w && w->requires_grad() ? rows : Tensor()});
    return weighted_sum(rows, row_of, w ? weights.data_ptr<float>() : nullptr);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return on_engine_thread([&]() -> variable_list {
      const auto saved = ctx->get_saved_variables();
      const Tensor &row_of = saved[0], &w = saved[1], &dout = grads[0];
      refuse_tangents({&dout, &w, &saved[2]}, NO_TANGENTS_BACK);
      if (!w.defined()) return {permute(dout, row_of), Tensor(), Tensor()};
      if (at::GradMode::is_enabled()) raise(PyExc_RuntimeError, "a weighted unpermute_tokens has no second derivative");
      const CUDAGuard guard(dout.device());
      const int64_t T = row_of.size(0), k = row_of.size(1), H = dout.size(1);
      const Tensor d = dout.contiguous(), rows = saved[2].defined() ? rows_with_pitch(saved[2]) : Tensor();
      Tensor drows, dw;
      if (ctx->needs_input_grad(0)) drows = fresh({T * k, H}, dout.scalar_type(), dout);
      if (rows.defined()) dw = fresh({T, k}, at::kFloat, w);
      if (T && (drows.defined() || dw.defined())) launched();
      check(b200_unpermute_rows_bwd(d.data_ptr(), rows.defined() ? rows.data_ptr() : nullptr, rows.defined() ? pitch_of(rows) : H, w.data_ptr<float>(),
                                    row_of.data_ptr<int>(), drows.defined() ? drows.data_ptr() : nullptr, dw.defined() ? dw.data_ptr<float>() : nullptr,
                                    T, static_cast<int>(k), static_cast<int>(H), dout.scalar_type() == at::kFloat, stream()),
            "b200_unpermute_rows_bwd");
      return {drows, Tensor(), dw};
    });
  }
};

Tensor permute(const Tensor& x, const Tensor& row_of) {
  refuse_tangents({&x}, NO_TANGENTS_THERE);
  return at::GradMode::is_enabled() && x.requires_grad() ? Permute::apply(x, row_of) : gather(x, row_of, Tensor(), nullptr);
}
Tensor unpermute(const Tensor& rows, const Tensor& row_of, const c10::optional<Tensor>& w) {
  refuse_tangents({&rows, w ? &*w : nullptr}, NO_TANGENTS_BACK);
  if (at::GradMode::is_enabled() && (rows.requires_grad() || (w && w->requires_grad()))) return Unpermute::apply(rows, row_of, w);
  const Tensor weights = w ? w->contiguous() : Tensor();
  return weighted_sum(rows, row_of, w ? weights.data_ptr<float>() : nullptr);
}

bool of_32_or_bf16(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat; }

variable_list permute_tokens(const Tensor& x, const Tensor& row_of, const c10::optional<Tensor>& scale) {
  const bool codes = x.scalar_type() == at::kFloat8_e4m3fn;
  require(x.is_cuda() && x.dim() == 2 && (codes || of_32_or_bf16(x)), "x is a bfloat16, float32 or float8_e4m3fn CUDA matrix");
  check_rows(row_of, x);
  require(x.size(0) == row_of.size(0), "x has a row for every token");
  require(x.size(1) > 0 && x.size(1) <= 1 << 29, "rows are neither empty nor of more than 2^29 elements");
  require(!scale || codes, "scales go with 8-bit rows");
  if (!codes) return {permute(x, row_of)};
  require(!scale || (scale->scalar_type() == at::kFloat && same_device(*scale, x) && scale->is_contiguous() && (scale->dim() == 1 || scale->dim() == 2) &&
                     scale->size(0) == x.size(0) && (scale->dim() == 1 || (scale->size(1) > 0 && scale->size(1) <= x.size(1)))),
          "scales are a contiguous float32 CUDA tensor of one row, or one number, for every row of x");
  refuse_gradients({&x, scale ? &*scale : nullptr}, "8-bit rows and their scales have no gradient: call it under torch.no_grad()");
  Tensor row_scale;
  const Tensor rows = gather(x, row_of, scale ? *scale : Tensor(), &row_scale);
  if (scale) return {rows, row_scale};
  return {rows};
}
Tensor unpermute_tokens(const Tensor& rows, const Tensor& row_of, const c10::optional<Tensor>& w) {
  require(rows.is_cuda() && rows.dim() == 2 && of_32_or_bf16(rows), "the rows are a bfloat16 or float32 CUDA matrix");
  check_rows(row_of, rows);
  require(rows.size(0) == row_of.numel(), "there is a row for every choice");
  require(rows.size(1) > 0 && rows.size(1) <= 1 << 29, "rows are neither empty nor of more than 2^29 elements");
  require(!w || (w->scalar_type() == at::kFloat && same_device(*w, rows) && w->sizes() == row_of.sizes()),
          "the weights are a float32 CUDA tensor of row_of's shape");
  return unpermute(rows, row_of, w);
}

// ------------------------------------------------------------------ AdamW over many tensors
using Range = std::pair<uintptr_t, uintptr_t>;
// Whether no two of the written ranges share a byte, nor one of them with one that is read, which may share theirs. A list of tensors mostly lies in
// order, so lists are sorted by themselves, if at all, and merged.
bool apart(std::initializer_list<std::vector<Range>*> lists, std::vector<Range>& read) {
  std::vector<Range> all;
  size_t total = 0;
  for (const std::vector<Range>* r : lists) total += r->size();
  all.reserve(total);
  auto sort = [](std::vector<Range>& r) {
    if (!std::is_sorted(r.begin(), r.end())) std::sort(r.begin(), r.end());
  };
  for (std::vector<Range>* r : lists) {
    sort(*r);
    const size_t before = all.size();
    all.insert(all.end(), r->begin(), r->end());
    if (before && !r->empty() && all[before] < all[before - 1]) std::inplace_merge(all.begin(), all.begin() + before, all.end());
  }
  for (size_t i = 1; i < all.size(); ++i)
    if (all[i].first < all[i - 1].second) return false;
  sort(read);
  auto w = all.begin();
  for (const Range& r : read) {
    while (w != all.end() && w->second <= r.first) ++w;
    if (w != all.end() && w->first < r.second) return false;
  }
  return true;
}

// A sequence of tensors, read as they lie in a tuple, which keeps them: converted to a vector they take 50 ns each, and a step has up to seven for
// every parameter. Needs the interpreter lock.
class Tensors {
 public:
  Tensors(const py::object& sequence, const char* what, bool may_lack) {
    if (sequence.is_none()) return;
    items_ = py::reinterpret_steal<py::object>(PySequence_Tuple(sequence.ptr()));
    if (!items_) throw py::error_already_set();
    for (size_t i = 0; i < size(); ++i) {
      PyObject* const item = PyTuple_GET_ITEM(items_.ptr(), i);
      if (!(may_lack && item == Py_None) && !THPVariable_Check(item)) raise(PyExc_TypeError, what);
    }
  }
  explicit operator bool() const { return static_cast<bool>(items_); }
  size_t size() const { return items_ ? PyTuple_GET_SIZE(items_.ptr()) : 0; }
  bool has(size_t i) const { return PyTuple_GET_ITEM(items_.ptr(), i) != Py_None; }
  const Tensor& operator[](size_t i) const { return THPVariable_Unpack(PyTuple_GET_ITEM(items_.ptr(), i)); }

 private:
  py::object items_;
};

void adamw_step_many(const py::object& param_list, const py::object& grad_list, const py::object& m_list, const py::object& v_list,
                     const py::object& m_scale_list, const py::object& v_scale_list, const py::object& master_list, const std::vector<double>& decay,
                     double lr, double beta1, double beta2, double eps, const py::object& step_or_steps, double grad_scale, bool zero_grad) {
  const Tensors params(param_list, "parameters are tensors", false), grads(grad_list, "gradients are tensors or None", true);
  const Tensors m(m_list, "moments are tensors", false), v(v_list, "moments are tensors", false);
  const Tensors m_scale(m_scale_list, "scales are tensors", false), v_scale(v_scale_list, "scales are tensors", false);
  const Tensors master(master_list, "master copies are tensors or None", true);
  const size_t count = params.size();
  require(grads.size() == count && m.size() == count && v.size() == count && (!master || master.size() == count),
          "gradients, moments and master copies are as many as the parameters");
  require(decay.size() == count, "the weight decay is a number, or one for every parameter");
  const bool one_step = PyIndex_Check(step_or_steps.ptr());
  int64_t step = 1;
  std::vector<int64_t> steps;
  try {
    if (one_step)
      step = step_or_steps.cast<int64_t>();
    else
      steps = step_or_steps.cast<std::vector<int64_t>>();
  } catch (const py::cast_error&) {
    raise(PyExc_TypeError, "the step is a whole number, or a list of one for every parameter");
  }
  require(one_step || steps.size() == count, "the step is a number, or one for every parameter");
  require(step >= 1 && std::all_of(steps.begin(), steps.end(), [](int64_t s) { return s >= 1; }), "steps count from one");
  require(lr >= 0 && beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0, "lr and eps are not negative, the betas lie in [0, 1)");
  if (count == 0) return;
  const bool eight = m[0].scalar_type() == at::kFloat8_e4m3fn;
  require(eight == static_cast<bool>(m_scale) && eight == static_cast<bool>(v_scale),
          "scales of both moments go with 8-bit moments, and only with those");
  require(!eight || (m_scale.size() == count && v_scale.size() == count), "scales are as many as the parameters");
  const auto state = eight ? at::kFloat8_e4m3fn : at::kFloat;
  const c10::Device device = params[0].device();
  require(device.is_cuda(), "parameters are CUDA tensors");
  auto fits = [&](const Tensor& t, at::ScalarType type, int64_t n) {
    return t.scalar_type() == type && t.device() == device && t.numel() == n && t.is_contiguous();
  };
  std::vector<B200AdamwTensor> list;
  std::vector<int64_t> step_of;   // where parameters have steps of their own
  std::vector<Range> of_p, of_g, of_m, of_v, of_ms, of_vs, of_master, read;   // all but the last are written
  std::vector<const Tensor*> changed;
  list.reserve(count);
  changed.reserve(4 * count);
  auto note = [count](std::vector<Range>& to, const Tensor& t) -> void* {
    void* const data = t.data_ptr();
    if (to.empty()) to.reserve(count);
    const uintptr_t at = reinterpret_cast<uintptr_t>(data);
    to.emplace_back(at, at + t.nbytes());
    return data;
  };
  auto write = [&](std::vector<Range>& to, const Tensor& t) -> void* {
    void* const data = note(to, t);
    changed.push_back(&t);
    return data;
  };
  for (size_t i = 0; i < count; ++i) {
    const Tensor& p = params[i];
    const int64_t n = p.numel();
    require(of_32_or_bf16(p) && p.device() == device && p.is_contiguous(), "parameters are contiguous bfloat16 or float32 tensors of one device");
    require(fits(m[i], state, n) && fits(v[i], state, n), "moments are contiguous, of their parameter's size and all float32 or all float8_e4m3fn");
    if (eight)
      require(fits(m_scale[i], at::kFloat, (n + 255) / 256) && fits(v_scale[i], at::kFloat, (n + 255) / 256),
              "scales are contiguous float32 tensors of one number for every 256 elements");
    const Tensor* copy = master && master.has(i) ? &master[i] : nullptr;
    require(!copy || (p.scalar_type() == at::kBFloat16 && fits(*copy, at::kFloat, n)), "a master copy is a contiguous float32 tensor beside a bfloat16 parameter");
    if (!grads.has(i)) continue;   // took no part in this step
    const Tensor& g = grads[i];
    require(of_32_or_bf16(g) && fits(g, g.scalar_type(), n), "gradients are contiguous bfloat16 or float32 tensors of their parameter's size");
    if (n == 0) continue;
    B200AdamwTensor t{};
    t.p = write(of_p, p);
    t.g = zero_grad ? write(of_g, g) : note(read, g);
    t.m = write(of_m, m[i]);
    t.v = write(of_v, v[i]);
    if (eight) {
      t.m_scale = static_cast<float*>(write(of_ms, m_scale[i]));
      t.v_scale = static_cast<float*>(write(of_vs, v_scale[i]));
    }
    if (copy) t.master = static_cast<float*>(write(of_master, *copy));
    t.n = n;
    t.keep = static_cast<float>(1.0 - lr * decay[i]);
    t.p_fp32 = p.scalar_type() == at::kFloat;
    t.g_fp32 = g.scalar_type() == at::kFloat;
    list.push_back(t);
    if (!one_step) step_of.push_back(steps[i]);
  }
  require(apart({&of_p, &of_g, &of_m, &of_v, &of_ms, &of_vs, &of_master}, read),
          "parameters, moments, scales, master copies and gradients that are zeroed share no memory, with each other or with a gradient that is read: "
          "is a parameter in the list twice?");
  if (list.empty()) return;
  const CUDAGuard guard(device);
  int launches = 0, rc = 0;
  {
    py::gil_scoped_release other_threads_run;   // while the launch waits for room in the queue
    auto launch = [&](const std::vector<B200AdamwTensor>& some, int64_t s) {
      int n = 0;
      rc = b200_adamw_many(some.data(), static_cast<int>(some.size()), eight ? 8 : 32, lr, beta1, beta2, eps, s, grad_scale, zero_grad, &n, stream());
      launches += n;
    };
    if (std::adjacent_find(step_of.begin(), step_of.end(), std::not_equal_to<>()) == step_of.end()) {
      launch(list, one_step ? step : step_of[0]);
    } else {
      std::map<int64_t, std::vector<B200AdamwTensor>> by_step;
      for (size_t i = 0; i < list.size(); ++i) by_step[step_of[i]].push_back(list[i]);
      for (const auto& [s, some] : by_step)
        if (rc == 0) launch(some, s);
    }
  }
  launched(launches);
  for (const Tensor* t : changed)
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();   // a graph that kept the old values is told
  check(rc, "b200_adamw_many");
}

// The current stream works on these tensors: memory of theirs that another stream allocated is not handed out again before it has.
void used_here(const py::object& list) {
  const Tensors tensors(list, "what is used is tensors or None", true);
  for (size_t i = 0; i < tensors.size(); ++i)
    if (tensors.has(i) && tensors[i].is_cuda() && tensors[i].has_storage())
      c10::cuda::CUDACachingAllocator::recordStream(tensors[i].storage().data_ptr(), c10::cuda::getCurrentCUDAStream(tensors[i].device().index()));
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(b200ops, m) {
  m.def("rmsnorm_fp8(Tensor x, Tensor? res, Tensor weight, float eps, int group) -> Tensor[]", rmsnorm_fp8);
  m.def("expert_order(Tensor topk_idx, int experts) -> Tensor[]", expert_order);
  m.def("permute_tokens(Tensor x, Tensor row_of, Tensor? scale) -> Tensor[]", permute_tokens);
  m.def("unpermute_tokens(Tensor rows, Tensor row_of, Tensor? topk_w) -> Tensor", unpermute_tokens);
}

void b200torch::bind_moe(py::module_& m) {
  m.def("rmsnorm_fp8", torch::wrap_pybind_function_no_gil([](const Tensor& x, const c10::optional<Tensor>& res, const Tensor& w, double eps, int64_t group) {
          return traced_or_direct("b200ops::rmsnorm_fp8", rmsnorm_fp8, x, res, w, eps, group);
        }));
  m.def("expert_order", torch::wrap_pybind_function_no_gil([](const Tensor& idx, int64_t experts) {
          return traced_or_direct("b200ops::expert_order", expert_order, idx, experts);
        }));
  m.def("permute_tokens", torch::wrap_pybind_function_no_gil([](const Tensor& x, const Tensor& row_of, const c10::optional<Tensor>& scale) {
          return traced_or_direct("b200ops::permute_tokens", permute_tokens, x, row_of, scale);
        }));
  m.def("unpermute_tokens", torch::wrap_pybind_function_no_gil([](const Tensor& rows, const Tensor& row_of, const c10::optional<Tensor>& w) {
          return traced_or_direct("b200ops::unpermute_tokens", unpermute_tokens, rows, row_of, w);
        }));
  m.def("used_here", torch::wrap_pybind_function(used_here));
  m.def("adamw_step_many", torch::wrap_pybind_function(adamw_step_many));
}
