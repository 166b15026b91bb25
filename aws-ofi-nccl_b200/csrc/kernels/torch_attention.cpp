// Attention with a sliding window and sinks as a native layer. It runs on the tensors' device, whichever is current, and on its current stream.
#include <algorithm>
#include <climits>
#include <cmath>

#include "torch_layer.h"

namespace {

using namespace b200torch;

constexpr const char* NO_TANGENTS = "attention has no forward-mode derivative";

// [B][S][heads][hd] that TMA can step through: as it is where a head's elements are contiguous and the rest lies on 16-byte boundaries, else a copy.
Tensor boxed(const Tensor& t) {
  bool fits = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int d = 0; d < 3; ++d) fits = fits && (t.size(d) == 1 || (t.stride(d) > 0 && t.stride(d) % 8 == 0));
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}
B200AttnTensor described(const Tensor& t) { return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)}; }

struct Window {
  int64_t window, sinks;
  double scale;
};
B200AttnArgs arguments(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, const Window& w) {
  B200AttnArgs a{};
  a.q = described(q), a.k = described(k), a.v = described(v);
  a.lengths = lengths.defined() ? lengths.data_ptr<int>() : nullptr;
  a.B = static_cast<int>(q.size(0)), a.S = static_cast<int>(q.size(1)), a.nq = static_cast<int>(q.size(2)), a.nkv = static_cast<int>(k.size(2));
  a.hd = static_cast<int>(q.size(3));
  // more tokens than there are are all of them
  a.window = static_cast<int>(std::min<int64_t>(w.window, INT_MAX)), a.sinks = static_cast<int>(std::min<int64_t>(w.sinks, INT_MAX));
  a.scale = static_cast<float>(w.scale);
  return a;
}
Tensor row_numbers(const Tensor& q) {   // a number for every row of every head, in whole tiles
  return fresh({q.size(0), q.size(2), (q.size(1) + 127) / 128 * 128}, at::kFloat, q);
}
// out, and what a backward pass needs of it: lse, and with `rest` what its rounding left
Tensor forward_of(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& lengths, const Window& w, Tensor& lse, Tensor* rest) {
  const CUDAGuard guard(q.device());
  Tensor out = fresh(q.sizes(), at::kBFloat16, q);
  lse = row_numbers(q);
  if (rest) *rest = fresh(q.sizes(), at::kByte, q);
  if (q.numel() == 0) return out;
  B200AttnArgs a = arguments(q, k, v, lengths, w);
  a.out = out.data_ptr(), a.rest = rest ? rest->data_ptr() : nullptr, a.lse = lse.data_ptr<float>();
  launched();
  check(b200_attention_fwd(&a, stream()), "b200_attention_fwd");
  return out;
}

struct Attention : public Function<Attention> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v, const c10::optional<Tensor>& lengths, int64_t window,
                        int64_t sinks, double scale) {
    const Tensor qb = boxed(q), kb = boxed(k), vb = boxed(v), n = lengths ? *lengths : Tensor();
    Tensor lse, rest, out = forward_of(qb, kb, vb, n, {window, sinks, scale}, lse, &rest);
    ctx->save_for_backward({qb, kb, vb, n, out, lse, rest});
    ctx->saved_data["window"] = window, ctx->saved_data["sinks"] = sinks, ctx->saved_data["scale"] = scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    return on_engine_thread([&]() -> variable_list {
      const auto saved = ctx->get_saved_variables();
      const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &lengths = saved[3], &out = saved[4], &lse = saved[5], &rest = saved[6];
      refuse_tangents({&grads[0], &q, &k, &v}, NO_TANGENTS);
      if (at::GradMode::is_enabled()) raise(PyExc_RuntimeError, "attention has no second derivative");
      const CUDAGuard guard(q.device());
      const Tensor dout = boxed(grads[0]);
      Tensor dq, dk, dv;
      if (ctx->needs_input_grad(0)) dq = fresh(q.sizes(), at::kBFloat16, q);
      if (ctx->needs_input_grad(1) || ctx->needs_input_grad(2)) dk = fresh(k.sizes(), at::kBFloat16, k), dv = fresh(v.sizes(), at::kBFloat16, v);
      if (q.numel()) {
        B200AttnArgs a =
            arguments(q, k, v, lengths, {ctx->saved_data["window"].toInt(), ctx->saved_data["sinks"].toInt(), ctx->saved_data["scale"].toDouble()});
        const Tensor delta = row_numbers(q);
        a.dout = described(dout), a.out = out.data_ptr(), a.rest = rest.data_ptr(), a.lse = lse.data_ptr<float>(), a.delta = delta.data_ptr<float>();
        a.dq = dq.defined() ? dq.data_ptr() : nullptr;
        Tensor sums;
        if (dk.defined()) {
          a.dk = dk.data_ptr(), a.dv = dv.data_ptr();
          const int64_t n = b200_attention_bwd_workspace(&a);
          if (n) sums = fresh({n}, at::kFloat, q), a.sums = sums.data_ptr<float>();
        }
        int launches = 0;
        const int rc = b200_attention_bwd(&a, &launches, stream());
        launched(launches);
        check(rc, "b200_attention_bwd");
      }
      return {dq, ctx->needs_input_grad(1) ? dk : Tensor(), ctx->needs_input_grad(2) ? dv : Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    });
  }
};

Tensor attention(const Tensor& q, const Tensor& k, const Tensor& v, const c10::optional<Tensor>& lengths, int64_t window, int64_t sinks,
                 c10::optional<double> scale) {
  require(bf16_cuda(q) && bf16_cuda(k) && bf16_cuda(v) && q.dim() == 4 && k.dim() == 4 && v.dim() == 4,
          "q, k and v are bfloat16 CUDA tensors [batch, tokens, heads, head_dim]");
  require(same_device(k, q) && same_device(v, q), "q, k and v are on one device");
  const int64_t B = q.size(0), S = q.size(1), nq = q.size(2), nkv = k.size(2), hd = q.size(3);
  require(k.sizes() == v.sizes() && k.size(0) == B && k.size(1) == S && k.size(3) == hd, "k and v have q's batch, tokens and head_dim");
  require(hd == 64 || hd == 128, "heads are of 64 or 128 elements");
  require(nq >= 1 && nkv >= 1 && nq % nkv == 0, "the heads of q are a multiple of those of k and v");
  require(S <= 1 << 30 && B * nq * ((S + 127) / 128) < 1 << 30, "more rows than a launch has tiles for");
  require(window >= 0 && sinks >= 0, "window and sinks are no negative numbers");
  require(window > 0 || sinks == 0, "sinks go with a window: without one all keys are visible");
  const double factor = scale ? *scale : 1.0 / std::sqrt(static_cast<double>(hd));
  require(factor > 0 && static_cast<float>(factor) > 0.f && std::isfinite(static_cast<float>(factor)), "the scale is a positive number");
  require(!lengths || (same_device(*lengths, q) && lengths->scalar_type() == at::kInt && lengths->dim() == 1 && lengths->size(0) == B && lengths->is_contiguous()),
          "lengths are a contiguous int32 CUDA tensor of one number for each sequence");
  refuse_tangents({&q, &k, &v}, NO_TANGENTS);
  if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return Attention::apply(q, k, v, lengths, window, sinks, factor);
  Tensor lse;
  return forward_of(boxed(q), boxed(k), boxed(v), lengths ? *lengths : Tensor(), {window, sinks, factor}, lse, nullptr);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(b200ops, m) {
  m.def("attention(Tensor q, Tensor k, Tensor v, Tensor? lengths, int window, int sinks, float? scale) -> Tensor", attention);
}

namespace b200torch {
void bind_attention(py::module_& m) {
  m.def("attention", torch::wrap_pybind_function_no_gil([](const Tensor& q, const Tensor& k, const Tensor& v, const c10::optional<Tensor>& lengths,
                                                           int64_t window, int64_t sinks, c10::optional<double> scale) {
          return traced_or_direct("b200ops::attention", attention, q, k, v, lengths, window, sinks, scale);
        }));
}
}  // namespace b200torch
