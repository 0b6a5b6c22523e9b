// Bindings of the kernels that keep activations in 8 bits (act8.cu), and the operators that autograd sees.  Those are nodes of the
// C++ kind: their backward passes run without the interpreter, which took longer than the kernels of short sequences.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <stdexcept>
#include <string>
#include <vector>

#include "ody_kernels.h"

namespace py = pybind11;

void ody_count_launches(int64_t n);
at::Tensor ody_gemm(const at::Tensor& a, const at::Tensor& b, const c10::optional<at::Tensor>& out, int64_t layout, bool accumulate);

namespace {

typedef std::vector<at::Tensor> Tensors;

// Parts are strings: a number put into a stream ends the process here (its locale's facets are another libstdc++'s).
template <class... A>
void req(bool ok, const A&... parts) {
  if (ok) return;
  std::string s = "odysseus_transformer_b200: ";
  ((s += parts), ...);
  throw std::runtime_error(s);
}

void check(int rc, const char* what, int64_t launches) {
  if (rc != 0)
    req(false, what, " failed with code ", std::to_string(rc), rc < 1000 ? std::string(" (") + cudaGetErrorString((cudaError_t)rc) + ")" : std::string());
  ody_count_launches(launches);
}

cudaStream_t stream() { return at::cuda::getCurrentCUDAStream().stream(); }

int format_of(const std::string& name) {
  req(name == "e4m3" || name == "int8", "activations are kept as e4m3 or int8, not ", name);
  return name == "int8" ? 1 : 0;
}

// bf16 rows of a whole number of 16-byte pieces that start on one; contiguous
at::Tensor rows_of(const at::Tensor& t, const char* name) {
  req(t.is_cuda() && t.scalar_type() == at::kBFloat16, name, " must be a bfloat16 CUDA tensor");
  req(t.dim() >= 1 && t.size(-1) > 0 && t.size(-1) % 8 == 0 && t.size(-1) <= (1 << 30), name, ": the last dim must be a multiple of 8");
  at::Tensor c = t.contiguous();
  return ((uintptr_t)c.data_ptr() & 15) ? c.clone() : c;
}
int64_t count(const at::Tensor& t) { return t.numel() / t.size(-1); }

struct Kept {
  const void* codes;
  const float* scales;
  int64_t rows;
  int n, fmt;                                  // columns of a half where there are two
};
Kept kept_of(const at::Tensor& data, const at::Tensor& scale, int halves) {
  req(data.is_cuda() && (data.scalar_type() == at::kChar || data.scalar_type() == at::kFloat8_e4m3fn) && data.dim() == 2 && data.is_contiguous(),
      "kept activations: data must be a contiguous int8 or float8_e4m3fn CUDA tensor [rows, columns]");
  const int64_t n = data.size(1) / halves;
  req(n > 0 && n * halves == data.size(1) && n % 8 == 0 && n <= (1 << 30), "kept activations: columns must be a multiple of 8");
  req(scale.is_cuda() && scale.scalar_type() == at::kFloat && scale.is_contiguous() && scale.dim() == 2 && scale.size(0) == data.size(0) &&
          scale.size(1) == halves * ((n + 127) / 128) && scale.get_device() == data.get_device(),
      "kept activations: scale must be a contiguous fp32 tensor of a scale for every 128 columns, on data's device");
  req(((uintptr_t)data.data_ptr() & 7) == 0, "kept activations: data must start on 8 bytes");
  return {data.data_ptr(), scale.data_ptr<float>(), data.size(0), (int)n, data.scalar_type() == at::kChar ? 1 : 0};
}
// An uninitialised tensor, without the dispatcher: a norm allocates eight, 0.6 us less each
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, like.device(), c10::nullopt));
}
std::pair<at::Tensor, at::Tensor> new_kept(const at::Tensor& like, int64_t rows, int64_t n, int halves, int fmt) {
  return {fresh({rows, halves * n}, fmt ? at::kChar : at::kFloat8_e4m3fn, like), fresh({rows, halves * ((n + 127) / 128)}, at::kFloat, like)};
}

Tensors pack8(const at::Tensor& any, const std::string& format) {
  const int fmt = format_of(format);
  req(any.is_cuda() && any.scalar_type() == at::kBFloat16 && any.dim() > 0 && any.size(-1) > 0, "pack8: a bfloat16 CUDA tensor with columns");
  c10::cuda::CUDAGuard guard(any.device());
  at::NoGradGuard no_grad;
  const at::Tensor x = any.dim() == 2 ? any : any.reshape({-1, any.size(-1)});
  // rows may lie apart
  const bool apart = x.stride(1) == 1 && x.stride(0) >= x.size(1) && x.stride(0) % 8 == 0 && ((uintptr_t)x.data_ptr() & 15) == 0;
  const at::Tensor c = apart && x.size(1) > 0 && x.size(1) % 8 == 0 ? x : rows_of(x, "pack8: x");
  const int64_t rows = c.size(0), n = c.size(1);
  req(n <= (1 << 30), "pack8: too many columns");
  auto [data, scale] = new_kept(c, rows, n, 1, fmt);
  check(ody_pack8(c.data_ptr(), rows > 1 ? c.stride(0) : n, data.data_ptr(), scale.data_ptr<float>(), rows, (int)n, fmt, stream()), "pack8", 1);
  return {data, scale};
}

at::Tensor unpack8(const at::Tensor& data, const at::Tensor& scale, const c10::optional<at::Tensor>& weight) {
  const Kept k = kept_of(data, scale, 1);
  c10::cuda::CUDAGuard guard(data.device());
  at::Tensor w;
  if (weight.has_value()) {
    w = rows_of(weight.value(), "unpack8: weight");
    req(w.numel() == k.n && w.get_device() == data.get_device(), "unpack8: one weight for every column, on data's device");
  }
  auto x = fresh({k.rows, k.n}, at::kBFloat16, data);
  check(ody_unpack8(k.codes, k.scales, w.defined() ? w.data_ptr() : nullptr, x.data_ptr(), k.rows, k.n, k.fmt, stream()), "unpack8", 1);
  return x;
}

Tensors swiglu8_fwd(const at::Tensor& gate_up, const std::string& format) {
  const int fmt = format_of(format);
  const at::Tensor gu = rows_of(gate_up, "swiglu8: gate_up");
  const int64_t n = gu.size(-1) / 2, rows = count(gu);
  req(gu.dim() == 2 && n % 8 == 0, "swiglu8: gate_up must be [rows, 2 n] with n a multiple of 8");
  c10::cuda::CUDAGuard guard(gu.device());
  auto h = fresh({rows, n}, at::kBFloat16, gu);
  auto [data, scale] = new_kept(gu, rows, n, 2, fmt);
  check(ody_swiglu8_fwd(gu.data_ptr(), h.data_ptr(), data.data_ptr(), scale.data_ptr<float>(), rows, (int)n, fmt, stream()), "swiglu8_fwd", 1);
  return {h, data, scale};
}

at::Tensor swiglu8_restore(const at::Tensor& data, const at::Tensor& scale) {
  const Kept k = kept_of(data, scale, 2);
  c10::cuda::CUDAGuard guard(data.device());
  auto h = fresh({k.rows, k.n}, at::kBFloat16, data);
  check(ody_swiglu8_restore(k.codes, k.scales, h.data_ptr(), k.rows, k.n, k.fmt, stream()), "swiglu8_restore", 1);
  return h;
}

at::Tensor swiglu8_bwd(const at::Tensor& dh_, const at::Tensor& data, const at::Tensor& scale) {
  const Kept k = kept_of(data, scale, 2);
  const at::Tensor dh = rows_of(dh_, "swiglu8: dh");
  req(dh.size(-1) == k.n && count(dh) == k.rows && dh.get_device() == data.get_device(), "swiglu8: dh must be [rows, n] on data's device");
  c10::cuda::CUDAGuard guard(data.device());
  auto dgu = fresh({k.rows, 2 * k.n}, at::kBFloat16, dh);
  check(ody_swiglu8_bwd(dh.data_ptr(), k.codes, k.scales, dgu.data_ptr(), k.rows, k.n, k.fmt, stream()), "swiglu8_bwd", 1);
  return dgu;
}

at::Tensor weight_of(const at::Tensor& w_, int64_t n, int device) {
  const at::Tensor w = rows_of(w_, "rmsnorm8: w");
  req(w.numel() == n && w.get_device() == device, "rmsnorm8: w must have x's last dim, on x's device");
  req(n <= ODY_RMSNORM8_MAX, "rmsnorm8: rows of up to ", std::to_string(ODY_RMSNORM8_MAX), " columns");
  return w;
}

// (x or x + delta, its norm, rstd, codes, scales)
Tensors rmsnorm8_fwd(const at::Tensor& x_, const c10::optional<at::Tensor>& delta_, const at::Tensor& w_, double eps, const std::string& format) {
  const int fmt = format_of(format);
  const at::Tensor x = rows_of(x_, "rmsnorm8: x");
  const int64_t n = x.size(-1), rows = count(x);
  const at::Tensor w = weight_of(w_, n, x.get_device());
  c10::cuda::CUDAGuard guard(x.device());
  at::Tensor delta, s = x;
  if (delta_.has_value()) {
    delta = rows_of(delta_.value(), "rmsnorm8: delta");
    req(delta.sizes() == x.sizes() && delta.get_device() == x.get_device(), "rmsnorm8: delta must match x");
    s = fresh(x.sizes(), at::kBFloat16, x);
  }
  auto y = fresh(x.sizes(), at::kBFloat16, x), rstd = fresh({rows}, at::kFloat, x);
  auto [data, scale] = new_kept(x, rows, n, 1, fmt);
  check(ody_rmsnorm8_fwd(x.data_ptr(), delta.defined() ? delta.data_ptr() : nullptr, w.data_ptr(), delta.defined() ? s.data_ptr() : nullptr,
                         y.data_ptr(), rstd.data_ptr<float>(), data.data_ptr(), scale.data_ptr<float>(), rows, (int)n, (float)eps, fmt, stream()),
        "rmsnorm8_fwd", 1);
  return {s, y, rstd, data, scale};
}

// (dx, dw): dw fp32, or dw_out (bf16) filled
Tensors rmsnorm8_bwd(const at::Tensor& dy_, const at::Tensor& data, const at::Tensor& scale, const at::Tensor& w_, const at::Tensor& rstd,
                     const c10::optional<at::Tensor>& ds_, const c10::optional<at::Tensor>& dw_out) {
  const Kept k = kept_of(data, scale, 1);
  const at::Tensor dy = rows_of(dy_, "rmsnorm8: dy");
  req(dy.size(-1) == k.n && count(dy) == k.rows && dy.get_device() == data.get_device(), "rmsnorm8: dy must match the kept rows");
  const at::Tensor w = weight_of(w_, k.n, dy.get_device());
  req(rstd.is_cuda() && rstd.scalar_type() == at::kFloat && rstd.is_contiguous() && rstd.numel() == k.rows && rstd.get_device() == dy.get_device(),
      "rmsnorm8: rstd must be a contiguous fp32 tensor with one entry per row, on dy's device");
  c10::cuda::CUDAGuard guard(dy.device());
  at::Tensor ds;
  if (ds_.has_value()) {
    ds = rows_of(ds_.value(), "rmsnorm8: ds");
    req(ds.sizes() == dy.sizes() && ds.get_device() == dy.get_device(), "rmsnorm8: ds must match dy");
  }
  if (dw_out.has_value())
    req(dw_out->is_cuda() && dw_out->scalar_type() == at::kBFloat16 && dw_out->is_contiguous() && dw_out->numel() == k.n &&
            dw_out->get_device() == dy.get_device(), "rmsnorm8: dw_out must be a contiguous bfloat16 tensor of x's last dim");
  auto dx = fresh(dy.sizes(), at::kBFloat16, dy);
  auto dw = dw_out.has_value() ? dw_out.value() : fresh({k.n}, at::kFloat, dy);
  auto partial = fresh({ody_rmsnorm8_bwd_blocks(k.rows, k.n), k.n}, at::kFloat, dy);
  check(ody_rmsnorm8_bwd(dy.data_ptr(), k.codes, k.scales, w.data_ptr(), rstd.data_ptr<float>(), ds.defined() ? ds.data_ptr() : nullptr,
                         dx.data_ptr(), dw.data_ptr(), dw_out.has_value() ? 1 : 0, partial.data_ptr<float>(), k.rows, k.n, k.fmt, stream()),
        "rmsnorm8_bwd", 2);
  return {dx, dw};
}

// ------------------------------------------------------------------------------------------- autograd

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients that cannot be differentiated again: where a graph of the backward is recorded, one that says so when it is used.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  for (auto& g : grads)
    if (g.defined()) g = g.detach().requires_grad_();
  auto node = std::make_shared<torch::autograd::DelayedError>("gradients of activations kept in 8 bits cannot be differentiated again", grads.size());
  return (*node)(std::move(grads));
}

// What the optimizer attached to a weight: its flat gradient, and whether this step has written it (``main_grad``,
// ``_grad_written``).  Made and used with the interpreter's lock held.
struct MainGrad {
  py::object w;
  at::Tensor grad;
  bool written = false;
  explicit MainGrad(const at::Tensor& weight) : w(py::cast(weight)) {
    py::object g = py::getattr(w, "main_grad", py::none());
    if (g.is_none()) return;
    grad = g.cast<at::Tensor>();
    written = py::getattr(w, "_grad_written", py::bool_(false)).cast<bool>();
  }
  void done() { w.attr("_grad_written") = true; }
};

struct RmsNorm8 : torch::autograd::Function<RmsNorm8> {
  // (x or x + delta, its norm, codes, scales)
  static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const c10::optional<at::Tensor>& delta, const at::Tensor& w, double eps,
                               const std::string& format) {
    auto out = rmsnorm8_fwd(x, delta, w, eps, format);
    ctx->save_for_backward({out[3], out[4], w, out[2]});
    ctx->mark_non_differentiable({out[3], out[4]});
    ctx->set_materialize_grads(false);
    ctx->saved_data["added"] = delta.has_value();
    return {delta.has_value() ? out[0] : x, out[1], out[3], out[4]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const at::Tensor &ds = grads[0], &dy = grads[1];
    at::Tensor dx = ds, dw;
    if (dy.defined()) {
      const auto saved = ctx->get_saved_variables();
      const at::Tensor& w = saved[2];
      const c10::optional<at::Tensor> dso = ds.defined() ? c10::optional<at::Tensor>(ds) : c10::nullopt;
      if (w.requires_grad()) {
        py::gil_scoped_acquire lock;
        MainGrad mg(w);
        if (mg.grad.defined()) {
          const bool in_place = !mg.written && mg.grad.scalar_type() == at::kBFloat16 && mg.grad.sizes() == w.sizes() && mg.grad.is_contiguous() &&
                                mg.grad.device() == dy.device();
          auto got = rmsnorm8_bwd(dy, saved[0], saved[1], w, saved[3], dso, in_place ? c10::optional<at::Tensor>(mg.grad) : c10::nullopt);
          if (in_place) mg.done();
          else py::module_::import("odysseus_transformer_b200.ops.functional").attr("deliver_grad")(mg.w, got[1]);
          return once({got[0], ctx->saved_data["added"].toBool() ? got[0] : at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()});
        }
      }
      dw = fresh(w.sizes(), at::kBFloat16, w);
      dx = rmsnorm8_bwd(dy, saved[0], saved[1], w, saved[3], dso, dw)[0];
    }
    return once({dx, ctx->saved_data["added"].toBool() ? dx : at::Tensor(), dw, at::Tensor(), at::Tensor()});
  }
};

struct SwiGlu8 : torch::autograd::Function<SwiGlu8> {
  static variable_list forward(AutogradContext* ctx, const at::Tensor& gate_up, const std::string& format) {
    auto out = swiglu8_fwd(gate_up.dim() == 2 ? gate_up : gate_up.reshape({-1, gate_up.size(-1)}), format);
    ctx->save_for_backward({out[1], out[2]});
    ctx->mark_non_differentiable({out[1], out[2]});
    ctx->set_materialize_grads(false);
    if (gate_up.dim() != 2) {
      auto shape = gate_up.sizes().vec();
      shape.back() /= 2;
      out[0] = out[0].view(shape);
    }
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return {at::Tensor(), at::Tensor()};
    const auto saved = ctx->get_saved_variables();
    at::Tensor dgu = swiglu8_bwd(grads[0], saved[0], saved[1]);
    if (grads[0].dim() != 2) {
      auto shape = grads[0].sizes().vec();
      shape.back() *= 2;
      dgu = dgu.view(shape);
    }
    return once({dgu, at::Tensor()});
  }
};

// y = x w^T; in the backward pass x is what (data, scale, weight, product) restore
struct Linear8 : torch::autograd::Function<Linear8> {
  static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& w, const at::Tensor& data, const at::Tensor& scale,
                            const c10::optional<at::Tensor>& weight, bool product) {
    ctx->save_for_backward({w, data, scale, weight.has_value() ? *weight : at::Tensor()});
    ctx->saved_data["product"] = product;
    ctx->saved_data["x"] = x.requires_grad();
    at::Tensor y = ody_gemm(x.dim() == 2 ? x : x.reshape({-1, x.size(-1)}), w, c10::nullopt, 0, false);
    if (x.dim() == 2) return y;
    auto shape = x.sizes().vec();
    shape.back() = w.size(0);
    return y.view(shape);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(6);
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &w = saved[0], &data = saved[1], &scale = saved[2];
    const at::Tensor dy = grads[0].reshape({-1, grads[0].size(-1)}).contiguous();
    at::Tensor dx, dw;
    py::gil_scoped_acquire lock;
    if (ctx->saved_data["x"].toBool()) {
      dx = ody_gemm(dy, w, c10::nullopt, 1, false);
      if (grads[0].dim() != 2) {
        auto shape = grads[0].sizes().vec();
        shape.back() = w.size(1);
        dx = dx.view(shape);
      }
    }
    if (w.requires_grad()) {
      const at::Tensor x = ctx->saved_data["product"].toBool()
                               ? swiglu8_restore(data, scale)
                               : unpack8(data, scale, saved[3].defined() ? c10::optional<at::Tensor>(saved[3]) : c10::nullopt);
      MainGrad mg(w);
      if (mg.grad.defined()) {
        ody_gemm(dy, x, mg.grad, 2, mg.written);
        mg.done();
      } else {
        dw = ody_gemm(dy, x, c10::nullopt, 2, false);
      }
    }
    return once({dx, dw, at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()});
  }
};

}  // namespace

void ody_register_act8(pybind11::module& m) {
  m.def("rmsnorm8", [](const at::Tensor& x, const c10::optional<at::Tensor>& delta, const at::Tensor& w, double eps, const std::string& fmt) {
    return RmsNorm8::apply(x, delta, w, eps, fmt);
  });
  m.def("swiglu8", [](const at::Tensor& gate_up, const std::string& fmt) { return SwiGlu8::apply(gate_up, fmt); });
  m.def("linear8", [](const at::Tensor& x, const at::Tensor& w, const at::Tensor& data, const at::Tensor& scale, const c10::optional<at::Tensor>& weight,
                      bool product) { return Linear8::apply(x, w, data, scale, weight, product); });
  m.def("pack8", &pack8, py::arg("x"), py::arg("fmt"));
  m.def("unpack8", &unpack8, py::arg("data"), py::arg("scale"), py::arg("weight") = py::none());
  m.def("swiglu8_fwd", &swiglu8_fwd, py::arg("gate_up"), py::arg("fmt"));
  m.def("swiglu8_restore", &swiglu8_restore, py::arg("data"), py::arg("scale"));
  m.def("swiglu8_bwd", &swiglu8_bwd, py::arg("dh"), py::arg("data"), py::arg("scale"));
  m.def("rmsnorm8_fwd", &rmsnorm8_fwd, py::arg("x"), py::arg("delta"), py::arg("w"), py::arg("eps"), py::arg("fmt"));
  m.def("rmsnorm8_bwd", &rmsnorm8_bwd, py::arg("dy"), py::arg("data"), py::arg("scale"), py::arg("w"), py::arg("rstd"), py::arg("ds") = py::none(),
        py::arg("dw_out") = py::none());
}
