// Bindings of the kernels that keep activations in 8 bits (act8.cu).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <stdexcept>
#include <string>
#include <vector>

#include "ody_kernels.h"

void ody_count_launches(int64_t n);

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
std::pair<at::Tensor, at::Tensor> new_kept(const at::Tensor& like, int64_t rows, int64_t n, int halves, int fmt) {
  return {at::empty({rows, halves * n}, like.options().dtype(fmt ? at::kChar : at::kFloat8_e4m3fn)),
          at::empty({rows, halves * ((n + 127) / 128)}, like.options().dtype(at::kFloat))};
}

Tensors pack8(const at::Tensor& x, const std::string& format) {
  const int fmt = format_of(format);
  req(x.is_cuda() && x.scalar_type() == at::kBFloat16 && x.dim() == 2, "pack8: a bfloat16 CUDA tensor [rows, columns]");
  c10::cuda::CUDAGuard guard(x.device());
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
  auto x = at::empty({k.rows, k.n}, data.options().dtype(at::kBFloat16));
  check(ody_unpack8(k.codes, k.scales, w.defined() ? w.data_ptr() : nullptr, x.data_ptr(), k.rows, k.n, k.fmt, stream()), "unpack8", 1);
  return x;
}

Tensors swiglu8_fwd(const at::Tensor& gate_up, const std::string& format) {
  const int fmt = format_of(format);
  const at::Tensor gu = rows_of(gate_up, "swiglu8: gate_up");
  const int64_t n = gu.size(-1) / 2, rows = count(gu);
  req(gu.dim() == 2 && n % 8 == 0, "swiglu8: gate_up must be [rows, 2 n] with n a multiple of 8");
  c10::cuda::CUDAGuard guard(gu.device());
  auto h = at::empty({rows, n}, gu.options());
  auto [data, scale] = new_kept(gu, rows, n, 2, fmt);
  check(ody_swiglu8_fwd(gu.data_ptr(), h.data_ptr(), data.data_ptr(), scale.data_ptr<float>(), rows, (int)n, fmt, stream()), "swiglu8_fwd", 1);
  return {h, data, scale};
}

at::Tensor swiglu8_restore(const at::Tensor& data, const at::Tensor& scale) {
  const Kept k = kept_of(data, scale, 2);
  c10::cuda::CUDAGuard guard(data.device());
  auto h = at::empty({k.rows, k.n}, data.options().dtype(at::kBFloat16));
  check(ody_swiglu8_restore(k.codes, k.scales, h.data_ptr(), k.rows, k.n, k.fmt, stream()), "swiglu8_restore", 1);
  return h;
}

at::Tensor swiglu8_bwd(const at::Tensor& dh_, const at::Tensor& data, const at::Tensor& scale) {
  const Kept k = kept_of(data, scale, 2);
  const at::Tensor dh = rows_of(dh_, "swiglu8: dh");
  req(dh.size(-1) == k.n && count(dh) == k.rows && dh.get_device() == data.get_device(), "swiglu8: dh must be [rows, n] on data's device");
  c10::cuda::CUDAGuard guard(data.device());
  auto dgu = at::empty({k.rows, 2 * k.n}, dh.options());
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
    s = at::empty_like(x);
  }
  auto y = at::empty_like(x), rstd = at::empty({rows}, x.options().dtype(at::kFloat));
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
  auto dx = at::empty_like(dy);
  auto dw = dw_out.has_value() ? dw_out.value() : at::empty({k.n}, dy.options().dtype(at::kFloat));
  auto partial = at::empty({ody_rmsnorm8_bwd_blocks(k.rows, k.n), k.n}, dy.options().dtype(at::kFloat));
  check(ody_rmsnorm8_bwd(dy.data_ptr(), k.codes, k.scales, w.data_ptr(), rstd.data_ptr<float>(), ds.defined() ? ds.data_ptr() : nullptr,
                         dx.data_ptr(), dw.data_ptr(), dw_out.has_value() ? 1 : 0, partial.data_ptr<float>(), k.rows, k.n, k.fmt, stream()),
        "rmsnorm8_bwd", 2);
  return {dx, dw};
}

}  // namespace

void ody_register_act8(pybind11::module& m) {
  namespace py = pybind11;
  m.def("pack8", &pack8, py::arg("x"), py::arg("fmt"));
  m.def("unpack8", &unpack8, py::arg("data"), py::arg("scale"), py::arg("weight") = py::none());
  m.def("swiglu8_fwd", &swiglu8_fwd, py::arg("gate_up"), py::arg("fmt"));
  m.def("swiglu8_restore", &swiglu8_restore, py::arg("data"), py::arg("scale"));
  m.def("swiglu8_bwd", &swiglu8_bwd, py::arg("dh"), py::arg("data"), py::arg("scale"));
  m.def("rmsnorm8_fwd", &rmsnorm8_fwd, py::arg("x"), py::arg("delta"), py::arg("w"), py::arg("eps"), py::arg("fmt"));
  m.def("rmsnorm8_bwd", &rmsnorm8_bwd, py::arg("dy"), py::arg("data"), py::arg("scale"), py::arg("w"), py::arg("rstd"), py::arg("ds") = py::none(),
        py::arg("dw_out") = py::none());
}
