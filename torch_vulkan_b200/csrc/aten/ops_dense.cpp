// The fused Linear layer and layer norm over tensors, and aten::native_layer_norm (with its backward) on device "vk": the layers
// between a model's quantised products.
//
// The functions here take "vk" tensors (queued on the backend's stream) and torch.cuda tensors (queued on torch's current stream,
// outputs and workspaces from torch's allocator, so that they behave like any CUDA op). The reference dispatches these
// layers as separate matrix, elementwise and reduction kernels (crates/pyvk/csrc/linalg.cpp:227-321).
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/library.h>

#include "backend.h"

namespace vkb {
namespace {

// Where a call runs: the operands' device made current for its duration, and the stream for the C ABI.
struct Where {
  explicit Where(const at::Tensor& t) : guard(t.device()), device(t.device().index()) {
    if (t.is_cuda()) {  // (asked through the device-independent interface: the extension needs no CUDA build of PyTorch to load)
      stream = c10::impl::VirtualGuardImpl(c10::DeviceType::CUDA).getStream(t.device()).native_handle();
      if (stream == nullptr) stream = reinterpret_cast<void*>(uintptr_t(1));  // cudaStreamLegacy: NULL means the backend's own
    }
  }
  c10::DeviceGuard guard;
  int device;
  void* stream = nullptr;
};

const void* address(const std::optional<at::Tensor>& t) { return t.has_value() ? gpu_address(*t) : nullptr; }
void* address_out(const at::Tensor& t) { return t.defined() ? gpu_address_out(t) : nullptr; }

int float_code(const char* fn, const at::Tensor& t) {
  const int d = dtype_code(t.scalar_type());
  TORCH_CHECK_TYPE(d == TVB_F32 || d == TVB_F16 || d == TVB_BF16, fn, ": float32, float16 or bfloat16 expected, got ", t.scalar_type());
  return d;
}

void check_device(const char* fn, const at::Tensor& t) {
  TORCH_CHECK_VALUE(is_vk(t) || t.is_cuda(), fn, ": tensors on \"vk\" or CUDA expected, got ", t.device());
}

// A [rows, cols] operand of `like`'s dtype and device with contiguous columns; returns its row stride in elements.
int64_t matrix(const char* fn, const char* name, const at::Tensor& t, int64_t rows, int64_t cols, const at::Tensor& like) {
  TORCH_CHECK_VALUE(t.dim() == 2 && t.size(0) == rows && t.size(1) == cols && t.scalar_type() == like.scalar_type() && t.device() == like.device(),
                    fn, ": ", name, " must be a ", like.scalar_type(), " matrix [", rows, ", ", cols, "] on ", like.device(), ", got ",
                    t.scalar_type(), " ", t.sizes(), " on ", t.device());
  TORCH_CHECK_VALUE((cols <= 1 || t.stride(1) == 1) && (rows <= 1 || t.stride(0) >= cols), fn, ": ", name,
                    " needs contiguous columns and rows that do not overlap (strides ", t.strides(), ")");
  return rows > 1 ? t.stride(0) : cols;
}

void vector(const char* fn, const char* name, const at::Tensor& t, int64_t n, const at::Tensor& like, bool or_float) {
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == n && t.device() == like.device() && t.is_contiguous() &&
                        (t.scalar_type() == like.scalar_type() || (or_float && t.scalar_type() == at::kFloat)),
                    fn, ": ", name, " must be a contiguous vector of ", n, " values on ", like.device(), " of ", like.scalar_type(),
                    or_float ? " or float32" : "", ", got ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
}

at::Tensor workspace(uint64_t bytes, const at::Tensor& like) {
  return bytes == 0 ? at::Tensor() : at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

at::Tensor optional_empty(bool want, at::IntArrayRef sizes, const at::TensorOptions& options) {
  return want ? at::empty(sizes, options) : at::Tensor();
}

// The dtype code that weight and bias share (x's where neither is given).
int param_code(const char* fn, const at::Tensor& x, int64_t d, const std::optional<at::Tensor>& weight, const std::optional<at::Tensor>& bias) {
  if (weight.has_value()) vector(fn, "weight", *weight, d, x, true);
  if (bias.has_value()) vector(fn, "bias", *bias, d, x, true);
  TORCH_CHECK_VALUE(!weight.has_value() || !bias.has_value() || weight->scalar_type() == bias->scalar_type(), fn,
                    ": weight and bias must have one dtype");
  return weight.has_value() ? dtype_code(weight->scalar_type()) : bias.has_value() ? dtype_code(bias->scalar_type()) : dtype_code(x.scalar_type());
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> linear_act(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias,
                                              const std::optional<at::Tensor>& residual, int64_t activation, bool save) {
  const char* fn = "linear";
  const int code = float_code(fn, x);
  TORCH_CHECK_VALUE(x.dim() == 2 && w.dim() == 2, fn, ": x [m, k] and w [n, k] expected");
  const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
  const int64_t x_sm = matrix(fn, "x", x, m, k, x), w_sn = matrix(fn, "w", w, n, k, x);
  if (bias.has_value()) vector(fn, "bias", *bias, n, x, false);
  const int64_t r_sm = residual.has_value() ? matrix(fn, "residual", *residual, m, n, x) : 0;
  check_device(fn, x);
  Where at(x);
  at::Tensor y = at::empty({m, n}, x.options());
  at::Tensor z = optional_empty(save, {m, n}, x.options());
  const void *xp = gpu_address(x), *wp = gpu_address(w);
  const uint64_t bytes = tvb_linear_workspace_bytes(code, xp, x_sm, wp, w_sn, m, n, k);
  at::Tensor ws = workspace(bytes, x);
  check(tvb_linear(at.device, xp, code, x_sm, wp, w_sn, address(bias), static_cast<int>(activation), address(residual), r_sm, address_out(y),
                   address_out(z), m, n, k, address_out(ws), bytes, at.stream));
  return {y, z};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_act_backward(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& w,
                                                                   const std::optional<at::Tensor>& z, int64_t activation, int64_t want) {
  const char* fn = "linear_backward";
  const int code = float_code(fn, x);
  TORCH_CHECK_VALUE(x.dim() == 2 && w.dim() == 2, fn, ": x [m, k] and w [n, k] expected");
  const int64_t m = x.size(0), k = x.size(1), n = w.size(0);
  const int64_t x_sm = matrix(fn, "x", x, m, k, x), w_sn = matrix(fn, "w", w, n, k, x), dy_sm = matrix(fn, "dy", dy, m, n, x);
  if (z.has_value()) {
    matrix(fn, "z", *z, m, n, x);
    TORCH_CHECK_VALUE(z->is_contiguous(), fn, ": z must be contiguous");
  }
  TORCH_CHECK_VALUE(z.has_value() || activation == TVB_ACT_NONE, fn, ": an activation's gradient needs z, the values before it");
  check_device(fn, x);
  Where at(x);
  at::Tensor dx = optional_empty((want & TVB_WANT_DX) != 0, {m, k}, x.options());
  at::Tensor dw = optional_empty((want & TVB_WANT_DW) != 0, {n, k}, x.options());
  at::Tensor db = optional_empty((want & TVB_WANT_DB) != 0, {n}, x.options());
  const void *dyp = gpu_address(dy), *xp = gpu_address(x), *wp = gpu_address(w);
  const uint64_t bytes = tvb_linear_backward_workspace_bytes(code, dyp, dy_sm, xp, x_sm, wp, w_sn, static_cast<int>(activation),
                                                             static_cast<int>(want), m, n, k);
  at::Tensor ws = workspace(bytes, x);
  check(tvb_linear_backward(at.device, dyp, code, dy_sm, address(z), xp, x_sm, wp, w_sn, static_cast<int>(activation), address_out(dx),
                            address_out(dw), address_out(db), m, n, k, address_out(ws), bytes, at.stream));
  return {dx, dw, db};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm(const at::Tensor& x, const std::optional<at::Tensor>& weight,
                                                          const std::optional<at::Tensor>& bias, double eps) {
  const char* fn = "layer_norm";
  const int code = float_code(fn, x);
  TORCH_CHECK_VALUE(x.dim() == 2, fn, ": x [rows, d] expected");
  const int64_t rows = x.size(0), d = x.size(1), x_sm = matrix(fn, "x", x, rows, d, x);
  const int pcode = param_code(fn, x, d, weight, bias);
  check_device(fn, x);
  Where at(x);
  at::Tensor y = at::empty({rows, d}, x.options());
  at::Tensor mean = at::empty({rows}, x.options().dtype(at::kFloat)), rstd = at::empty({rows}, x.options().dtype(at::kFloat));
  if (d == 0) {  // (rows of nothing have no statistics)
    mean.zero_();
    rstd.zero_();
  }
  check(tvb_layer_norm(at.device, gpu_address(x), code, x_sm, address(weight), address(bias), pcode, static_cast<float>(eps), address_out(y),
                       static_cast<float*>(address_out(mean)), static_cast<float*>(address_out(rstd)), rows, d, at.stream));
  return {y, mean, rstd};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> layer_norm_backward(const at::Tensor& dy, const at::Tensor& x, const at::Tensor& mean,
                                                                   const at::Tensor& rstd, const std::optional<at::Tensor>& weight,
                                                                   bool need_x, bool need_weight, bool need_bias,
                                                                   std::optional<at::ScalarType> param_type) {
  const char* fn = "layer_norm_backward";
  const int code = float_code(fn, x);
  TORCH_CHECK_VALUE(x.dim() == 2, fn, ": x [rows, d] expected");
  const int64_t rows = x.size(0), d = x.size(1), x_sm = matrix(fn, "x", x, rows, d, x), dy_sm = matrix(fn, "dy", dy, rows, d, x);
  // without a weight the gradients of the parameters are of param_type (the bias's), or of x's
  const at::ScalarType ptype = weight.has_value() ? weight->scalar_type() : param_type.value_or(x.scalar_type());
  const int pcode = weight.has_value() ? param_code(fn, x, d, weight, std::nullopt) : dtype_code(ptype);
  TORCH_CHECK_VALUE(ptype == x.scalar_type() || ptype == at::kFloat, fn, ": parameters must be of ", x.scalar_type(), " or float32, got ", ptype);
  for (const at::Tensor* t : {&mean, &rstd})
    TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == rows && t->device() == x.device() && t->is_contiguous() && t->scalar_type() == at::kFloat,
                      fn, ": mean and rstd must be contiguous float32 vectors of ", rows, " values on ", x.device());
  check_device(fn, x);
  Where at(x);
  const at::TensorOptions params = x.options().dtype(ptype);
  at::Tensor dx = optional_empty(need_x, {rows, d}, x.options());
  at::Tensor dw = optional_empty(need_weight, {d}, params), db = optional_empty(need_bias, {d}, params);
  const uint64_t bytes = need_weight || need_bias ? tvb_layer_norm_backward_workspace_bytes(rows, d) : 0;
  at::Tensor ws = workspace(bytes, x);
  check(tvb_layer_norm_backward(at.device, gpu_address(dy), code, dy_sm, gpu_address(x), x_sm, static_cast<const float*>(gpu_address(mean)),
                                static_cast<const float*>(gpu_address(rstd)), address(weight), pcode, address_out(dx), address_out(dw),
                                address_out(db), rows, d, address_out(ws), bytes, at.stream));
  return {dx, dw, db};
}

namespace {

// ------------------------------------------------------------------ aten::native_layer_norm

struct NormShape {
  int64_t rows, d;
  std::vector<int64_t> stat;  // the leading sizes, then ones: the shape of mean and rstd
};

NormShape norm_shape(const at::Tensor& input, at::IntArrayRef normalized_shape, const std::optional<at::Tensor>& weight,
                     const std::optional<at::Tensor>& bias) {
  const int64_t nd = static_cast<int64_t>(normalized_shape.size());
  TORCH_CHECK(nd >= 1, "Expected normalized_shape to be at least 1-dimensional, i.e., containing at least one element, but got ",
              "normalized_shape = ", normalized_shape);
  TORCH_CHECK(!weight.has_value() || !weight->defined() || weight->sizes().equals(normalized_shape),
              "Expected weight to be of same shape as normalized_shape, but got weight of shape ", weight->sizes(),
              " and normalized_shape = ", normalized_shape);
  TORCH_CHECK(!bias.has_value() || !bias->defined() || bias->sizes().equals(normalized_shape),
              "Expected bias to be of same shape as normalized_shape, but got bias of shape ", bias->sizes(), " and normalized_shape = ",
              normalized_shape);
  TORCH_CHECK(input.dim() >= nd && input.sizes().slice(input.dim() - nd).equals(normalized_shape), "Given normalized_shape=", normalized_shape,
              ", expected input with shape [*", normalized_shape, "], but got input of size", input.sizes());
  NormShape s{1, 1, {}};
  for (int64_t i = 0; i < input.dim(); i++) {
    const bool lead = i < input.dim() - nd;
    (lead ? s.rows : s.d) *= input.size(i);
    s.stat.push_back(lead ? input.size(i) : 1);
  }
  return s;
}

std::optional<at::Tensor> flat(const std::optional<at::Tensor>& t) {
  if (!t.has_value() || !t->defined()) return std::nullopt;
  return t->contiguous().view({t->numel()});
}

// A [rows, d] view where the last dimensions are one run of memory, else a copy.
at::Tensor as_rows(const at::Tensor& t, const NormShape& s) {
  if (t.dim() == 2 && t.size(1) == s.d && (s.d <= 1 || t.stride(1) == 1) && (s.rows <= 1 || t.stride(0) >= s.d)) return t;
  return t.contiguous().view({s.rows, s.d});
}

void require_all_vk(const char* op, std::initializer_list<const std::optional<at::Tensor>*> tensors) {
  for (const std::optional<at::Tensor>* t : tensors)
    if (t->has_value() && (*t)->defined() && !is_vk(**t)) no_fallback(op, "an operand is not on \"vk\"");
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> native_layer_norm(const at::Tensor& input, at::IntArrayRef normalized_shape,
                                                                 const std::optional<at::Tensor>& weight,
                                                                 const std::optional<at::Tensor>& bias, double eps) {
  const NormShape s = norm_shape(input, normalized_shape, weight, bias);
  const std::optional<at::Tensor> in = input;
  require_all_vk("aten::native_layer_norm", {&in, &weight, &bias});
  auto [y, mean, rstd] = layer_norm(as_rows(input, s), flat(weight), flat(bias), eps);
  return {y.view(input.sizes()), mean.view(s.stat), rstd.view(s.stat)};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> native_layer_norm_backward(const at::Tensor& grad_out, const at::Tensor& input,
                                                                          at::IntArrayRef normalized_shape, const at::Tensor& mean,
                                                                          const at::Tensor& rstd, const std::optional<at::Tensor>& weight,
                                                                          const std::optional<at::Tensor>& bias, std::array<bool, 3> mask) {
  const NormShape s = norm_shape(input, normalized_shape, weight, bias);
  const std::optional<at::Tensor> go = grad_out, in = input, me = mean, rs = rstd;
  require_all_vk("aten::native_layer_norm_backward", {&go, &in, &me, &rs, &weight, &bias});
  const std::optional<at::Tensor> w = flat(weight);
  const bool has_bias = bias.has_value() && bias->defined();
  auto [dx, dw, db] = layer_norm_backward(as_rows(grad_out, s), as_rows(input, s), mean.contiguous().view({s.rows}),
                                          rstd.contiguous().view({s.rows}), w, mask[0], mask[1], mask[2],
                                          has_bias ? std::optional<at::ScalarType>(bias->scalar_type()) : std::nullopt);
  if (dx.defined()) dx = dx.view(input.sizes());
  if (dw.defined()) dw = dw.view(normalized_shape);
  if (db.defined()) db = db.view(normalized_shape);
  return {dx, dw, db};
}

}  // namespace
}  // namespace vkb

TORCH_LIBRARY_IMPL(aten, PrivateUse1, m) {
  using namespace vkb;
  m.impl("native_layer_norm", &native_layer_norm);
  m.impl("native_layer_norm_backward", &native_layer_norm_backward);
}
