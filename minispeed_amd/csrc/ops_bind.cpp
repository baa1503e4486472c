// Python binding of libminispeed_ops.so (include/minispeed_ops.h).
//
// Each function checks its tensors, allocates its outputs and workspace
// through torch's caching allocator on the current stream, and makes one call
// into the library.  Host code only; done from Python the same checks cost
// several times what the smallest kernels take.

#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>
#include <pybind11/stl.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/ops/empty.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <cmath>
#include <cstdint>
#include <limits>
#include <optional>
#include <string>
#include <vector>

#include "minispeed_ops.h"

namespace py = pybind11;

namespace {

using at::Tensor;

[[noreturn]] void bad_value(const std::string& what) { throw py::value_error(what); }

std::string shape_of(const Tensor& t) {
  std::string s = "[";
  for (int64_t d = 0; d < t.dim(); ++d) s += (d ? ", " : "") + std::to_string(t.size(d));
  return s + "]";
}

// The operators compute on HIP devices only; anything else is an error.
void need_hip(const Tensor& t, const char* what) {
  if (!t.is_cuda())
    throw std::runtime_error(std::string(what) + " is on " + t.device().str() +
                             "; minispeed_amd.ops runs HIP kernels and needs tensors on a ROCm "
                             "GPU (device 'cuda')");
}

// The kernels have no forward-mode derivatives; run below autograd they would drop a tangent.
void need_no_tangent(const Tensor& t, const char* what) {
  TORCH_CHECK_NOT_IMPLEMENTED(
      !c10::AutogradState::get_tls_state().get_fw_grad_mode() || !t._fw_grad(0).defined(), what,
      " has a tangent; minispeed_amd.ops has no forward-mode derivatives");
}

void need_device(const Tensor& t, const Tensor& like, const char* what) {
  if (t.device() != like.device())
    throw std::runtime_error(std::string(what) + " is on " + t.device().str() + ", expected " +
                             like.device().str());
}

int32_t dtype_of(at::ScalarType t, const char* what) {
  switch (t) {
    case at::kFloat: return MS_OPS_F32;
    case at::kHalf: return MS_OPS_F16;
    case at::kBFloat16: return MS_OPS_BF16;
    default:
      throw py::type_error(std::string(what) + " has dtype " + c10::toString(t) +
                           "; expected float32, float16 or bfloat16");
  }
}

void check(int rc, const char* what) {
  if (rc != 0)
    throw std::runtime_error(std::string(what) + " failed with code " + std::to_string(rc) + ": " +
                             ms_ops_error_string(rc));
}

// Leading dimensions 0 .. dims-1 as (inner, outer_stride, inner_stride);
// false when they need more than two strides.
bool two_strides(const Tensor& t, int64_t dims, int64_t& inner, int64_t& outer_stride,
                 int64_t& inner_stride) {
  int64_t size[2] = {1, 1}, stride[2] = {0, 0};
  int k = -1;
  for (int64_t d = dims - 1; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (k >= 0 && t.stride(d) == size[k] * stride[k]) {
      size[k] *= t.size(d);
      continue;
    }
    if (++k == 2) return false;
    size[k] = t.size(d);
    stride[k] = t.stride(d);
  }
  inner = size[0] > 0 ? size[0] : 1;
  inner_stride = stride[0];
  outer_stride = stride[1];
  return true;
}

int64_t product(const Tensor& t, int64_t dims) {
  int64_t n = 1;
  for (int64_t d = 0; d < dims; ++d) n *= t.size(d);
  return n;
}

// A tensor [..., width] as rows; `hold` keeps the copy where the layout needs one.
ms_rows_t rows_of(const Tensor& t, const char* what, Tensor& hold) {
  ms_rows_t m{};
  m.dtype = dtype_of(t.scalar_type(), what);
  if (t.dim() < 1) bad_value(std::string(what) + " needs at least one dimension");
  const int64_t dims = t.dim() - 1;
  m.width = t.size(dims);
  m.n = product(t, dims);
  hold = t;
  if ((m.width > 1 && t.stride(dims) != 1) ||
      !two_strides(t, dims, m.inner, m.outer_stride, m.inner_stride)) {
    hold = t.contiguous();
    two_strides(hold, dims, m.inner, m.outer_stride, m.inner_stride);
  }
  m.data = hold.data_ptr();
  return m;
}

ms_tokens_t tokens_of(const Tensor& t, const char* what, Tensor& hold) {
  ms_tokens_t k{};
  if (t.scalar_type() != at::kLong && t.scalar_type() != at::kInt)
    throw py::type_error(std::string(what) + " has dtype " + c10::toString(t.scalar_type()) +
                         "; expected int64 or int32");
  k.wide = t.scalar_type() == at::kLong;
  k.n = t.numel();
  hold = t;
  if (!two_strides(t, t.dim(), k.inner, k.outer_stride, k.inner_stride)) {
    hold = t.contiguous();
    two_strides(hold, t.dim(), k.inner, k.outer_stride, k.inner_stride);
  }
  k.data = hold.data_ptr();
  return k;
}

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

Tensor make(const Tensor& like, at::IntArrayRef shape, at::ScalarType type) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(like.device()));
}

Tensor scratch(const Tensor& like, int64_t bytes) {
  if (bytes < 0) bad_value("sizes too large");
  return bytes ? make(like, {bytes}, at::kByte) : Tensor();
}
void* data_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// One float per row, dense, on the logits' device.
const float* per_row(const std::optional<Tensor>& t, const Tensor& logits, int64_t n,
                     const char* what, Tensor& hold) {
  if (!t) return nullptr;
  need_device(*t, logits, what);
  if (t->scalar_type() != at::kFloat)
    throw py::type_error(std::string(what) + " has dtype " + c10::toString(t->scalar_type()) +
                         "; expected float32");
  if (t->numel() != n)
    bad_value(std::string(what) + " has shape " + shape_of(*t) + ", expected one value for each of " +
              std::to_string(n) + " rows");
  hold = t->contiguous();
  return static_cast<const float*>(hold.data_ptr());
}

// ---------------------------------------------------------------------------

Tensor embedding(const Tensor& ids, const Tensor& weight, double scale) {
  need_no_tangent(weight, "weight");
  need_hip(weight, "weight");
  need_device(ids, weight, "ids");
  if (weight.dim() != 2) bad_value("weight has shape " + shape_of(weight) + ", expected [rows, width]");
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(weight.device());
  Tensor hold_w, hold_i;
  const ms_rows_t w = rows_of(weight, "weight", hold_w);
  const ms_tokens_t k = tokens_of(ids, "ids", hold_i);
  if (k.n && w.width && !w.n) bad_value("weight has no rows");
  std::vector<int64_t> shape(ids.sizes().begin(), ids.sizes().end());
  shape.push_back(w.width);
  Tensor out = make(weight, shape, weight.scalar_type());
  check(ms_embedding(&k, &w, static_cast<float>(scale), out.data_ptr(), stream_of(weight)),
        "ms_embedding");
  return out;
}

Tensor embedding_grad(const Tensor& grad, const Tensor& ids, int64_t rows, double scale,
                      int64_t padding_idx) {
  need_no_tangent(grad, "grad");
  need_hip(grad, "grad");
  need_device(ids, grad, "ids");
  if (rows < 0) bad_value("rows is " + std::to_string(rows));
  bool match = grad.dim() == ids.dim() + 1;
  for (int64_t d = 0; match && d < ids.dim(); ++d) match = grad.size(d) == ids.size(d);
  if (!match)
    bad_value("grad has shape " + shape_of(grad) + ", expected that of ids " + shape_of(ids) +
              " and a width");
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(grad.device());
  Tensor hold_g, hold_i;
  const ms_rows_t g = rows_of(grad, "grad", hold_g);
  const ms_tokens_t k = tokens_of(ids, "ids", hold_i);
  Tensor out = make(grad, {rows, g.width}, grad.scalar_type());
  const int64_t bytes = ms_embedding_grad_workspace(k.n, rows, g.width);
  const Tensor work = scratch(grad, bytes);
  check(ms_embedding_grad(&k, &g, rows, static_cast<float>(scale), padding_idx, out.data_ptr(),
                          data_of(work), bytes, stream_of(grad)),
        "ms_embedding_grad");
  return out;
}

void need_targets(const Tensor& logits, const Tensor& targets) {
  need_no_tangent(logits, "logits");
  need_hip(logits, "logits");
  need_device(targets, logits, "targets");
  bool match = logits.dim() >= 1 && targets.dim() == logits.dim() - 1;
  for (int64_t d = 0; match && d < targets.dim(); ++d) match = targets.size(d) == logits.size(d);
  if (!match)
    bad_value("targets has shape " + shape_of(targets) + ", expected the leading dimensions of logits " +
              shape_of(logits));
  if (logits.size(-1) < 1 || logits.size(-1) > std::numeric_limits<int32_t>::max())
    bad_value("logits has shape " + shape_of(logits) + ", expected a vocabulary of 1 to 2^31 - 1");
}

py::object wrap(const Tensor& t) {
  return t.defined() ? py::reinterpret_steal<py::object>(THPVariable_Wrap(t)) : py::none();
}

py::tuple token_logprobs(const Tensor& logits, const Tensor& targets, int64_t top, bool entropy,
                         int64_t ignore_index) {
  need_targets(logits, targets);
  if (top < 0 || top > MS_OPS_MAX_TOP || top > logits.size(-1))
    bad_value("top is " + std::to_string(top) + ", expected 0 to " +
              std::to_string(std::min<int64_t>(MS_OPS_MAX_TOP, logits.size(-1))));
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(logits.device());
  Tensor hold_l, hold_t;
  const ms_rows_t x = rows_of(logits, "logits", hold_l);
  const ms_tokens_t y = tokens_of(targets, "targets", hold_t);
  const Tensor logprob = make(logits, targets.sizes(), at::kFloat);
  const Tensor lse = make(logits, targets.sizes(), at::kFloat);
  const Tensor ent = entropy ? make(logits, targets.sizes(), at::kFloat) : Tensor();
  Tensor top_logprob, top_id;
  if (top) {
    std::vector<int64_t> shape(targets.sizes().begin(), targets.sizes().end());
    shape.push_back(top);
    top_logprob = make(logits, shape, at::kFloat);
    top_id = make(logits, shape, at::kLong);
  }
  const int64_t bytes =
      ms_logprobs_workspace(x.n, x.width, x.dtype, static_cast<int32_t>(top));
  const Tensor work = scratch(logits, bytes);
  check(ms_logprobs(&x, &y, ignore_index, static_cast<int32_t>(top),
                    static_cast<float*>(logprob.data_ptr()), static_cast<float*>(data_of(ent)),
                    static_cast<float*>(lse.data_ptr()), static_cast<float*>(data_of(top_logprob)),
                    static_cast<int64_t*>(data_of(top_id)), data_of(work), bytes,
                    stream_of(logits)),
        "ms_logprobs");
  return py::make_tuple(wrap(logprob), wrap(ent), wrap(lse), wrap(top_logprob), wrap(top_id));
}

Tensor token_logprobs_grad(const Tensor& logits, const Tensor& targets, const Tensor& lse,
                           const std::optional<Tensor>& grad_logprob,
                           const std::optional<Tensor>& entropy,
                           const std::optional<Tensor>& grad_entropy, int64_t ignore_index) {
  need_no_tangent(lse, "lse");
  if (grad_logprob) need_no_tangent(*grad_logprob, "grad_logprob");
  if (entropy) need_no_tangent(*entropy, "entropy");
  if (grad_entropy) need_no_tangent(*grad_entropy, "grad_entropy");
  need_targets(logits, targets);
  if (grad_entropy && !entropy) bad_value("grad_entropy needs entropy");
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(logits.device());
  Tensor hold_x, hold_t, hold[4];
  const ms_rows_t x = rows_of(logits, "logits", hold_x);
  const ms_tokens_t y = tokens_of(targets, "targets", hold_t);
  const float* l = per_row(lse, logits, x.n, "lse", hold[0]);
  const float* g = per_row(grad_logprob, logits, x.n, "grad_logprob", hold[1]);
  const float* h = per_row(grad_entropy, logits, x.n, "grad_entropy", hold[2]);
  const float* e = h ? per_row(entropy, logits, x.n, "entropy", hold[3]) : nullptr;
  const Tensor out = make(logits, logits.sizes(), logits.scalar_type());
  check(ms_logprobs_grad(&x, &y, ignore_index, l, e, g, h, out.data_ptr(), stream_of(logits)),
        "ms_logprobs_grad");
  return out;
}

int64_t blocks_of(int64_t n) { return (n + MS_OPS_BLOCK - 1) / MS_OPS_BLOCK; }

py::tuple pack8(const Tensor& x) {
  need_no_tangent(x, "x");
  need_hip(x, "x");
  const int32_t type = dtype_of(x.scalar_type(), "x");
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(x.device());
  const Tensor dense = x.contiguous();
  const int64_t n = x.numel();
  const Tensor codes = make(x, {n}, at::kChar);
  const Tensor exponents = make(x, {blocks_of(n)}, at::kByte);
  check(ms_pack8(dense.data_ptr(), type, n, static_cast<int8_t*>(codes.data_ptr()),
                 static_cast<uint8_t*>(exponents.data_ptr()), stream_of(x)),
        "ms_pack8");
  return py::make_tuple(wrap(codes), wrap(exponents));
}

void need_held(const Tensor& codes, const Tensor& exponents, int64_t n) {
  need_hip(codes, "codes");
  need_device(exponents, codes, "exponents");
  if (codes.scalar_type() != at::kChar || exponents.scalar_type() != at::kByte)
    throw py::type_error("codes and exponents are int8 and uint8");
  if (codes.numel() != n || exponents.numel() != blocks_of(n) || !codes.is_contiguous() ||
      !exponents.is_contiguous())
    bad_value("codes " + shape_of(codes) + " and exponents " + shape_of(exponents) +
              " do not hold " + std::to_string(n) + " values");
}

Tensor unpack8(const Tensor& codes, const Tensor& exponents, const std::vector<int64_t>& shape,
               py::object dtype) {
  if (!THPDtype_Check(dtype.ptr()))
    throw py::type_error("the checkpoint's dtype is " + std::string(py::repr(dtype)) +
                         ", expected a torch.dtype");
  const at::ScalarType as = reinterpret_cast<THPDtype*>(dtype.ptr())->scalar_type;
  const int32_t type = dtype_of(as, "the checkpoint");
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(codes.device());
  int64_t n = 1;
  for (int64_t s : shape) n *= s;
  need_held(codes, exponents, n);
  const Tensor out = make(codes, shape, as);
  check(ms_unpack8(static_cast<const int8_t*>(codes.data_ptr()),
                   static_cast<const uint8_t*>(exponents.data_ptr()), n, type, out.data_ptr(),
                   stream_of(codes)),
        "ms_unpack8");
  return out;
}

py::tuple act8(const Tensor& h, const std::optional<Tensor>& up, int64_t kind) {
  need_no_tangent(h, "h");
  if (up) need_no_tangent(*up, "up");
  need_hip(h, "h");
  if ((kind == MS_ACT_SWIGLU) != up.has_value())
    bad_value(up ? "up is for the gated kind only" : "the gated kind needs up");
  if (up) {
    need_device(*up, h, "up");
    if (up->scalar_type() != h.scalar_type())
      throw py::type_error("up has another dtype than h");
    if (up->sizes() != h.sizes())
      bad_value("up has shape " + shape_of(*up) + ", expected " + shape_of(h));
  }
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(h.device());
  Tensor hold_h, hold_u;
  const ms_rows_t x = rows_of(h, "h", hold_h);
  const ms_rows_t u = up ? rows_of(*up, "up", hold_u) : ms_rows_t{};
  const int64_t n = h.numel();
  const Tensor a = make(h, h.sizes(), h.scalar_type());
  Tensor codes[2], exponents[2];
  for (int k = 0; k < (up ? 2 : 1); ++k) {
    codes[k] = make(h, {n}, at::kChar);
    exponents[k] = make(h, {blocks_of(n)}, at::kByte);
  }
  check(ms_act8(&x, up ? &u : nullptr, static_cast<int32_t>(kind), a.data_ptr(),
                static_cast<int8_t*>(codes[0].data_ptr()),
                static_cast<uint8_t*>(exponents[0].data_ptr()),
                static_cast<int8_t*>(data_of(codes[1])),
                static_cast<uint8_t*>(data_of(exponents[1])), stream_of(h)),
        "ms_act8");
  return py::make_tuple(wrap(a), wrap(codes[0]), wrap(exponents[0]), wrap(codes[1]),
                        wrap(exponents[1]));
}

py::tuple act8_grad(const Tensor& codes, const Tensor& exponents,
                    const std::optional<Tensor>& up_codes,
                    const std::optional<Tensor>& up_exponents, const Tensor& grad, int64_t kind,
                    bool again) {
  need_no_tangent(grad, "grad");
  need_hip(grad, "grad");
  const int32_t type = dtype_of(grad.scalar_type(), "grad");
  const bool gated = kind == MS_ACT_SWIGLU;
  if (gated != up_codes.has_value() || gated != up_exponents.has_value())
    bad_value(gated ? "the gated kind needs two checkpoints" : "one checkpoint is expected");
  need_device(codes, grad, "codes");
  need_held(codes, exponents, grad.numel());
  if (gated) {
    need_device(*up_codes, grad, "up_codes");
    need_held(*up_codes, *up_exponents, grad.numel());
  }
  at::AutoDispatchBelowADInplaceOrView below;
  const c10::DeviceGuard guard(grad.device());
  const Tensor g = grad.contiguous();
  const Tensor dh = make(grad, grad.sizes(), grad.scalar_type());
  const Tensor dup = gated ? make(grad, grad.sizes(), grad.scalar_type()) : Tensor();
  const Tensor a = again ? make(grad, grad.sizes(), grad.scalar_type()) : Tensor();
  check(ms_act8_grad(static_cast<const int8_t*>(codes.data_ptr()),
                     static_cast<const uint8_t*>(exponents.data_ptr()),
                     gated ? static_cast<const int8_t*>(up_codes->data_ptr()) : nullptr,
                     gated ? static_cast<const uint8_t*>(up_exponents->data_ptr()) : nullptr,
                     g.data_ptr(), type, static_cast<int32_t>(kind), grad.numel(), dh.data_ptr(),
                     data_of(dup), data_of(a), stream_of(grad)),
        "ms_act8_grad");
  return py::make_tuple(wrap(dh), wrap(dup), wrap(a));
}

}  // namespace

PYBIND11_MODULE(_ops, m) {
  using torch::wrap_pybind_function;
  m.doc() = "language-model operators: argument checks, outputs and launches";
  m.def("abi_version", &ms_ops_abi_version);
  m.def("embedding", wrap_pybind_function(embedding));
  m.def("embedding_grad", wrap_pybind_function(embedding_grad));
  m.def("token_logprobs", wrap_pybind_function(token_logprobs));
  m.def("token_logprobs_grad", wrap_pybind_function(token_logprobs_grad));
  m.def("pack8", wrap_pybind_function(pack8));
  m.def("unpack8", wrap_pybind_function(unpack8));
  m.def("act8", wrap_pybind_function(act8));
  m.def("act8_grad", wrap_pybind_function(act8_grad));
}
