// torch binding of include/wc_fp8.h: argument checks, output tensors, the
// current stream.  The calls of a small batch take a few microseconds on the
// GPU, less than the same checks and allocations take in Python.  The C
// functions come in as addresses of the library that witchcraft_b200._lib
// loaded, so there is one instance of it.
#include <ATen/ATen.h>
#include <ATen/EmptyTensor.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <string>

#include "../../include/wc_fp8.h"

namespace py = pybind11;
using at::Tensor;

namespace {

struct Api {
  decltype(&wc_fp8_quantize_rows) rows = nullptr;
  decltype(&wc_fp8_quantize_weight) weight = nullptr;
  decltype(&wc_fp8_rmsnorm) rmsnorm = nullptr;
  decltype(&wc_fp8_matmul) matmul = nullptr;
  decltype(&wc_fp8_gated_matmul) gated = nullptr;
  decltype(&wc_fp8_last_error) error = nullptr;
} api;

constexpr int64_t kBlock = 128;
int64_t blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }

[[noreturn]] void refuse(const std::string& msg) { throw py::value_error(msg); }

std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}
std::string shape(int64_t r, int64_t c) { return "(" + std::to_string(r) + ", " + std::to_string(c) + ")"; }

// Nothing here has a gradient: results would leave the graph without a word.
void no_grad(const Tensor& t, const char* name) {
  if (t.requires_grad() && at::GradMode::is_enabled())
    refuse(std::string(name) + " requires grad, and the 8-bit operators have no gradient; call them under torch.no_grad()");
}
// What autograd saved of `out` is another value now.
void written(const Tensor& out) {
  if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}

void matrix(const Tensor& t, const char* name, const Tensor& like) {
  no_grad(t, name);
  if (!t.is_cuda() || t.dim() != 2 || (t.stride(1) != 1 && t.size(1) > 1))
    refuse(std::string(name) + " must be a CUDA matrix with contiguous rows");
  if (t.get_device() != like.get_device())
    refuse(std::string(name) + " is on " + t.device().str() + ", not on " + like.device().str());
}
void sized(const Tensor& t, const char* name, int64_t r, int64_t c) {
  if (t.size(0) != r || t.size(1) != c)
    refuse(std::string(name) + " has shape " + shape_of(t) + ", expected " + shape(r, c));
}
int type_code(at::ScalarType t) {
  return t == at::kFloat ? WC_T_F32 : t == at::kHalf ? WC_T_F16 : t == at::kBFloat16 ? WC_T_BF16 : -1;
}
int values(const Tensor& t, const char* name, const Tensor& like) {
  matrix(t, name, like);
  const int code = type_code(t.scalar_type());
  if (code < 0)
    refuse(std::string(name) + " must be float32, float16 or bfloat16, not " + c10::toString(t.scalar_type()));
  return code;
}
void columns(const Tensor& t, const char* name) {
  if (t.size(1) < 1) refuse(std::string(name) + " has no columns");
}
void operand(const Tensor& codes, const Tensor& scales, const char* name, const Tensor& like, int64_t rows_per_scale) {
  matrix(codes, name, like);
  if (codes.scalar_type() != at::kFloat8_e4m3fn)
    refuse(std::string(name) + " must be float8_e4m3fn codes, not " + c10::toString(codes.scalar_type()));
  columns(codes, name);
  const std::string sname = std::string("scales of ") + name;
  matrix(scales, sname.c_str(), like);
  sized(scales, sname.c_str(), (codes.size(0) + rows_per_scale - 1) / rows_per_scale, blocks(codes.size(1)));
  if (scales.scalar_type() != at::kFloat)
    refuse(sname + " must be float32, not " + c10::toString(scales.scalar_type()));
}

// Leading dimensions; a single row may have any stride.
int64_t ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1)); }
int64_t codes_ld(const Tensor& t) {
  return t.size(0) > 1 ? t.stride(0) : (std::max(t.stride(0), t.size(1)) + 15) / 16 * 16;
}

// An uninitialised tensor on the current device (the callers' guards make it
// the operands'): torch's CUDA allocator without its dispatcher.
Tensor empty_bytes(c10::IntArrayRef sizes, at::ScalarType type) {
  return at::detail::empty_generic(sizes, c10::cuda::CUDACachingAllocator::get(),
                                   c10::DispatchKeySet(c10::DispatchKey::CUDA), type, std::nullopt);
}
Tensor empty(int64_t r, int64_t c, at::ScalarType type) { return empty_bytes({r, c}, type); }
// Codes [r][c] and scales [sr][ceil(c / 128)] in one allocation (an allocation
// costs about as much as a launch): two tensors over one storage.
std::tuple<Tensor, Tensor> empty_quantized(int64_t r, int64_t c, int64_t sr) {
  const int64_t wide = (c + 15) / 16 * 16, kb = blocks(c), offset = (r * wide + 255) / 256 * 64;  // in floats
  const Tensor buf = empty_bytes({4 * (offset + sr * kb)}, at::kByte);
  auto over = [&](at::ScalarType type, int64_t at0, int64_t rows, int64_t cols, int64_t ld) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buf.storage()), buf.key_set(),
                                                        c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_storage_offset(at0);
    t.unsafeGetTensorImpl()->set_sizes_and_strides(c10::IntArrayRef{rows, cols}, c10::IntArrayRef{ld, 1});
    return t;
  };
  return {over(at::kFloat8_e4m3fn, 0, r, c, wide), over(at::kFloat, offset, sr, kb, kb)};
}

float* floats(const Tensor& t) { return static_cast<float*>(t.data_ptr()); }

void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

void check(int rc) {
  if (rc == 0) return;
  const char* msg = api.error();
  const py::object error = py::module_::import("witchcraft_b200._lib").attr("WcError");
  const py::object e = error(rc, std::string(msg ? msg : ""));
  PyErr_SetObject(error.ptr(), e.ptr());
  throw py::error_already_set();
}

using Pair = std::tuple<Tensor, Tensor>;

Pair quantize(const Tensor& x) {
  const int code = values(x, "x", x);
  columns(x, "x");
  const int64_t m = x.size(0), k = x.size(1);
  const c10::cuda::CUDAGuard guard(x.device());
  auto [codes, scales] = empty_quantized(m, k, m);
  if (m)
    check(api.rows(x.data_ptr(), code, m, k, ld(x), codes.data_ptr(), codes_ld(codes), floats(scales), scales.size(1),
                   stream_of(x)));
  return {codes, scales};
}

Pair quantize_weight(const Tensor& w) {
  const int code = values(w, "w", w);
  const int64_t n = w.size(0), k = w.size(1);
  if (n < 1 || k < 1) refuse("w is empty");
  const c10::cuda::CUDAGuard guard(w.device());
  auto [codes, scales] = empty_quantized(n, k, blocks(n));
  check(api.weight(w.data_ptr(), code, n, k, ld(w), codes.data_ptr(), codes_ld(codes), floats(scales), scales.size(1),
                   stream_of(w)));
  return {codes, scales};
}

py::tuple rmsnorm(const Tensor& x, const Tensor& weight, double eps, const std::optional<Tensor>& delta,
                  const std::optional<Tensor>& out) {
  const int code = values(x, "x", x);
  columns(x, "x");
  const int64_t m = x.size(0), k = x.size(1);
  no_grad(weight, "weight");
  if (weight.scalar_type() != at::kFloat || weight.dim() != 1 || weight.size(0) != k || !weight.is_cuda() ||
      weight.get_device() != x.get_device() || (weight.stride(0) != 1 && k > 1))
    refuse("weight must be " + std::to_string(k) + " contiguous float32 values on " + x.device().str());
  if (!(eps >= 0)) refuse("eps must not be negative");
  if (out && !delta) refuse("out is the sum with delta; there is no delta");
  int dcode = 0;
  if (delta) {
    dcode = values(*delta, "delta", x);
    sized(*delta, "delta", m, k);
    if (out) {
      if (values(*out, "out", x) != code) refuse(std::string("out must have x's type ") + c10::toString(x.scalar_type()));
      sized(*out, "out", m, k);
    }
  }
  const c10::cuda::CUDAGuard guard(x.device());
  Tensor sum = !delta ? Tensor() : out ? *out : empty(m, k, x.scalar_type());
  auto [codes, scales] = empty_quantized(m, k, m);
  if (m)
    check(api.rmsnorm(x.data_ptr(), code, ld(x), delta ? delta->data_ptr() : nullptr, dcode, delta ? ld(*delta) : 0,
                      delta ? sum.data_ptr() : nullptr, delta ? ld(sum) : 0, floats(weight), m, k,
                      static_cast<float>(eps), codes.data_ptr(), codes_ld(codes), floats(scales), scales.size(1),
                      stream_of(x)));
  if (out) written(*out);
  return delta ? py::make_tuple(sum, codes, scales) : py::make_tuple(codes, scales);
}

Tensor matmul(const Tensor& a, const Tensor& a_scales, const Tensor& w, const Tensor& w_scales,
              const std::optional<at::ScalarType>& out_dtype, const std::optional<Tensor>& residual,
              const std::optional<Tensor>& out) {
  operand(a, a_scales, "a", a, 1);
  operand(w, w_scales, "w", a, kBlock);
  const int64_t m = a.size(0), k = a.size(1), n = w.size(0);
  if (w.size(1) != k || n < 1)
    refuse("w has shape " + shape_of(w) + ", expected [n >= 1, " + std::to_string(k) + "]");
  at::ScalarType type = out_dtype.value_or(at::kHalf);
  if (residual) {
    values(*residual, "residual", a);
    sized(*residual, "residual", m, n);
    type = residual->scalar_type();
  }
  const int code = type_code(type);
  if (code < 0) refuse(std::string("out_dtype must be float32, float16 or bfloat16, not ") + c10::toString(type));
  const c10::cuda::CUDAGuard guard(a.device());
  Tensor y;
  if (out) {
    if (values(*out, "out", a) != code)
      refuse(std::string("out is ") + c10::toString(out->scalar_type()) + ", expected " + c10::toString(type));
    sized(*out, "out", m, n);
    y = *out;
  } else {
    y = empty(m, n, type);
  }
  if (m)
    check(api.matmul(a.data_ptr(), codes_ld(a), floats(a_scales), ld(a_scales), m, k, w.data_ptr(), codes_ld(w),
                     floats(w_scales), ld(w_scales), n, residual ? residual->data_ptr() : nullptr,
                     residual ? ld(*residual) : 0, y.data_ptr(), code, ld(y), stream_of(a)));
  if (out) written(*out);
  return y;
}

py::object gated_matmul(const Tensor& a, const Tensor& a_scales, const Tensor& gate, const Tensor& gate_scales,
                        const Tensor& up, const Tensor& up_scales, const std::optional<at::ScalarType>& out_dtype,
                        const std::string& act) {
  operand(a, a_scales, "a", a, 1);
  operand(gate, gate_scales, "gate", a, kBlock);
  operand(up, up_scales, "up", a, kBlock);
  const int64_t m = a.size(0), k = a.size(1), n = gate.size(0);
  if (gate.size(1) != k || n < 1 || up.size(0) != n || up.size(1) != k)
    refuse("gate " + shape_of(gate) + " and up " + shape_of(up) + " must both be [n >= 1, " + std::to_string(k) + "]");
  const int acode = act == "gelu" ? WC_ACT_GELU : act == "silu" ? WC_ACT_SILU : -1;
  if (acode < 0) refuse("act must be 'gelu' or 'silu', not '" + act + "'");
  const int code = out_dtype ? type_code(*out_dtype) : WC_T_E4M3;
  if (code < 0)
    refuse(std::string("out_dtype must be None, float32, float16 or bfloat16, not ") + c10::toString(*out_dtype));
  const c10::cuda::CUDAGuard guard(a.device());
  Tensor y, scales;
  if (out_dtype)
    y = empty(m, n, *out_dtype);
  else
    std::tie(y, scales) = empty_quantized(m, n, m);
  if (m)
    check(api.gated(a.data_ptr(), codes_ld(a), floats(a_scales), ld(a_scales), m, k, gate.data_ptr(), codes_ld(gate),
                    floats(gate_scales), ld(gate_scales), up.data_ptr(), codes_ld(up), floats(up_scales),
                    ld(up_scales), n, acode, y.data_ptr(), code, out_dtype ? ld(y) : codes_ld(y),
                    out_dtype ? nullptr : floats(scales), out_dtype ? 0 : scales.size(1), stream_of(a)));
  return out_dtype ? py::cast(y) : py::object(py::make_tuple(y, scales));
}

}  // namespace

PYBIND11_MODULE(_fp8_torch, m) {
  m.def("bind", [](uintptr_t rows, uintptr_t weight, uintptr_t rmsnorm, uintptr_t matmul, uintptr_t gated,
                   uintptr_t error) {
    api.rows = reinterpret_cast<decltype(api.rows)>(rows);
    api.weight = reinterpret_cast<decltype(api.weight)>(weight);
    api.rmsnorm = reinterpret_cast<decltype(api.rmsnorm)>(rmsnorm);
    api.matmul = reinterpret_cast<decltype(api.matmul)>(matmul);
    api.gated = reinterpret_cast<decltype(api.gated)>(gated);
    api.error = reinterpret_cast<decltype(api.error)>(error);
  });
  m.def("quantize", &quantize);
  m.def("quantize_weight", &quantize_weight);
  m.def("rmsnorm", &rmsnorm);
  m.def("matmul", &matmul);
  m.def("gated_matmul", &gated_matmul);
}
