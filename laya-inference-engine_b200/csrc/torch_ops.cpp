// The calls of laya_b200/ops.py on torch tensors (module laya_b200._torch_ops):
// argument checks, output and workspace allocation through torch, and the C ABI
// of include/laya_b200.h on the tensors' device and its current stream.  In C++
// because a single row is bound by its host time: the same checks in Python took
// 19 us a projection and 20 us a quantised norm.  Refusals raise ValueError
// before anything is launched, failures of the library RuntimeError.
#include "laya_b200.h"

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/DynamicTypes.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <initializer_list>
#include <sstream>
#include <string>
#include <vector>

namespace {

using at::ScalarType;
using at::Tensor;

constexpr ScalarType kBF16 = ScalarType::BFloat16, kF32 = ScalarType::Float, kE4M3 = ScalarType::Float8_e4m3fn;

[[noreturn]] void refuse(const std::string& m) {
  throw c10::ValueError({__func__, __FILE__, static_cast<uint32_t>(__LINE__)}, m);
}

std::string shape_of(at::IntArrayRef s) {
  std::ostringstream o;
  o << "(";
  for (size_t i = 0; i < s.size(); ++i) o << (i ? ", " : "") << s[i];
  o << ")";
  return o.str();
}

// A tensor argument, or a null pointer for None.
const Tensor* tensor(PyObject* o, const char* name, bool needed) {
  if (o == Py_None && !needed) return nullptr;
  if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
  return &THPVariable_Unpack(o);
}

struct Rows {
  int64_t rows, columns, stride;
};

// A [..., columns] tensor whose rows lie at one stride and do not overlap.
Rows rows_of(const char* name, const Tensor& t, std::initializer_list<ScalarType> types, int64_t columns = -1) {
  bool known = false;
  for (auto s : types) known = known || t.scalar_type() == s;
  if (!known) {
    std::string m = std::string(name) + " must be a tensor of ";
    for (auto s : types) m += std::string(s == *types.begin() ? "" : " or ") + c10::toString(s);
    refuse(m);
  }
  const auto shape = t.sizes(), strides = t.strides();
  const int64_t dims = t.dim();
  if (dims < 1 || (columns >= 0 && shape[dims - 1] != columns))
    refuse(std::string(name) + " must have " + (columns >= 0 ? std::to_string(columns) : std::string("some")) +
           " columns; got shape " + shape_of(shape));
  const int64_t n = shape[dims - 1];
  int64_t rows = 1, stride = n, outer = -1;  // outer: stride an axis further out has to have
  for (int64_t d = dims - 2; d >= 0; --d) {
    rows *= shape[d];
    if (shape[d] <= 1) continue;
    if (outer < 0)
      stride = strides[d];
    else if (strides[d] != outer)
      refuse(std::string(name) + "'s rows must lie at one stride; got strides " + shape_of(strides));
    outer = strides[d] * shape[d];
  }
  if (n > 1 && strides[dims - 1] != 1) refuse(std::string(name) + "'s columns must be contiguous");
  if (rows <= 1)
    stride = n;
  else if (stride < n)
    refuse(std::string(name) + "'s rows overlap");
  return {rows, n, stride};
}

void contiguous(const char* name, const Tensor& t, at::IntArrayRef shape, ScalarType type) {
  if (t.scalar_type() != type || t.sizes() != shape || !t.is_contiguous())
    refuse(std::string(name) + " must be a contiguous " + c10::toString(type) + " tensor of shape " + shape_of(shape));
}

// The CUDA device that all the tensors are on; tensors that a derivative would have
// to be recorded for are refused.
at::Device device_of(std::initializer_list<const Tensor*> all) {
  const Tensor& first = **all.begin();
  if (!first.is_cuda()) refuse("the operators run on CUDA tensors only");
  bool grad = false, tangent = false;
  for (const Tensor* t : all)
    if (t) {
      if (t->device() != first.device()) refuse("tensors on " + t->device().str() + " and " + first.device().str());
      grad = grad || t->requires_grad();
      tangent = tangent || t->_fw_grad(0).defined();
    }
  if (tangent && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    refuse("the operators compute no tangents; call them on fwAD.unpack_dual(x).primal");
  if (grad && c10::GradMode::is_enabled())
    refuse("the operators record no gradient; call them under torch.no_grad() or on detached tensors");
  return first.device();
}

// The bytes that t covers: [lo, hi), and, where its rows lie at one stride, that
// stride and their width.
struct Span {
  const char *lo, *hi;
  int64_t stride = 0, width = 0;
};
Span span_of(const Tensor& t) {
  Span s{static_cast<const char*>(t.data_ptr()), static_cast<const char*>(t.data_ptr())};
  if (t.numel() == 0) return s;
  const int64_t size = (int64_t)t.element_size(), dims = t.dim();
  int64_t last = 0, outer = -1;
  bool even = dims > 1 && (t.stride(dims - 1) == 1 || t.size(dims - 1) == 1);
  for (int64_t d = dims - 1; d >= 0; --d) last += (t.size(d) - 1) * t.stride(d);
  for (int64_t d = dims - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    if (outer < 0)
      s.stride = t.stride(d) * size;
    else
      even = even && t.stride(d) == outer;
    outer = t.stride(d) * t.size(d);
  }
  s.hi = s.lo + (last + 1) * size;
  s.width = dims ? t.size(dims - 1) * size : size;
  if (!even) s.stride = 0;
  return s;
}

// Whether no byte is in both: apart, or columns of the same rows.
bool apart(const Span& a, const Span& b) {
  if (a.lo >= b.hi || b.lo >= a.hi) return true;
  if (a.stride <= 0 || a.stride != b.stride) return false;
  const int64_t at = (((b.lo - a.lo) % a.stride) + a.stride) % a.stride;  // where b's rows begin in a's
  return at >= a.width && at + b.width <= a.stride;
}

void disjoint(const char* name, const Tensor& out, std::initializer_list<const Tensor*> others) {
  const Span s = span_of(out);
  for (const Tensor* t : others)
    if (t && !apart(s, span_of(*t))) refuse(std::string(name) + " overlaps another argument");
}

// A tensor that a call has written: autograd refuses a graph that saved what it
// held before, as it does after torch's in-place operators.  (Inference tensors have
// no version.)
void written(const Tensor* t) {
  if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}

void* ptr(const Tensor* t) { return t ? t->data_ptr() : nullptr; }

void check(const char* what, int status) {
  if (status) {
    const char* m = laya_b200_last_error(nullptr);
    TORCH_CHECK(false, what, ": ", m && *m ? m : "unknown error");
  }
}

int32_t narrow(const char* name, int64_t v) {
  if (v > INT32_MAX) refuse(std::string(name) + " is too large");
  return (int32_t)v;
}

// y, codes, scale: the outputs to write, where asked for.
void run_rms_norm(const Tensor& x, const Tensor* weight, double eps, const Tensor* residual, const Tensor* y,
                  bool y_given, const Tensor* codes, const Tensor* scale) {
  const Rows rx = rows_of("x", x, {kBF16, kF32});
  const int64_t d = rx.columns;
  if (d < 1 || d > 16384) refuse("x must have 1 to 16384 columns");
  if (!((float)eps > 0) || std::isinf((float)eps)) refuse("eps must be positive and finite in fp32");
  if (weight) contiguous("weight", *weight, {d}, kF32);
  laya_b200_rms_norm_args a{};
  if (residual) {
    a.residual_stride = rows_of("residual", *residual, {kBF16, kF32}, d).stride;
    if (residual->sizes() != x.sizes()) refuse("residual must have x's shape " + shape_of(x.sizes()));
    disjoint("residual", *residual, {&x, weight});
  }
  if (y) {
    a.y_stride = d;
    if (y_given) {
      a.y_stride = rows_of("out", *y, {kBF16, kF32}, d).stride;
      disjoint("out", *y, {weight, residual});
      if (y->data_ptr() != x.data_ptr() || y->scalar_type() != x.scalar_type() || a.y_stride != rx.stride)
        disjoint("out", *y, {&x});  // in place is allowed
    }
  }
  const at::Device dev = device_of({&x, weight, residual, y});
  if (rx.rows == 0) return;
  a.rows = narrow("rows", rx.rows);
  a.columns = (int32_t)d;
  a.eps = (float)eps;
  a.x_f32 = x.scalar_type() == kF32;
  a.residual_f32 = residual && residual->scalar_type() == kF32;
  a.y_f32 = y && y->scalar_type() == kF32;
  a.x = x.data_ptr();
  a.x_stride = rx.stride;
  a.residual = ptr(residual);
  a.weight = static_cast<const float*>(ptr(weight));
  a.y = ptr(y);
  a.codes = ptr(codes);
  a.codes_stride = d;
  a.scale = static_cast<float*>(ptr(scale));
  const c10::cuda::CUDAGuard guard(dev);
  check("rms_norm", laya_b200_rms_norm(&a, c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  written(residual);
  if (y_given) written(y);
}

// A new tensor beside x, without the dispatcher's microsecond (a tensor that is
// not on a GPU is refused later).
Tensor empty_beside(const Tensor& x, at::IntArrayRef sizes, ScalarType type) {
  if (!x.is_cuda()) return at::empty(sizes, x.options().dtype(type).requires_grad(false));
  return at::detail::empty_cuda(sizes, type, x.device(), c10::nullopt);
}

// rms_norm(x, weight, eps, residual, out, dtype)
PyObject* py_rms_norm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 6) refuse("rms_norm takes 6 arguments");
  const Tensor& x = *tensor(args[0], "x", true);
  const Tensor *weight = tensor(args[1], "weight", false), *residual = tensor(args[3], "residual", false);
  const double eps = PyFloat_AsDouble(args[2]);
  if (PyErr_Occurred()) throw python_error();
  ScalarType type = x.scalar_type();
  const bool typed = args[5] != Py_None;
  if (typed) {
    if (!THPDtype_Check(args[5])) refuse("dtype must be a torch.dtype");
    type = reinterpret_cast<THPDtype*>(args[5])->scalar_type;
  }
  const Tensor* given = tensor(args[4], "out", false);
  if (given && (given->sizes() != x.sizes() || (typed && given->scalar_type() != type)))
    refuse("out must have x's shape " + shape_of(x.sizes()) + (typed ? " and be of dtype" : ""));
  if (!given && type != kBF16 && type != kF32) refuse("dtype must be torch.bfloat16 or torch.float32");
  const Tensor out = given ? *given : empty_beside(x, x.sizes(), type);
  run_rms_norm(x, weight, eps, residual, &out, given != nullptr, nullptr, nullptr);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// rms_norm_quant(x, weight, eps, residual, rows) -> (codes, scale[, y])
PyObject* py_rms_norm_quant(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 5) refuse("rms_norm_quant takes 5 arguments");
  const Tensor& x = *tensor(args[0], "x", true);
  const Tensor *weight = tensor(args[1], "weight", false), *residual = tensor(args[3], "residual", false);
  const double eps = PyFloat_AsDouble(args[2]);
  if (PyErr_Occurred()) throw python_error();
  const int keep = PyObject_IsTrue(args[4]);
  if (keep < 0) throw python_error();
  if (x.dim() < 1) refuse("x must be a tensor of rows");
  const Tensor codes = empty_beside(x, x.sizes(), kE4M3);
  const Tensor scale = empty_beside(x, x.sizes().slice(0, x.dim() - 1), kF32);
  const Tensor y = keep ? empty_beside(x, x.sizes(), x.scalar_type()) : Tensor();
  run_rms_norm(x, weight, eps, residual, keep ? &y : nullptr, false, &codes, &scale);
  PyObject* out = PyTuple_New(keep ? 3 : 2);
  if (!out) throw python_error();
  PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(codes));
  PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(scale));
  if (keep) PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(y));
  return out;
  END_HANDLE_TH_ERRORS
}

// lora(x, codes, code_scale, weight, weight_scale, lora_a, lora_b, index, scaling, bias, rows_per_index, out)
PyObject* py_lora(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 12) refuse("lora takes 12 arguments");
  const Tensor& x = *tensor(args[0], "x", true);
  const Tensor* codes = tensor(args[1], "codes", false);
  const bool fp8 = codes != nullptr;
  const Tensor* code_scale = tensor(args[2], "scale", fp8);
  const Tensor& weight = *tensor(args[3], "weight", true);
  const Tensor* weight_scale = tensor(args[4], "weight_scale", fp8);
  const Tensor &la = *tensor(args[5], "lora_a", true), &lb = *tensor(args[6], "lora_b", true);
  const Tensor& index = *tensor(args[7], "index", true);
  const Tensor *scaling = tensor(args[8], "scaling", false), *bias = tensor(args[9], "bias", false);
  const int64_t per = PyLong_AsLongLong(args[10]);
  if (PyErr_Occurred()) throw python_error();
  const Tensor* given = tensor(args[11], "out", false);

  const Rows rx = rows_of("x", x, {kBF16});
  const int64_t k = rx.columns;
  const Rows rw = rows_of("weight", weight, {fp8 ? kE4M3 : kBF16}, k);
  if (weight.dim() != 2) refuse("weight must be [out_features, " + std::to_string(k) + "]");
  const int64_t n = rw.rows;
  if (la.dim() != 3) refuse("lora_a must be [slots, rank, in_features]");
  const int64_t slots = la.size(0), rank = la.size(1);
  contiguous("lora_a", la, {slots, rank, k}, kBF16);
  contiguous("lora_b", lb, {slots, n, rank}, kBF16);
  if (slots < 1 || rank % 8 || rank < 8 || rank > 256)
    refuse("the adapters need at least one slot and a rank that is a multiple of 8 up to 256");
  if (per < 1) refuse("rows_per_index must be positive");
  contiguous("index", index, {rx.rows / per + (rx.rows % per != 0)}, ScalarType::Int);
  if (scaling) contiguous("scaling", *scaling, {slots}, kF32);
  if (bias) contiguous("bias", *bias, {n}, kBF16);
  laya_b200_lora_args a{};
  if (fp8) {
    a.codes_stride = rows_of("codes", *codes, {kE4M3}, k).stride;
    if (codes->sizes() != x.sizes()) refuse("codes must have x's shape " + shape_of(x.sizes()));
    contiguous("scale", *code_scale, x.sizes().slice(0, x.dim() - 1), kF32);
    contiguous("weight_scale", *weight_scale, {n}, kF32);
  }
  if (k % (fp8 ? 16 : 8)) refuse(std::string("in_features must be a multiple of ") + (fp8 ? "16" : "8"));
  const at::Device dev =
      device_of({&x, codes, code_scale, &weight, weight_scale, &la, &lb, &index, scaling, bias, given});
  c10::SmallVector<int64_t, 5> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = n;
  a.out_stride = n;
  if (given) {
    if (given->sizes() != at::IntArrayRef(shape)) refuse("out must have shape " + shape_of(shape));
    a.out_stride = rows_of("out", *given, {kBF16}, n).stride;
    disjoint("out", *given, {&x, codes, code_scale, &weight, weight_scale, &la, &lb, &index, scaling, bias});
  }
  const Tensor out = given ? *given : empty_beside(x, shape, kBF16);
  if (rx.rows == 0 || n == 0) return THPVariable_Wrap(out);
  a.rows = narrow("rows", rx.rows);
  a.in_features = narrow("in_features", k);
  a.out_features = narrow("out_features", n);
  a.slots = narrow("slots", slots);
  a.rank = (int32_t)rank;
  a.rows_per_index = (int32_t)std::min<int64_t>(per, INT32_MAX);
  a.x = x.data_ptr();
  a.x_stride = rx.stride;
  a.codes = ptr(codes);
  a.code_scale = static_cast<const float*>(ptr(code_scale));
  a.weight = weight.data_ptr();
  a.weight_stride = rw.stride;
  a.weight_scale = static_cast<const float*>(ptr(weight_scale));
  a.lora_a = la.data_ptr();
  a.lora_b = lb.data_ptr();
  a.scaling = static_cast<const float*>(ptr(scaling));
  a.index = static_cast<const int32_t*>(index.data_ptr());
  a.bias = ptr(bias);
  a.out = out.data_ptr();
  const c10::cuda::CUDAGuard guard(dev);
  size_t bytes = 0;
  check("lora_linear", laya_b200_lora_workspace(&a, &bytes));
  // the caching allocator hands this memory to later work of this stream only
  const c10::DataPtr work = c10::cuda::CUDACachingAllocator::get()->allocate(bytes);
  check("lora_linear", laya_b200_lora_linear(&a, work.get(), bytes,
                                             c10::cuda::getCurrentCUDAStream(dev.index()).stream()));
  written(given);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

PyMethodDef kMethods[] = {
    {"rms_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_rms_norm)), METH_FASTCALL, nullptr},
    {"rms_norm_quant", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_rms_norm_quant)), METH_FASTCALL,
     nullptr},
    {"lora", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_lora)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__torch_ops() { return PyModule_Create(&kModule); }
