// The host's side of rows8.py's calls: checks of arguments, results from torch's allocator, the launch.  A Python extension, because a call for a few tokens is 1 to 8 us of GPU time, and
// the same work in Python (attributes, two or three allocations, a dozen numbers through ctypes) took 10 to 13.
//
// It calls the C ABI (include/mistral_b200_rows8.h) by addresses that bind() is given; what does not fit raises AssertionError, what the library refuses bind()'s error class.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../../include/mistral_b200_rows8.h"

namespace {

struct Library {
  decltype(&mb8_last_error) last_error;
  decltype(&mb8_quantise) quantise;
  decltype(&mb8_norm) norm;
  decltype(&mb8_multiply) multiply;
  decltype(&mb8_gate) gate;
  decltype(&mb8_product_scratch) product_scratch;
} lib = {};
PyObject* failure = nullptr;  // class of what the library refuses

constexpr int64_t BLOCK = 128;
constexpr const char* NO_FALLBACK = "libmb200_rows8 runs on CUDA only; no fallback exists";

#define ASSERT(cond, ...)                          \
  do {                                             \
    if (!(cond)) {                                 \
      PyErr_Format(PyExc_AssertionError, __VA_ARGS__); \
      throw python_error();                        \
    }                                              \
  } while (0)

int64_t width_of(int64_t cols) { return (cols + BLOCK - 1) / BLOCK * BLOCK; }

const at::Tensor& tensor(PyObject* o, const char* what) {
  ASSERT(THPVariable_Check(o), "%s: a tensor", what);
  return THPVariable_Unpack(o);
}
// bf16 or fp32 rows that do not overlap; rows may be part of wider ones
struct Numbers {
  void* at;
  int64_t T, K, ld;
  int wide, device;
};
Numbers numbers(PyObject* o, const char* what) {
  const at::Tensor& x = tensor(o, what);
  const auto type = x.scalar_type();
  ASSERT(x.dim() == 2 && (type == at::kBFloat16 || type == at::kFloat) && x.size(1) >= 1, "%s [rows, columns], bf16 or fp32, at least one column", what);
  Numbers n{nullptr, x.size(0), x.size(1), x.stride(0), type == at::kFloat, -1};
  ASSERT((x.stride(1) == 1 || n.K == 1) && (n.ld >= n.K || n.T <= 1), "%s: contiguous rows that do not overlap", what);
  ASSERT(x.is_cuda(), "%s: %s", what, NO_FALLBACK);
  n.at = x.data_ptr();
  n.device = x.get_device();
  return n;
}
// a matrix of 8-bit rows: codes, scales, columns
struct Rows {
  void *codes, *scales;
  int64_t T, K;
  int device;
};
Rows rows(PyObject* codes, PyObject* scales, int64_t K, const char* what) {
  const at::Tensor &c = tensor(codes, what), &s = tensor(scales, what);
  ASSERT(c.dim() == 2 && c.scalar_type() == at::kFloat8_e4m3fn && K >= 1 && c.size(1) == width_of(K), "%s: codes [rows, %lld] e4m3 of %lld columns", what, (long long)width_of(K), (long long)K);
  const int64_t T = c.size(0), tiles = (T + 127) / 128, quads = (K + 4 * BLOCK - 1) / (4 * BLOCK);
  ASSERT(s.scalar_type() == at::kFloat8_e8m0fnu && s.sizes() == at::IntArrayRef({tiles, quads, 32, 4, 4}), "%s: scales [%lld, %lld, 32, 4, 4] e8m0", what, (long long)tiles, (long long)quads);
  ASSERT(c.is_cuda(), "%s: %s", what, NO_FALLBACK);
  ASSERT(s.is_cuda() && s.get_device() == c.get_device() && c.is_contiguous() && s.is_contiguous(), "%s: contiguous codes and scales of one device", what);
  return {c.data_ptr(), s.data_ptr(), T, K, (int)c.get_device()};
}

at::Tensor make(at::IntArrayRef sizes, at::IntArrayRef strides, at::ScalarType type, int device) {
  return at::Tensor(at::detail::empty_strided_cuda(sizes, strides, type, at::Device(at::kCUDA, (c10::DeviceIndex)device)));
}
struct Result {
  at::Tensor codes, scales;
};
Result make_rows(int64_t T, int64_t K, int device) {
  const int64_t width = width_of(K), tiles = (T + 127) / 128, quads = (K + 4 * BLOCK - 1) / (4 * BLOCK);
  ASSERT(T <= MB8_MAX_ROWS && K <= MB8_MAX_ROWS, "%lld rows of %lld entries (at most %d)", (long long)T, (long long)K, MB8_MAX_ROWS);
  // one allocation for both, 0.4 us less than two
  at::Tensor codes = make({T * width + tiles * quads * 512}, {1}, at::kFloat8_e4m3fn, device);
  at::Tensor scales = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(codes.storage()), codes.key_set(), c10::scalarTypeToTypeMeta(at::kFloat8_e8m0fnu));
  scales.unsafeGetTensorImpl()->set_storage_offset(T * width);
  scales.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef({tiles, quads, 32, 4, 4}), at::IntArrayRef({quads * 512, 512, 16, 4, 1}));
  codes.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef({T, width}), at::IntArrayRef({width, 1}));
  return {std::move(codes), std::move(scales)};
}
PyObject* wrapped(const at::Tensor& t) { return THPVariable_Wrap(t); }
PyObject* pair_of(const Result& r) {
  PyObject* const t = PyTuple_New(2);
  if (t == nullptr) throw python_error();
  PyTuple_SET_ITEM(t, 0, wrapped(r.codes));
  PyTuple_SET_ITEM(t, 1, wrapped(r.scales));
  return t;
}

struct Unlocked {  // without the interpreter's lock
  PyThreadState* const state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};
// call(stream) on the device's current stream, whatever the current device is
template <typename F>
void launch(const char* what, int device, F call) {
  int rc;
  {
    const Unlocked unlocked;
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)device);
    rc = call((void*)c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream());
  }
  if (rc != 0) {
    PyErr_Format(failure, "%s failed (%d): %s", what, rc, lib.last_error());
    throw python_error();
  }
}

int64_t integer(PyObject* o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v != 0;
}
void arguments(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", want, n);
    throw python_error();
  }
}
void call_arguments(Py_ssize_t n, Py_ssize_t want) {
  arguments(n, want);
  ASSERT(failure != nullptr, "bind() first");
}

// bind(error class, addresses of last_error, quantise, norm, multiply, gate, product_scratch)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 7);
  auto address = [&](int i) { return (uintptr_t)integer(a[i]); };
  lib = {(decltype(lib.last_error))address(1), (decltype(lib.quantise))address(2), (decltype(lib.norm))address(3), (decltype(lib.multiply))address(4), (decltype(lib.gate))address(5),
         (decltype(lib.product_scratch))address(6)};
  Py_INCREF(a[0]);
  Py_XDECREF(failure);
  failure = a[0];
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

// quantise(x) -> (codes, scales)
PyObject* quantise(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  call_arguments(n, 1);
  const Numbers x = numbers(a[0], "x");
  const Result r = make_rows(x.T, x.K, x.device);
  launch("mb8_quantise", x.device, [&](void* st) { return lib.quantise(x.at, x.ld, x.wide, r.codes.data_ptr(), r.scales.data_ptr(), x.T, x.K, st); });
  return pair_of(r);
  END_HANDLE_TH_ERRORS
}

// norm(x, weight, eps, add or None) -> (codes, scales, h or None)
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  call_arguments(n, 4);
  const Numbers x = numbers(a[0], "x");
  ASSERT(x.K <= MB8_MAX_NORM, "rows of %lld entries (at most %d)", (long long)x.K, MB8_MAX_NORM);
  const at::Tensor& w = tensor(a[1], "weight");
  const at::ScalarType type = x.wide ? at::kFloat : at::kBFloat16;
  ASSERT(w.scalar_type() == type && w.dim() == 1 && w.size(0) == x.K && w.is_contiguous() && w.is_cuda() && w.get_device() == x.device, "weight [%lld] of x's type and device, contiguous",
         (long long)x.K);
  const double eps = PyFloat_AsDouble(a[2]);
  if (eps == -1.0 && PyErr_Occurred()) throw python_error();
  const bool adds = a[3] != Py_None;
  Numbers add{};
  at::Tensor h;
  if (adds) {
    add = numbers(a[3], "add");
    ASSERT(add.wide == x.wide && add.T == x.T && add.K == x.K && add.device == x.device, "add [%lld, %lld] of x's type and device", (long long)x.T, (long long)x.K);
    h = make({x.T, x.K}, {x.K, 1}, type, x.device);
  }
  const Result r = make_rows(x.T, x.K, x.device);
  launch("mb8_norm", x.device, [&](void* st) {
    return lib.norm(x.at, x.ld, add.at, add.ld, w.data_ptr(), x.wide, adds ? h.data_ptr() : nullptr, r.codes.data_ptr(), r.scales.data_ptr(), x.T, x.K, (float)eps, st);
  });
  PyObject* const t = PyTuple_New(3);
  if (t == nullptr) throw python_error();
  PyTuple_SET_ITEM(t, 0, wrapped(r.codes));
  PyTuple_SET_ITEM(t, 1, wrapped(r.scales));
  if (!adds) Py_INCREF(Py_None);
  PyTuple_SET_ITEM(t, 2, adds ? wrapped(h) : Py_None);
  return t;
  END_HANDLE_TH_ERRORS
}

// x and w of a product: codes, scales, columns of each; room for the parts of prompts
struct Product {
  Rows x, w;
  at::Tensor scratch;
  int64_t bytes = 0;
  explicit Product(PyObject* const* a) : x(rows(a[0], a[1], integer(a[2]), "x")), w(rows(a[3], a[4], integer(a[5]), "w")) {
    ASSERT(x.device == w.device && x.K == w.K && w.T >= 1, "rows of one length on one device: %lld and %lld of %lld", (long long)x.K, (long long)w.T, (long long)w.K);
    const c10::cuda::CUDAGuard guard((c10::DeviceIndex)x.device);
    bytes = lib.product_scratch(x.T, w.T, x.K);  // (how a product is cut goes by its device's SMs)
    if (bytes > 0) scratch = make({bytes}, {1}, at::kByte, x.device);
  }
  void* room() const { return bytes > 0 ? scratch.data_ptr() : nullptr; }
};

// multiply(x codes, scales, columns, w codes, scales, columns, w is fixed, results in fp32, out or None) -> out
PyObject* multiply(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  call_arguments(n, 9);
  const Product p(a);
  const bool fixed = truth(a[6]);
  Numbers out{nullptr, p.x.T, p.w.T, p.w.T, truth(a[7]), p.x.device};
  at::Tensor made;
  if (a[8] == Py_None) {
    made = make({out.T, out.K}, {out.K, 1}, out.wide ? at::kFloat : at::kBFloat16, out.device);
    out.at = made.data_ptr();
  } else {
    out = numbers(a[8], "out");
    ASSERT(out.T == p.x.T && out.K == p.w.T && out.device == p.x.device, "out [%lld, %lld] on x's device", (long long)p.x.T, (long long)p.w.T);
  }
  launch("mb8_multiply", p.x.device, [&](void* st) {
    return lib.multiply(p.x.codes, p.x.scales, p.w.codes, p.w.scales, out.at, out.ld, out.wide, p.x.T, p.w.T, p.x.K, fixed, p.room(), p.bytes, st);
  });
  if (a[8] == Py_None) return wrapped(made);
  Py_INCREF(a[8]);
  return a[8];
  END_HANDLE_TH_ERRORS
}

// gate(x codes, scales, columns, w codes, scales, columns, w is fixed) -> (codes, scales)
PyObject* gate(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  call_arguments(n, 7);
  const Product p(a);
  ASSERT(p.w.T >= 2 && p.w.T % 2 == 0, "pairs of rows, got %lld", (long long)p.w.T);
  const bool fixed = truth(a[6]);
  const Result r = make_rows(p.x.T, p.w.T / 2, p.x.device);
  launch("mb8_gate", p.x.device, [&](void* st) {
    return lib.gate(p.x.codes, p.x.scales, p.w.codes, p.w.scales, r.codes.data_ptr(), r.scales.data_ptr(), p.x.T, p.w.T / 2, p.x.K, fixed, p.room(), p.bytes, st);
  });
  return pair_of(r);
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"bind", (PyCFunction)(void (*)(void))bind, METH_FASTCALL, nullptr},     {"quantise", (PyCFunction)(void (*)(void))quantise, METH_FASTCALL, nullptr},
                         {"norm", (PyCFunction)(void (*)(void))norm, METH_FASTCALL, nullptr},     {"multiply", (PyCFunction)(void (*)(void))multiply, METH_FASTCALL, nullptr},
                         {"gate", (PyCFunction)(void (*)(void))gate, METH_FASTCALL, nullptr},     {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "mb200_rows8_host", nullptr, -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit_mb200_rows8_host() { return PyModule_Create(&module); }
