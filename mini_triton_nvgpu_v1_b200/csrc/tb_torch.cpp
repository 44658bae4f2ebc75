// tb_torch.cpp — the calls of grouped.py on torch tensors, without the
// interpreter's share of their cost (module _tbtorch).
//
// A call whose tensors have sizes, strides, types and device as an earlier
// call's had needs no checks and no desc of its own: grouped.py checks the
// first such call and leaves here what it found (remember), by those
// properties, never by address. call() then compares the tensors with what it
// knows, reads their addresses and the current stream, and calls the C ABI.
// Reading five tensors' properties into a key and handing twelve arguments to
// the library took the interpreter about as long as the launch itself.
//
// call() returns 0 (done), a tbStatus of the library, or -1: not a call that
// it knows (other properties, another current device), for which grouped.py
// takes the long way. Operands with rows off 16-byte boundaries get their
// workspace here, from torch's allocator on the call's stream (the long way
// took the interpreter 22 µs a call; now 10, with the copy).
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <mutex>
#include <vector>

#include "../../include/tb_gemm.h"

namespace {

enum Op : int { kRows = 0, kWgrad = 1, kQuantize = 2, kBytes = 3, kRowsBytes = 4, kOps = 5 };
constexpr int kTensors[kOps] = {4, 4, 3, 5, 6};
constexpr unsigned kOutputs[kOps] = {1u << 2, 1u << 2, 1u << 1 | 1u << 2, 1u << 4, 1u << 4};  // bit i: tensor i is written

// The C ABI, handed over by the binding that loaded the library.
struct {
  decltype(&tb_grouped_matmul) rows;
  decltype(&tb_grouped_matmul_wgrad) wgrad;
  decltype(&tb_quantize_blocks) quantize;
  decltype(&tb_matmul_blockscaled) bytes;
  decltype(&tb_grouped_matmul_blockscaled) rows_bytes;
  decltype(&tb_grouped_matmul_workspace_bytes) need_rows;
  decltype(&tb_grouped_matmul_wgrad_workspace_bytes) need_wgrad;
} g_abi;
constexpr int kAbi = 7;

// One tensor: dimensions, type, device, sizes and strides.
constexpr int kWords = 9, kMaxTensors = 6;
struct Signature {
  int64_t w[kMaxTensors * kWords + 2];
  int n;
};

bool sign(PyObject* const* args, int op, int64_t x, int64_t y, Signature* s, const at::Tensor** t) try {
  s->n = 0;
  for (int i = 0; i < kTensors[op]; ++i) {
    if (!THPVariable_Check(args[i])) return false;
    const at::Tensor& a = THPVariable_Unpack(args[i]);
    if (!a.defined() || !a.is_cuda() || a.layout() != c10::kStrided || a.dim() > 3) return false;
    t[i] = &a;
    int64_t* w = s->w + s->n;
    std::memset(w, 0, kWords * sizeof(int64_t));
    w[0] = a.dim();
    w[1] = (int64_t)a.scalar_type();
    w[2] = a.get_device();
    for (int64_t d = 0; d < a.dim(); ++d) {
      w[3 + d] = a.sizes()[d];
      w[6 + d] = a.strides()[d];
    }
    s->n += kWords;
  }
  s->w[s->n++] = x;
  s->w[s->n++] = y;
  return true;
} catch (const std::exception&) {  // tensors without plain sizes or strides
  return false;
}

struct Known {
  Signature s;
  tb_grouped_desc d;
  tb_quantize_desc q;
  int64_t a[8];
  tb_scales sa, sb;
  int device;
};
std::vector<Known> g_known[kOps];  // under the interpreter's lock; the latest found first
constexpr size_t kMostKnown = 64;

// call(op, tensors…, x, y): x, y are the block's extent, or beta and whether the
// caller has a workspace of its own (for which grouped.py takes the long way).
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  const int op = n > 0 ? (int)PyLong_AsLong(args[0]) : -1;
  if (op < 0 || op >= kOps || n != 1 + kTensors[op] + 2) {
    PyErr_SetString(PyExc_TypeError, "call(op, tensors..., x, y)");
    return nullptr;
  }
  if (!PyLong_Check(args[n - 2]) || !PyLong_Check(args[n - 1])) return PyLong_FromLong(-1);
  const int64_t x = PyLong_AsLongLong(args[n - 2]), y = PyLong_AsLongLong(args[n - 1]);
  if (PyErr_Occurred()) {  // beyond 64 bits
    PyErr_Clear();
    return PyLong_FromLong(-1);
  }
  Signature s;
  const at::Tensor* t[kMaxTensors];
  if (!sign(args + 1, op, x, op == kQuantize ? y : 0, &s, t)) return PyLong_FromLong(-1);
  auto& known = g_known[op];
  size_t i = 0;
  while (i < known.size() && std::memcmp(known[i].s.w, s.w, s.n * sizeof(int64_t)) != 0) ++i;
  if (i == known.size()) return PyLong_FromLong(-1);
  if (i) std::swap(known[i], known[i / 2]), i /= 2;
  const Known k = known[i];
  tbStatus st = TB_OK;
  try {
    if (c10::cuda::current_device() != k.device) return PyLong_FromLong(-1);
    void* stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)k.device).stream();
    void* p[kMaxTensors];
    // A written tensor that shares its storage until then (copy on write) gets its own here.
    for (int j = 0; j < kTensors[op]; ++j)
      p[j] = kOutputs[op] >> j & 1 ? t[j]->mutable_data_ptr() : const_cast<void*>(t[j]->const_data_ptr());
    size_t need = 0;
    if (op == kWgrad) need = g_abi.need_wgrad(&k.d, p[0], k.a[0], p[1], k.a[1]);
    else if (op != kQuantize)
      need = g_abi.need_rows(&k.d, p[0], k.a[0], p[op == kRows ? 1 : 2], k.a[1], op == kBytes ? 0 : k.a[2]);
    if (need && y) return PyLong_FromLong(-1);
    c10::DataPtr scratch;  // given back, in stream order, when the call has been enqueued
    if (need) scratch = c10::cuda::CUDACachingAllocator::get()->allocate(need);
    void* const ws = scratch.get();
    tb_scales sa = k.sa, sb = k.sb;
    if (op == kBytes || op == kRowsBytes) {
      sa.ptr = static_cast<const float*>(p[1]);
      sb.ptr = static_cast<const float*>(p[3]);
    }
    Py_BEGIN_ALLOW_THREADS
    switch (op) {
      case kRows:
        st = g_abi.rows(&k.d, p[0], k.a[0], p[1], k.a[1], k.a[2], p[2], k.a[3], p[3], ws, need, stream);
        break;
      case kWgrad:
        st = g_abi.wgrad(&k.d, p[0], k.a[0], p[1], k.a[1], p[2], k.a[2], k.a[3], p[3], ws, need, stream);
        break;
      case kQuantize:
        st = g_abi.quantize(&k.q, p[0], k.a[0], k.a[1], p[1], k.a[2], k.a[3], static_cast<float*>(p[2]), k.a[4], k.a[5],
                            k.a[6], stream);
        break;
      case kBytes:
        st = g_abi.bytes(&k.d, p[0], k.a[0], &sa, p[2], k.a[1], &sb, p[4], k.a[2], ws, need, stream);
        break;
      case kRowsBytes:
        st = g_abi.rows_bytes(&k.d, p[0], k.a[0], &sa, p[2], k.a[1], k.a[2], &sb, p[4], k.a[3], p[5], ws, need, stream);
        break;
    }
    Py_END_ALLOW_THREADS
  } catch (const std::exception&) {
    return PyLong_FromLong(-1);
  }
  return PyLong_FromLong(st);
}

bool bytes_of(PyObject* o, void* to, size_t n) {
  if (o == Py_None) return true;
  Py_buffer b;
  if (PyObject_GetBuffer(o, &b, PyBUF_SIMPLE) != 0) return false;
  const bool ok = (size_t)b.len == n;
  if (ok) std::memcpy(to, b.buf, n);
  else PyErr_SetString(PyExc_ValueError, "a struct of another size");
  PyBuffer_Release(&b);
  return ok;
}

// remember(op, tensors…, x, y, desc, ints, sa, sb): what call() may do for such tensors.
PyObject* remember(PyObject*, PyObject* const* args, Py_ssize_t n) {
  const int op = n > 0 ? (int)PyLong_AsLong(args[0]) : -1;
  if (op < 0 || op >= kOps || n != 1 + kTensors[op] + 6) {
    PyErr_SetString(PyExc_TypeError, "remember(op, tensors..., x, y, desc, ints, sa, sb)");
    return nullptr;
  }
  PyObject* const* rest = args + 1 + kTensors[op];
  Known k;
  std::memset(&k, 0, sizeof(k));
  const at::Tensor* t[kMaxTensors];
  const int64_t x = PyLong_AsLongLong(rest[0]), y = PyLong_AsLongLong(rest[1]);
  if (PyErr_Occurred()) return nullptr;
  if (!sign(args + 1, op, x, y, &k.s, t)) Py_RETURN_NONE;
  k.device = t[0]->get_device();
  if (!(op == kQuantize ? bytes_of(rest[2], &k.q, sizeof(k.q)) : bytes_of(rest[2], &k.d, sizeof(k.d)))) return nullptr;
  if (!bytes_of(rest[4], &k.sa, sizeof(k.sa)) || !bytes_of(rest[5], &k.sb, sizeof(k.sb))) return nullptr;
  if (!PyTuple_Check(rest[3]) || PyTuple_GET_SIZE(rest[3]) > 8) {
    PyErr_SetString(PyExc_TypeError, "ints must be a tuple of at most 8");
    return nullptr;
  }
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(rest[3]); ++i) k.a[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(rest[3], i));
  if (PyErr_Occurred()) return nullptr;
  auto& known = g_known[op];
  for (const Known& e : known)
    if (std::memcmp(e.s.w, k.s.w, k.s.n * sizeof(int64_t)) == 0) Py_RETURN_NONE;
  if (known.size() >= kMostKnown) known.pop_back();
  known.insert(known.begin(), k);
  Py_RETURN_NONE;
}

// library(addresses): the five entry points, in the order of Op, and the two that size workspaces.
PyObject* library(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kAbi) {
    PyErr_SetString(PyExc_TypeError, "library(seven addresses)");
    return nullptr;
  }
  void* p[kAbi];
  for (int i = 0; i < kAbi; ++i) p[i] = PyLong_AsVoidPtr(args[i]);
  if (PyErr_Occurred()) return nullptr;
  g_abi.rows = reinterpret_cast<decltype(g_abi.rows)>(p[0]);
  g_abi.wgrad = reinterpret_cast<decltype(g_abi.wgrad)>(p[1]);
  g_abi.quantize = reinterpret_cast<decltype(g_abi.quantize)>(p[2]);
  g_abi.bytes = reinterpret_cast<decltype(g_abi.bytes)>(p[3]);
  g_abi.rows_bytes = reinterpret_cast<decltype(g_abi.rows_bytes)>(p[4]);
  g_abi.need_rows = reinterpret_cast<decltype(g_abi.need_rows)>(p[5]);
  g_abi.need_wgrad = reinterpret_cast<decltype(g_abi.need_wgrad)>(p[6]);
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(call)), METH_FASTCALL, nullptr},
    {"remember", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(remember)), METH_FASTCALL, nullptr},
    {"library", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(library)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_tbtorch", "Calls of the C ABI on torch tensors.", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tbtorch() { return PyModule_Create(&g_module); }
