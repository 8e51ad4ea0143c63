// CPython module between torch tensors and the C ABI, for the operators of a decode step.
//
// Such a call is over in 3 us on the GPU, but checking ten tensors and converting 26 arguments in Python took 10 us of
// the host.  Here it is: tensors are looked at through ATen (a few ns each), the entry point is called with the current
// stream of the tensors' device.  A function returns the entry point's status, or None if some tensor is not what the
// arguments say; the caller (neptune_mlir/runtime.py) then goes through the checks that name it.  Nothing is computed
// here, and libnb200.so itself knows nothing of torch.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <stdexcept>

#include "nb200.h"

namespace {

constexpr int kMaxDevices = 64;
int *g_status[kMaxDevices];
decltype(&nb200_qk_norm_rope) g_qk_norm_rope;
decltype(&nb200_rope_append) g_rope_append;
decltype(&nb200_attn_paged) g_attn_paged;
size_t g_attn_paged_workspace;

struct NotATensor : std::exception {};

// The tensor behind a Python object; null for None.
const at::Tensor *tensor(PyObject *o) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) throw NotATensor();
  return &THPVariable_Unpack(o);
}
const at::Tensor &needed(PyObject *o) {
  const at::Tensor *t = tensor(o);
  if (!t) throw NotATensor();
  return *t;
}
int integer(PyObject *o) {
  const long x = PyLong_AsLong(o);
  if (x == -1 && PyErr_Occurred()) throw std::invalid_argument("");
  if (x != static_cast<int>(x)) {
    PyErr_SetString(PyExc_OverflowError, "nb200: an extent does not fit 32 bits");
    throw std::invalid_argument("");
  }
  return static_cast<int>(x);
}
float real(PyObject *o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw std::invalid_argument("");
  return static_cast<float>(x);
}
bool truth(PyObject *o) {
  const int x = PyObject_IsTrue(o);
  if (x < 0) throw std::invalid_argument("");
  return x != 0;
}
bool storage_type(int code, at::ScalarType *out) {
  if (code == NB200_F16) return *out = at::kHalf, true;
  if (code == NB200_BF16) return *out = at::kBFloat16, true;
  if (code == NB200_F32) return *out = at::kFloat, true;
  return false;
}

// Whether a tensor is on this device, of this type and shape, and contiguous (`rows`: in its last dimension at least).
bool fits(const at::Tensor &t, c10::DeviceIndex device, at::ScalarType type, std::initializer_list<int64_t> shape, bool rows = false) {
  if (!t.is_cuda() || t.get_device() != device || t.scalar_type() != type || t.dim() != static_cast<int64_t>(shape.size())) return false;
  int64_t i = 0;
  for (int64_t n : shape)
    if (t.size(i++) != n) return false;
  return rows ? t.stride(-1) == 1 : t.is_contiguous();
}
bool weight_fits(const at::Tensor *w, c10::DeviceIndex device, at::ScalarType type, int D) { return !w || fits(*w, device, type, {D}); }

struct Paged {
  const at::Tensor &k_pages, &v_pages, &block_table, &cu_seqlens, &seq_lens;
  int B, Hkv, max_pages, page_size, D;
  bool fit(c10::DeviceIndex device, at::ScalarType type) const {
    if (k_pages.dim() != 4) return false;
    const int64_t pages = k_pages.size(0);
    return pages == static_cast<int>(pages) && fits(k_pages, device, type, {pages, Hkv, page_size, D}) &&
           fits(v_pages, device, type, {pages, Hkv, page_size, D}) && fits(block_table, device, at::kInt, {B, max_pages}) &&
           fits(cu_seqlens, device, at::kInt, {int64_t{B} + 1}) && fits(seq_lens, device, at::kInt, {B});
  }
};
int *ints(const at::Tensor &t) { return static_cast<int *>(t.data_ptr()); }
void *pointer(const at::Tensor *t) { return t ? t->data_ptr() : nullptr; }
int *status_of(c10::DeviceIndex device) { return device >= 0 && device < kMaxDevices ? g_status[device] : nullptr; }

PyObject *none() { Py_RETURN_NONE; }

// Runs a call and turns C++ exceptions into Python ones.
template <typename F> PyObject *guarded(const char *name, Py_ssize_t given, Py_ssize_t wanted, F &&f) {
  if (given != wanted) return PyErr_Format(PyExc_TypeError, "%s: %zd arguments, %zd given", name, wanted, given);
  try {
    return f();
  } catch (const NotATensor &) {
    return none();
  } catch (const std::exception &e) {
    if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s: %s", name, e.what());
    return nullptr;
  }
}

PyObject *qk_norm_rope(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded("qk_norm_rope", n, 17, [&]() -> PyObject * {
    const at::Tensor &q = needed(a[0]), &k = needed(a[1]), &positions = needed(a[2]), &inv_freq = needed(a[3]), &q_out = needed(a[4]),
                     &k_out = needed(a[5]);
    const at::Tensor *wq = tensor(a[6]), *wk = tensor(a[7]);
    const int B = integer(a[8]), S = integer(a[9]), Hq = integer(a[10]), Hkv = integer(a[11]), D = integer(a[12]), rot = integer(a[13]);
    const bool interleaved = truth(a[14]);
    const float eps = real(a[15]);
    const int dtype = integer(a[16]);
    at::ScalarType type;
    if (!q.is_cuda() || !storage_type(dtype, &type)) return none();
    const auto dev = q.get_device();
    const bool one_row = positions.dim() == 1;
    if (!fits(q, dev, type, {B, S, Hq, D}, true) || !fits(k, dev, type, {B, S, Hkv, D}, true) || !fits(q_out, dev, type, {B, Hq, S, D}, true) ||
        !fits(k_out, dev, type, {B, Hkv, S, D}, true) || !(one_row ? fits(positions, dev, at::kInt, {S}) : fits(positions, dev, at::kInt, {B, S})) ||
        !fits(inv_freq, dev, at::kFloat, {rot / 2}) || !weight_fits(wq, dev, type, D) || !weight_fits(wk, dev, type, D))
      return none();
    const long long strides[13] = {q.stride(0), q.stride(1), q.stride(2), k.stride(0), k.stride(1), k.stride(2), q_out.stride(0),
                                   q_out.stride(2), q_out.stride(1), k_out.stride(0), k_out.stride(2), k_out.stride(1), one_row ? 0 : S};
    const c10::cuda::CUDAGuard guard(dev);
    return PyLong_FromLong(g_qk_norm_rope(q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(), ints(positions),
                                          static_cast<float *>(inv_freq.data_ptr()), pointer(wq), pointer(wk), strides, B, S, Hq, Hkv, D, rot,
                                          interleaved, eps, dtype, c10::cuda::getCurrentCUDAStream(dev).stream()));
  });
}

PyObject *rope_append(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded("rope_append", n, 23, [&]() -> PyObject * {
    const at::Tensor *q = tensor(a[0]), *q_out = tensor(a[9]), *wq = tensor(a[10]), *wk = tensor(a[11]);
    const at::Tensor &k = needed(a[1]), &v = needed(a[2]), &inv_freq = needed(a[8]);
    const int T = integer(a[12]), B = integer(a[13]), Hq = integer(a[14]), Hkv = integer(a[15]), max_pages = integer(a[16]),
              page_size = integer(a[17]), D = integer(a[18]), rot = integer(a[19]);
    const bool interleaved = truth(a[20]);
    const float eps = real(a[21]);
    const int dtype = integer(a[22]);
    const Paged paged{needed(a[3]), needed(a[4]), needed(a[5]), needed(a[6]), needed(a[7]), B, Hkv, max_pages, page_size, D};
    at::ScalarType type;
    if (!k.is_cuda() || !storage_type(dtype, &type)) return none();
    const auto dev = k.get_device();
    int *status = status_of(dev);
    if (!status || !fits(k, dev, type, {T, Hkv, D}, true) || !fits(v, dev, type, {T, Hkv, D}, true) || !paged.fit(dev, type) ||
        !fits(inv_freq, dev, at::kFloat, {rot / 2}) || !weight_fits(wq, dev, type, D) || !weight_fits(wk, dev, type, D))
      return none();
    if (Hq == 0 ? (q || q_out) : (!q || !q_out || !fits(*q, dev, type, {T, Hq, D}, true) || !fits(*q_out, dev, type, {T, Hq, D}, true))) return none();
    const long long strides[8] = {Hq ? q->stride(0) : 0, Hq ? q->stride(1) : 0, k.stride(0), k.stride(1), v.stride(0), v.stride(1),
                                  Hq ? q_out->stride(0) : 0, Hq ? q_out->stride(1) : 0};
    const c10::cuda::CUDAGuard guard(dev);
    return PyLong_FromLong(g_rope_append(pointer(q), k.data_ptr(), v.data_ptr(), pointer(q_out), paged.k_pages.data_ptr(), paged.v_pages.data_ptr(),
                                         ints(paged.block_table), ints(paged.cu_seqlens), ints(paged.seq_lens),
                                         static_cast<float *>(inv_freq.data_ptr()), pointer(wq), pointer(wk), strides, T, B, Hq, Hkv,
                                         static_cast<int>(paged.k_pages.size(0)), max_pages, page_size, D, rot, interleaved, eps, dtype, status,
                                         c10::cuda::getCurrentCUDAStream(dev).stream()));
  });
}

PyObject *attn_paged(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded("attn_paged", n, 17, [&]() -> PyObject * {
    const at::Tensor &q = needed(a[0]), &workspace = needed(a[6]), &out = needed(a[7]);
    const int T = integer(a[8]), B = integer(a[9]), Hq = integer(a[10]), Hkv = integer(a[11]), max_pages = integer(a[12]),
              page_size = integer(a[13]), D = integer(a[14]), dtype = integer(a[15]);
    const float scale_log2 = real(a[16]);
    const Paged paged{needed(a[1]), needed(a[2]), needed(a[3]), needed(a[4]), needed(a[5]), B, Hkv, max_pages, page_size, D};
    at::ScalarType type;
    if (!q.is_cuda() || !storage_type(dtype, &type)) return none();
    const auto dev = q.get_device();
    int *status = status_of(dev);
    if (!status || !fits(q, dev, type, {T, Hq, D}, true) || !fits(out, dev, type, {T, Hq, D}, true) || !paged.fit(dev, type)) return none();
    if (!workspace.is_cuda() || workspace.get_device() != dev || !workspace.is_contiguous() ||
        static_cast<size_t>(workspace.numel()) * workspace.element_size() < g_attn_paged_workspace)
      return none();
    const long long strides[4] = {q.stride(0), q.stride(1), out.stride(0), out.stride(1)};
    const c10::cuda::CUDAGuard guard(dev);
    return PyLong_FromLong(g_attn_paged(q.data_ptr(), paged.k_pages.data_ptr(), paged.v_pages.data_ptr(), ints(paged.block_table),
                                        ints(paged.cu_seqlens), ints(paged.seq_lens), workspace.data_ptr(), out.data_ptr(), strides, T, B, Hq, Hkv,
                                        static_cast<int>(paged.k_pages.size(0)), max_pages, page_size, D, dtype, scale_log2, status,
                                        c10::cuda::getCurrentCUDAStream(dev).stream()));
  });
}

// bind(addresses of the three entry points, workspace bytes of attn_paged): the library that the ctypes binding loaded.
PyObject *bind(PyObject *, PyObject *args) {
  unsigned long long rope, append, attn, bytes;
  if (!PyArg_ParseTuple(args, "KKKK", &rope, &append, &attn, &bytes)) return nullptr;
  g_qk_norm_rope = reinterpret_cast<decltype(g_qk_norm_rope)>(rope);
  g_rope_append = reinterpret_cast<decltype(g_rope_append)>(append);
  g_attn_paged = reinterpret_cast<decltype(g_attn_paged)>(attn);
  g_attn_paged_workspace = static_cast<size_t>(bytes);
  Py_RETURN_NONE;
}
// set_status(device, address): the device's status words; until then calls on it return None.
PyObject *set_status(PyObject *, PyObject *args) {
  int device;
  unsigned long long address;
  if (!PyArg_ParseTuple(args, "iK", &device, &address)) return nullptr;
  if (device < 0 || device >= kMaxDevices) return PyErr_Format(PyExc_ValueError, "device %d", device);
  g_status[device] = reinterpret_cast<int *>(address);
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"set_status", set_status, METH_VARARGS, nullptr},
    {"qk_norm_rope", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(qk_norm_rope)), METH_FASTCALL, nullptr},
    {"rope_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rope_append)), METH_FASTCALL, nullptr},
    {"attn_paged", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attn_paged)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "nb200_torch", "Calls of the nb200 C ABI with torch tensors.", -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// torch_version: the version whose headers this was compiled against; the loader compares it with the one that runs.
PyMODINIT_FUNC PyInit_nb200_torch(void) {
  PyObject *module = PyModule_Create(&g_module);
  if (module && PyModule_AddStringConstant(module, "torch_version", NB200_TORCH_VERSION) < 0) Py_CLEAR(module);
  return module;
}
