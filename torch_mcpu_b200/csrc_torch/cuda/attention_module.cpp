// Python functions of the attention path on CUDA tensors (torch_mcpu_b200/
// attention.py is their public face): arguments taken straight from the
// interpreter, checked and enqueued in about a microsecond, where the small
// calls of a decoding step are otherwise spent in Python.  The C entry points'
// addresses come from the device library the package has loaded.
#include <Python.h>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../attention_ops.h"

namespace {

using mcpu_torch::attention::Api;
using mcpu_torch::attention::Opt;

orStream_t cuda_stream(c10::DeviceIndex i) {
  return reinterpret_cast<orStream_t>(c10::cuda::getCurrentCUDAStream(i).stream());
}

Api g_api = {nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, c10::DeviceType::CUDA, &cuda_stream};

// The tensors' device as the current one while a call is enqueued.
struct OnDevice {
  explicit OnDevice(const at::Tensor& t) : before(-1) {
    if (!t.is_cuda()) return;  // refused by the checks
    const c10::DeviceIndex now = c10::cuda::current_device();
    if (now == t.device().index()) return;
    before = now;
    c10::cuda::set_device(t.device().index());
  }
  ~OnDevice() {
    if (before >= 0) c10::cuda::set_device(before);
  }
  c10::DeviceIndex before;
};

const at::Tensor& tensor(PyObject* o, const char* op, const char* name) {
  TORCH_CHECK(THPVariable_Check(o), op, ": ", name, " must be a tensor");
  return THPVariable_Unpack(o);
}
Opt optional(PyObject* o, const char* op, const char* name) {
  if (o == Py_None) return std::nullopt;
  return tensor(o, op, name);
}
int64_t integer(PyObject* o, const char* op, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK(false, op, ": ", name, " must be an int");
  }
  return v;
}
double number(PyObject* o, const char* op, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    TORCH_CHECK(false, op, ": ", name, " must be a float");
  }
  return v;
}
bool truth(PyObject* o, const char* op, const char* name) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) {
    PyErr_Clear();
    TORCH_CHECK(false, op, ": ", name, " must be a bool");
  }
  return v == 1;
}
void arguments(Py_ssize_t n, Py_ssize_t want, const char* op) {
  TORCH_CHECK(n == want, op, ": ", want, " arguments expected, got ", n);
  TORCH_CHECK(g_api.rotary != nullptr, op, ": the device library is not loaded");
}

PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK(n == 6, "bind: 6 addresses expected");
  void* p[6];
  for (int i = 0; i < 6; ++i) p[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  g_api.rotary = reinterpret_cast<decltype(g_api.rotary)>(p[0]);
  g_api.write = reinterpret_cast<decltype(g_api.write)>(p[1]);
  g_api.gather = reinterpret_cast<decltype(g_api.gather)>(p[2]);
  g_api.attend = reinterpret_cast<decltype(g_api.attend)>(p[3]);
  g_api.workspace = reinterpret_cast<decltype(g_api.workspace)>(p[4]);
  g_api.error = reinterpret_cast<decltype(g_api.error)>(p[5]);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* py_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* op = "rotary_embedding";
  arguments(n, 6, op);
  const at::Tensor& q = tensor(a[1], op, "query");
  OnDevice on(q);
  mcpu_torch::attention::rotary_embedding(g_api, tensor(a[0], op, "positions"), q, optional(a[2], op, "key"),
                                          integer(a[3], op, "head_size"), tensor(a[4], op, "cos_sin_cache"),
                                          truth(a[5], op, "is_neox"));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* py_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* op = n == 11 && a[4] != Py_None ? "rotary_reshape_and_cache" : "reshape_and_cache";
  arguments(n, 11, op);
  const at::Tensor& key = tensor(a[2], op, "key");
  OnDevice on(key);
  mcpu_torch::attention::write(g_api, optional(a[0], op, "positions"), optional(a[1], op, "query"), key, tensor(a[3], op, "value"),
                               optional(a[4], op, "cos_sin_cache"), truth(a[5], op, "is_neox"), tensor(a[6], op, "key_cache"),
                               tensor(a[7], op, "value_cache"), tensor(a[8], op, "slot_mapping"), optional(a[9], op, "k_scale"),
                               optional(a[10], op, "v_scale"));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* py_gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* op = "gather_cache";
  arguments(n, 9, op);
  const at::Tensor& kc = tensor(a[0], op, "key_cache");
  OnDevice on(kc);
  mcpu_torch::attention::gather_cache(g_api, kc, tensor(a[1], op, "value_cache"), tensor(a[2], op, "block_table"),
                                      tensor(a[3], op, "cu_seq_lens"), tensor(a[4], op, "key_out"), tensor(a[5], op, "value_out"),
                                      optional(a[6], op, "k_scale"), optional(a[7], op, "v_scale"), optional(a[8], op, "seq_starts"));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject* py_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const char* op = "tree_attention";
  arguments(n, 13, op);
  const at::Tensor& q = tensor(a[0], op, "query");
  OnDevice on(q);
  const bool lse = truth(a[12], op, "return_lse");
  const auto r = mcpu_torch::attention::tree_attention(
      g_api, q, tensor(a[1], op, "key_cache"), tensor(a[2], op, "value_cache"), tensor(a[3], op, "block_table"),
      tensor(a[4], op, "seq_lens"), tensor(a[5], op, "cu_query_lens"), integer(a[6], op, "max_query_len"),
      number(a[7], op, "scale"), optional(a[8], op, "tree_mask"), optional(a[9], op, "k_scale"), optional(a[10], op, "v_scale"),
      optional(a[11], op, "out"), lse);
  if (!lse) return THPVariable_Wrap(std::get<0>(r));
  PyObject* t = PyTuple_New(2);
  if (!t) return nullptr;
  PyTuple_SET_ITEM(t, 0, THPVariable_Wrap(std::get<0>(r)));
  PyTuple_SET_ITEM(t, 1, THPVariable_Wrap(std::get<1>(r)));
  return t;
  END_HANDLE_TH_ERRORS
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr
PyMethodDef kMethods[] = {{"bind", FAST(py_bind)},          {"rotary_embedding", FAST(py_rotary)}, {"write", FAST(py_write)},
                          {"gather_cache", FAST(py_gather)}, {"tree_attention", FAST(py_attend)},  {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "torch_mcpu_b200_ops", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit_torch_mcpu_b200_ops() { return PyModule_Create(&kModule); }
