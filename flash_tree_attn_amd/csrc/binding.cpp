// Repeat calls of the package's functions without the interpreter's share of the work.
//
// A serving loop calls the same function with the same shapes over and over, and for small calls the Python side (an
// attribute of a tensor costs 0.1 to 0.3 us, an empty tensor 2) takes longer than the kernel. Once a call has been
// checked in full, `remember` keeps what does not depend on the tensors' contents: the filled argument struct, where
// the tensors' addresses go in it, which outputs and workspace to allocate. `recall` forms the call's signature
// (sizes, strides, dtype, device and 16-byte alignment of every tensor, whether it asks for gradients, every other
// argument's value), and if that is known patches a copy of the struct, allocates, and launches on the current stream
// of the tensors' device. Nothing is kept by a tensor's address or identity. The struct
// is copied per call, and the entry held, so that neither threads nor a garbage collection in between disturb it.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <memory>
#include <string>
#include <vector>

namespace {

constexpr Py_ssize_t kMostEntries = 256;   // signatures kept; a loop that makes a new one every step starts over

struct Output {
  Py_ssize_t offset;               // of its address in the struct
  Py_ssize_t given;                // the argument that is it, or -1: allocated
  std::vector<int64_t> sizes, strides;
  at::ScalarType dtype;
};
struct Entry {
  int (*fn)(const void*, void*);
  std::string args;                // the struct, filled
  std::vector<std::pair<Py_ssize_t, Py_ssize_t>> inputs;   // argument, offset
  std::vector<Output> outputs;
  Py_ssize_t workspace_offset;
  int64_t workspace_bytes;
  at::Device device{at::kCPU};
};

void append(std::string& key, const void* data, size_t n) { key.append(static_cast<const char*>(data), n); }

// False for an argument that has no place in a signature. tangents: tensors may carry some (a forward-mode level is live).
bool sign(PyObject* arg, std::string& key, bool tangents) {
  if (THPVariable_Check(arg)) {
    const at::Tensor& t = THPVariable_Unpack(arg);
    if (t.layout() != at::kStrided || !t.has_storage() || (tangents && t._fw_grad(0).defined())) return false;   // (a tangent: refused by the full checks)
    const auto sizes = t.sizes(), strides = t.strides();
    const char head[6] = {'t', static_cast<char>(t.scalar_type()), static_cast<char>(t.device().type()), static_cast<char>(t.device().index()),
                          static_cast<char>(sizes.size()), static_cast<char>(reinterpret_cast<uintptr_t>(t.data_ptr()) & 15)};
    append(key, head, sizeof head);
    key.push_back(t.requires_grad() && c10::GradMode::is_enabled() ? 'g' : '.');
    append(key, sizes.data(), sizes.size() * sizeof(int64_t));
    append(key, strides.data(), strides.size() * sizeof(int64_t));
  } else if (arg == Py_None || PyBool_Check(arg)) {
    key.push_back(arg == Py_None ? 'n' : arg == Py_True ? 'T' : 'F');
  } else if (PyFloat_CheckExact(arg)) {
    const double v = PyFloat_AS_DOUBLE(arg);
    key.push_back('f');
    append(key, &v, sizeof v);
  } else if (PyLong_CheckExact(arg)) {
    int overflow = 0;
    const long long v = PyLong_AsLongLongAndOverflow(arg, &overflow);
    if (overflow) return false;
    key.push_back('i');
    append(key, &v, sizeof v);
  } else if (PyUnicode_CheckExact(arg)) {   // the function's name
    Py_ssize_t n;
    const char* text = PyUnicode_AsUTF8AndSize(arg, &n);
    if (!text) {
      PyErr_Clear();
      return false;
    }
    key.push_back('s');
    append(key, &n, sizeof n);
    append(key, text, static_cast<size_t>(n));
  } else if (THPDtype_Check(arg)) {
    key.push_back('d');
    key.push_back(static_cast<char>(reinterpret_cast<THPDtype*>(arg)->scalar_type));
  } else {
    return false;
  }
  return true;
}

void put(std::string& args, Py_ssize_t offset, const void* address) { std::memcpy(&args[offset], &address, sizeof address); }

struct Release {
  void operator()(PyObject* object) const { Py_DECREF(object); }
};
using Held = std::unique_ptr<PyObject, Release>;

PyObject* launch(const Entry& e, PyObject* const* args) {
  try {
    std::string filled = e.args;
    for (const auto& [arg, offset] : e.inputs) put(filled, offset, THPVariable_Unpack(args[arg]).data_ptr());
    const c10::OptionalDeviceGuard guard(e.device);
    Held result(PyTuple_New(static_cast<Py_ssize_t>(1 + e.outputs.size())));
    if (!result) return nullptr;
    for (size_t k = 0; k < e.outputs.size(); ++k) {
      const Output& o = e.outputs[k];
      PyObject* item;
      if (o.given >= 0) {
        item = args[o.given];
        Py_INCREF(item);
      } else {
        item = THPVariable_Wrap(at::empty_strided(o.sizes, o.strides, at::TensorOptions().dtype(o.dtype).device(e.device)));
        if (!item) return nullptr;
      }
      PyTuple_SET_ITEM(result.get(), static_cast<Py_ssize_t>(1 + k), item);
      put(filled, o.offset, THPVariable_Unpack(item).data_ptr());
    }
    at::Tensor workspace;
    if (e.workspace_bytes > 0) {
      workspace = at::empty({e.workspace_bytes}, at::TensorOptions().dtype(at::kByte).device(e.device));
      put(filled, e.workspace_offset, workspace.data_ptr());
    }
    void* stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(e.device.index()).stream();
    PyThreadState* released = PyEval_SaveThread();   // a launch waits where the queue is full
    const int status = e.fn(filled.data(), stream);
    PyEval_RestoreThread(released);
    PyTuple_SET_ITEM(result.get(), 0, PyLong_FromLong(status));
    return result.release();
  } catch (const c10::OutOfMemoryError& error) {
    const Held torch_module(PyImport_ImportModule("torch"));
    const Held type(torch_module ? PyObject_GetAttrString(torch_module.get(), "OutOfMemoryError") : nullptr);
    if (type) PyErr_SetString(type.get(), error.what_without_backtrace());
    return nullptr;
  } catch (const std::exception& error) {
    PyErr_SetString(PyExc_RuntimeError, error.what());
    return nullptr;
  }
}

// recall(cache, arguments...) -> (status, outputs...) if the signature is known, else the signature (bytes), or None
// for a call without one.
PyObject* recall(PyObject*, PyObject* const* argv, Py_ssize_t argc) {
  if (argc < 2 || !PyDict_Check(argv[0])) {
    PyErr_SetString(PyExc_TypeError, "recall(cache, arguments...)");
    return nullptr;
  }
  PyObject* const* args = argv + 1;
  std::string key;
  key.reserve(512);
  try {
    const bool tangents = torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;   // (there is one level at most)
    for (Py_ssize_t i = 0; i < argc - 1; ++i)
      if (!sign(args[i], key, tangents)) Py_RETURN_NONE;
  } catch (const std::exception&) {   // a tensor without memory of its own: the full checks have the say
    Py_RETURN_NONE;
  }
  key.push_back(static_cast<char>(argc));
  Held signature(PyBytes_FromStringAndSize(key.data(), static_cast<Py_ssize_t>(key.size())));
  if (!signature) return nullptr;
  PyObject* known = PyDict_GetItemWithError(argv[0], signature.get());
  if (!known) return PyErr_Occurred() ? nullptr : signature.release();
  Py_INCREF(known);
  const Held capsule(known);
  const Entry* e = static_cast<const Entry*>(PyCapsule_GetPointer(known, "fta.entry"));
  return e ? launch(*e, args) : nullptr;
}

// remember(cache, signature, fn address, struct bytes, ((argument, offset), ...), ((offset, given, tensor), ...),
// workspace offset, workspace bytes, device index). An output is described by a tensor like it.
PyObject* remember(PyObject*, PyObject* all) {
  PyObject *cache, *signature, *inputs, *outputs;
  unsigned long long fn;
  const char* data;
  Py_ssize_t size, workspace_offset;
  long long workspace_bytes;
  int device;
  if (!PyArg_ParseTuple(all, "O!SKy#O!O!nLi", &PyDict_Type, &cache, &signature, &fn, &data, &size, &PyTuple_Type, &inputs, &PyTuple_Type, &outputs,
                        &workspace_offset, &workspace_bytes, &device))
    return nullptr;
  Entry* e = new Entry;
  e->fn = reinterpret_cast<int (*)(const void*, void*)>(static_cast<uintptr_t>(fn));
  e->args.assign(data, static_cast<size_t>(size));
  e->workspace_offset = workspace_offset;
  e->workspace_bytes = workspace_bytes;
  e->device = at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(device));
  const Py_ssize_t last = size - static_cast<Py_ssize_t>(sizeof(void*));
  bool ok = workspace_bytes == 0 || (workspace_offset >= 0 && workspace_offset <= last);
  for (Py_ssize_t i = 0; ok && i < PyTuple_GET_SIZE(inputs); ++i) {
    Py_ssize_t arg, offset;
    ok = PyArg_ParseTuple(PyTuple_GET_ITEM(inputs, i), "nn", &arg, &offset) && arg >= 0 && offset >= 0 && offset <= last;
    if (ok) e->inputs.emplace_back(arg, offset);
  }
  for (Py_ssize_t i = 0; ok && i < PyTuple_GET_SIZE(outputs); ++i) {
    Output o;
    PyObject* like;
    ok = PyArg_ParseTuple(PyTuple_GET_ITEM(outputs, i), "nnO", &o.offset, &o.given, &like) && THPVariable_Check(like) && o.offset >= 0 && o.offset <= last;
    if (!ok) break;
    const at::Tensor& t = THPVariable_Unpack(like);
    o.sizes = t.sizes().vec();
    o.strides = t.strides().vec();
    o.dtype = t.scalar_type();
    e->outputs.push_back(std::move(o));
  }
  if (!ok) {
    delete e;
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "remember: an address that does not lie in the struct");
    return nullptr;
  }
  PyObject* capsule = PyCapsule_New(e, "fta.entry", [](PyObject* c) { delete static_cast<Entry*>(PyCapsule_GetPointer(c, "fta.entry")); });
  if (!capsule) {
    delete e;
    return nullptr;
  }
  if (PyDict_Size(cache) >= kMostEntries) PyDict_Clear(cache);
  const int failed = PyDict_SetItem(cache, signature, capsule);
  Py_DECREF(capsule);
  if (failed) return nullptr;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"recall", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(recall)), METH_FASTCALL, "Launch a remembered call, or give its signature."},
    {"remember", remember, METH_VARARGS, "Keep a checked call under its signature."},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
