// _tensors.cpp -- the learned layers' calls on torch tensors, from Python into
// libaf2cuda.so's C ABI: argument checks, outputs and the stream, in C++
// because a step has hundreds of tensors and its smallest calls take less time
// on the GPU than an interpreted check of their arguments (a dense layer of one
// row: 4.8 us there, 11 us in Python; clipping 384 tensors: 25 and 394 us).
//
// The module links nothing of the library: bind() takes the entry points'
// addresses, so that one loaded libaf2cuda.so serves all of the package.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <optional>
#include <string>
#include <vector>

#include "af2cuda.h"

namespace {

struct Entry {
  decltype(&af2_dense_saved_bytes) dense_saved_bytes;
  decltype(&af2_dense_workspace_bytes) dense_workspace_bytes;
  decltype(&af2_dense) dense;
  decltype(&af2_dense_backward) dense_backward;
  decltype(&af2_gated_transition_saved_bytes) gated_saved_bytes;
  decltype(&af2_gated_transition_workspace_bytes) gated_workspace_bytes;
  decltype(&af2_gated_transition) gated;
  decltype(&af2_gated_transition_backward) gated_backward;
  decltype(&af2_gradient_norm_workspace_bytes) norm_workspace_bytes;
  decltype(&af2_gradient_norm) gradient_norm;
  decltype(&af2_clip_gradients) clip_gradients;
} entry;
PyObject *range_error = nullptr, *check_status = nullptr;

// A Python error is set.
struct Failed {};

[[noreturn]] void refuse(const std::string &message) {
  PyErr_SetString(range_error, message.c_str());
  throw Failed();
}

std::string shape_text(at::IntArrayRef s) {
  std::string t = "(";
  for (size_t i = 0; i < s.size(); ++i) t += (i ? ", " : "") + std::to_string(s[i]);
  return t + (s.size() == 1 ? ",)" : ")");
}

const at::Tensor &tensor_of(PyObject *o, const char *name) {
  if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a torch tensor");
  return THPVariable_Unpack(o);
}
const at::Tensor *optional_tensor(PyObject *o, const char *name) {
  return o == Py_None ? nullptr : &tensor_of(o, name);
}

int dtype_code(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return AF2_F32;
    case at::kHalf: return AF2_F16;
    case at::kBFloat16: return AF2_BF16;
    default: refuse(std::string("tensors must be float32, float16 or bfloat16; received ") + c10::toString(t.scalar_type()));
  }
}
const char *dtype_name(int code) {
  return code == AF2_F32 ? "torch.float32" : code == AF2_F16 ? "torch.float16" : "torch.bfloat16";
}

// One call: the context, where it is, and the type of its tensors.
struct Call {
  af2_ctx *ctx;
  int ordinal;
  int code = 0;
  at::ScalarType type = at::kFloat;

  explicit Call(PyObject *const *args)
      : ctx(reinterpret_cast<af2_ctx *>(PyLong_AsUnsignedLongLong(args[0]))),
        ordinal(static_cast<int>(PyLong_AsLong(args[1]))) {
    if (PyErr_Occurred()) throw Failed();
  }
  void set_type(const at::Tensor &t) {
    code = dtype_code(t);
    type = t.scalar_type();
  }
  bool placed(const at::Tensor &t) const {
    return t.scalar_type() == type && t.is_cuda() && t.get_device() == ordinal;
  }
  // A [rows, width] tensor (rows < 0: any): its row stride.
  int64_t rows(const char *name, const at::Tensor &t, int64_t rows, int64_t width) const {
    const auto s = t.sizes();
    if (s.size() != 2 || s[1] != width || (rows >= 0 && s[0] != rows))
      refuse(std::string(name) + " has shape " + shape_text(s) + "; expected (" +
             (rows < 0 ? "rows" : std::to_string(rows)) + ", " + std::to_string(width) + ")");
    if (!placed(t))
      refuse(std::string(name) + " must be a " + dtype_name(code) + " tensor on cuda:" + std::to_string(ordinal));
    if (t.is_contiguous()) return width;
    if ((t.stride(1) != 1 && width > 1) || (t.stride(0) < width && s[0] > 1))
      refuse(std::string(name) + " must have contiguous rows a width or more apart; its strides are " +
             shape_text(t.strides()));
    return std::max<int64_t>(t.stride(0), width);
  }
  // A contiguous tensor of this shape: its address.
  void *whole(const char *name, const at::Tensor &t, at::IntArrayRef shape) const {
    if (t.sizes() != shape) refuse(std::string(name) + " has shape " + shape_text(t.sizes()) + "; expected " + shape_text(shape));
    if (!placed(t) || !t.is_contiguous())
      refuse(std::string(name) + " must be a contiguous " + dtype_name(code) + " tensor on cuda:" +
             std::to_string(ordinal));
    return t.data_ptr();
  }
  at::Tensor make(at::IntArrayRef shape) const {
    return at::empty(shape, at::TensorOptions().dtype(type).device(c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(ordinal))));
  }
  at::Tensor bytes(uint64_t n) const {
    return at::empty({static_cast<int64_t>(n)},
                     at::TensorOptions().dtype(at::kByte).device(c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(ordinal))));
  }
  // At least `n` bytes, contiguous, here.
  void *block(const at::Tensor *t, uint64_t n, const char *name, const char *what) const {
    if (!t || !t->is_cuda() || t->get_device() != ordinal || !t->is_contiguous() ||
        static_cast<uint64_t>(t->numel()) * t->element_size() < n)
      refuse(std::string(name) + " must " + what + " (" + std::to_string(n) + " bytes on cuda:" + std::to_string(ordinal) + ")");
    return t->data_ptr();
  }
  // -1: torch's current stream (its default stream by cudaStreamLegacy's handle: the null one means
  // the context's own stream to the library); else a handle.  Comes before the call's allocations: a block
  // that torch hands out on its current stream may still be read there by what was queued before, and no
  // other stream waits for that.  A named stream's tensors are allocated on it; for the context's own (0),
  // which torch's allocator does not know, the host waits.
  std::optional<c10::cuda::CUDAStreamGuard> named;
  void *use_stream(long long handle) {
    const auto device = static_cast<c10::DeviceIndex>(ordinal);
    const cudaStream_t current = c10::cuda::getCurrentCUDAStream(device).stream();
    if (handle == -1) return current ? static_cast<void *>(current) : reinterpret_cast<void *>(uintptr_t(1));
    if (handle != 0)
      named.emplace(c10::cuda::getStreamFromExternal(reinterpret_cast<cudaStream_t>(handle), device));
    else if (!capturing(current))
      C10_CUDA_CHECK(cudaStreamSynchronize(current));
    return reinterpret_cast<void *>(handle);
  }
  // Scratch: the caller's; else none (the context's is used), but while the stream is being captured a block
  // from torch's allocator, which keeps it for the graph as it keeps the outputs.  query(bytes) asks for the
  // size.
  at::Tensor own_scratch;
  template <typename F>
  void *scratch(const at::Tensor *given, void *stream, F &&query) {
    if (!given && !capturing(stream)) return nullptr;
    uint64_t need = 0;
    done(query(&need));
    if (given) return block(given, need, "workspace", "hold what the call needs");
    own_scratch = bytes(need);
    return need ? own_scratch.data_ptr() : nullptr;
  }
  static bool capturing(void *stream) {
    // (no capture takes in the context's own stream or the legacy default one)
    if (!stream || stream == reinterpret_cast<void *>(uintptr_t(1))) return false;
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    C10_CUDA_CHECK(cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &status));
    return status != cudaStreamCaptureStatusNone;
  }
  void done(af2_status status) const {
    if (status == AF2_OK) return;
    PyObject *r = PyObject_CallFunction(check_status, "iK", static_cast<int>(status),
                                        reinterpret_cast<unsigned long long>(ctx));
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "the library refused the call");
    throw Failed();
  }
};

long long integer(PyObject *o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Failed();
  return v;
}
bool truth(PyObject *o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Failed();
  return v == 1;
}
void *ptr(const at::Tensor *t) { return t ? t->data_ptr() : nullptr; }
// A tensor of the caller's was written: what autograd has saved of it shows as stale.
void written(const at::Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
PyObject *wrap(const at::Tensor &t) { return THPVariable_Wrap(t); }

// (y, saved) or y.
PyObject *with_saved(const at::Tensor &y, const at::Tensor &saved, bool save) {
  if (!save) return wrap(y);
  return Py_BuildValue("NN", wrap(y), wrap(saved));
}
void put(PyObject *dict, const char *key, const at::Tensor &t) {
  PyObject *o = wrap(t);
  PyDict_SetItemString(dict, key, o);
  Py_DECREF(o);
}

// handle, ordinal, x, weight, bias, residual, activation, out, save, stream, workspace
PyObject *dense(PyObject *const *a) {
  Call c(a);
  void *const stream = c.use_stream(integer(a[9]));
  const at::Tensor &x = tensor_of(a[2], "x"), &w = tensor_of(a[3], "weight");
  const at::Tensor *bias = optional_tensor(a[4], "bias"), *residual = optional_tensor(a[5], "residual"),
                   *given = optional_tensor(a[7], "out"), *workspace = optional_tensor(a[10], "workspace");
  const int act = static_cast<int>(integer(a[6]));
  const bool save = truth(a[8]);
  if (w.dim() != 2) refuse("weight has shape " + shape_text(w.sizes()) + "; expected (inner, columns)");
  const int64_t inner = w.size(0), columns = w.size(1);
  c.set_type(x);
  af2_layer_options o{act, 0, c.rows("x", x, -1, inner), columns, columns, inner};
  const int64_t rows = x.size(0);
  const af2_linear_shape shape{rows, inner, columns};
  void *wp = c.whole("weight", w, {inner, columns});
  void *bp = bias ? c.whole("bias", *bias, {columns}) : nullptr;
  if (residual) o.residual_stride = c.rows("residual", *residual, rows, columns);
  if (given) o.out_stride = c.rows("out", *given, rows, columns);
  const at::Tensor y = given ? *given : c.make({rows, columns});
  at::Tensor saved;
  uint64_t bytes = 0;
  if (save) {
    c.done(entry.dense_saved_bytes(&shape, c.code, act, &bytes));
    saved = c.bytes(bytes);
  }
  void *const ws = c.scratch(
      workspace, stream, [&](uint64_t *need) { return entry.dense_workspace_bytes(&shape, c.code, act, 0, need); });
  c.done(entry.dense(c.ctx, &shape, c.code, x.data_ptr(), wp, bp, ptr(residual), &o, y.data_ptr(),
                     bytes ? saved.data_ptr() : nullptr, ws, stream));
  if (given) written(*given);
  return with_saved(y, saved, save);
}

// handle, ordinal, d_out, x, weight, saved, bias, activation, need x, need weight, stream, workspace
PyObject *dense_backward(PyObject *const *a) {
  Call c(a);
  void *const stream = c.use_stream(integer(a[10]));
  const at::Tensor &dy = tensor_of(a[2], "d_out"), &x = tensor_of(a[3], "x"), &w = tensor_of(a[4], "weight");
  const at::Tensor *saved = optional_tensor(a[5], "saved"), *workspace = optional_tensor(a[11], "workspace");
  const int act = static_cast<int>(integer(a[7]));
  if (w.dim() != 2) refuse("weight has shape " + shape_text(w.sizes()) + "; expected (inner, columns)");
  const int64_t inner = w.size(0), columns = w.size(1);
  c.set_type(x);
  af2_layer_options o{act, 0, c.rows("x", x, -1, inner), columns, columns, inner};
  const int64_t rows = x.size(0);
  const af2_linear_shape shape{rows, inner, columns};
  o.out_stride = c.rows("d_out", dy, rows, columns);
  void *wp = c.whole("weight", w, {inner, columns}), *kept = nullptr;
  if (act != AF2_ACTIVATION_NONE) {
    uint64_t bytes = 0;
    c.done(entry.dense_saved_bytes(&shape, c.code, act, &bytes));
    kept = c.block(saved, bytes, "saved", "be what the forward pass returned");
  }
  void *const ws = c.scratch(
      workspace, stream, [&](uint64_t *need) { return entry.dense_workspace_bytes(&shape, c.code, act, 1, need); });
  at::Tensor dx, dw, db;
  if (truth(a[8])) dx = c.make({rows, inner});
  if (truth(a[9])) dw = c.make({inner, columns});
  if (truth(a[6])) db = c.make({columns});
  auto at_of = [](const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; };
  c.done(entry.dense_backward(c.ctx, &shape, c.code, dy.data_ptr(), x.data_ptr(), wp, kept, &o, at_of(dx), at_of(dw),
                              at_of(db), ws, stream));
  PyObject *d = PyDict_New();
  if (dx.defined()) put(d, "x", dx);
  if (dw.defined()) put(d, "weight", dw);
  if (db.defined()) put(d, "bias", db);
  return d;
}

const char *const kGatedNames[6] = {"gateWeight", "gateBias", "valueWeight", "valueBias", "outputWeight", "outputBias"};

// The weights of a dict, checked; their sizes.
struct GatedTensors {
  int64_t channels = 0, hidden = 0;
  const at::Tensor *t[6] = {};
  std::vector<int64_t> shape(int i) const {
    switch (i) {
      case 0: case 2: return {channels, hidden};
      case 1: case 3: return {hidden};
      case 4: return {hidden, channels};
      default: return {channels};
    }
  }
};
GatedTensors gated_tensors(const Call &c, PyObject *dict, af2_gated_weights *w) {
  if (!PyDict_Check(dict)) refuse("weights must be a dict");
  GatedTensors g;
  Py_ssize_t known = 0;
  for (int i = 0; i < 6; ++i) {
    PyObject *o = PyDict_GetItemString(dict, kGatedNames[i]);
    if (o) ++known;
    if (o && o != Py_None) g.t[i] = &tensor_of(o, kGatedNames[i]);
    if (!g.t[i] && i % 2 == 0) refuse(std::string(kGatedNames[i]) + " is missing");
  }
  if (known != PyDict_Size(dict))
    refuse("unknown weights; expected gateWeight, gateBias, valueWeight, valueBias, outputWeight, outputBias");
  if (g.t[0]->dim() != 2) refuse("gateWeight has shape " + shape_text(g.t[0]->sizes()) + "; expected (channels, hidden)");
  g.channels = g.t[0]->size(0);
  g.hidden = g.t[0]->size(1);
  const void **slots[6] = {&w->gate_weight, &w->gate_bias, &w->value_weight, &w->value_bias, &w->output_weight,
                           &w->output_bias};
  for (int i = 0; i < 6; ++i) *slots[i] = g.t[i] ? c.whole(kGatedNames[i], *g.t[i], g.shape(i)) : nullptr;
  return g;
}

// handle, ordinal, x, weights, residual, activation, out, save, stream, workspace
PyObject *gated(PyObject *const *a) {
  Call c(a);
  void *const stream = c.use_stream(integer(a[8]));
  const at::Tensor &x = tensor_of(a[2], "x");
  const at::Tensor *residual = optional_tensor(a[4], "residual"), *given = optional_tensor(a[6], "out"),
                   *workspace = optional_tensor(a[9], "workspace");
  const int act = static_cast<int>(integer(a[5]));
  const bool save = truth(a[7]);
  c.set_type(x);
  af2_gated_weights w{};
  const GatedTensors g = gated_tensors(c, a[3], &w);
  af2_layer_options o{act, 0, c.rows("x", x, -1, g.channels), g.channels, g.channels, g.channels};
  const int64_t rows = x.size(0);
  const af2_transition_shape shape{rows, g.channels, g.hidden};
  if (residual) o.residual_stride = c.rows("residual", *residual, rows, g.channels);
  if (given) o.out_stride = c.rows("out", *given, rows, g.channels);
  const at::Tensor y = given ? *given : c.make({rows, g.channels});
  at::Tensor saved;
  uint64_t bytes = 0;
  if (save) {
    c.done(entry.gated_saved_bytes(&shape, c.code, &bytes));
    saved = c.bytes(bytes);
  }
  void *const ws = c.scratch(
      workspace, stream, [&](uint64_t *need) { return entry.gated_workspace_bytes(&shape, c.code, 0, need); });
  c.done(entry.gated(c.ctx, &shape, c.code, x.data_ptr(), &w, ptr(residual), &o, y.data_ptr(),
                     bytes ? saved.data_ptr() : nullptr, ws, stream));
  if (given) written(*given);
  return with_saved(y, saved, save);
}

// handle, ordinal, d_out, x, weights, saved, activation, need (None or a container of names), stream, workspace
PyObject *gated_backward(PyObject *const *a) {
  Call c(a);
  void *const stream = c.use_stream(integer(a[8]));
  const at::Tensor &dy = tensor_of(a[2], "d_out"), &x = tensor_of(a[3], "x");
  const at::Tensor *saved = optional_tensor(a[5], "saved"), *workspace = optional_tensor(a[9], "workspace");
  const int act = static_cast<int>(integer(a[6]));
  c.set_type(x);
  af2_gated_weights w{};
  const GatedTensors g = gated_tensors(c, a[4], &w);
  af2_layer_options o{act, 0, c.rows("x", x, -1, g.channels), g.channels, g.channels, g.channels};
  const int64_t rows = x.size(0);
  const af2_transition_shape shape{rows, g.channels, g.hidden};
  o.out_stride = c.rows("d_out", dy, rows, g.channels);
  uint64_t bytes = 0;
  c.done(entry.gated_saved_bytes(&shape, c.code, &bytes));
  void *kept = c.block(saved, bytes, "saved", "be what the forward pass returned");
  void *const ws = c.scratch(
      workspace, stream, [&](uint64_t *need) { return entry.gated_workspace_bytes(&shape, c.code, 1, need); });
  auto needed = [&](const char *name) {
    if (a[7] == Py_None) return true;
    PyObject *key = PyUnicode_FromString(name);
    const int r = PySequence_Contains(a[7], key);
    Py_DECREF(key);
    if (r < 0) throw Failed();
    return r == 1;
  };
  af2_gated_gradients out{};
  void **slots[6] = {&out.gate_weight, &out.gate_bias, &out.value_weight, &out.value_bias, &out.output_weight,
                     &out.output_bias};
  at::Tensor dx, d[6];
  if (needed("x")) {
    dx = c.make({rows, g.channels});
    out.x = dx.data_ptr();
  }
  for (int i = 0; i < 6; ++i)
    if (g.t[i] && needed(kGatedNames[i])) {
      d[i] = c.make(g.shape(i));
      *slots[i] = d[i].data_ptr();
    }
  c.done(entry.gated_backward(c.ctx, &shape, c.code, dy.data_ptr(), x.data_ptr(), &w, kept, &o, &out, ws, stream));
  PyObject *r = PyDict_New();
  if (dx.defined()) put(r, "x", dx);
  for (int i = 0; i < 6; ++i)
    if (d[i].defined()) put(r, kGatedNames[i], d[i]);
  return r;
}

std::vector<af2_tensor_ref> refs(const Call &c, PyObject *list, const char *name) {
  std::vector<af2_tensor_ref> r;
  const Py_ssize_t n = PyList_Size(list);
  r.reserve(static_cast<size_t>(n));
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject *o = PyList_GET_ITEM(list, i);
    if (!THPVariable_Check(o)) refuse(std::string(name) + " " + std::to_string(i) + " must be a torch tensor");
    const at::Tensor &t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.get_device() != c.ordinal || !t.is_contiguous())
      refuse(std::string(name) + " " + std::to_string(i) + " must be a contiguous tensor on cuda:" +
             std::to_string(c.ordinal));
    r.push_back({t.data_ptr(), t.numel(), dtype_code(t), 0});
  }
  return r;
}

// handle, ordinal, gradients (a list), out (a list or None), max_norm (None: the norm alone), stream, workspace
PyObject *gradients(PyObject *const *a) {
  Call c(a);
  void *const stream = c.use_stream(integer(a[5]));
  const std::vector<af2_tensor_ref> in = refs(c, a[2], "gradient");
  const int64_t n = static_cast<int64_t>(in.size());
  std::vector<af2_tensor_ref> out;
  if (a[3] != Py_None) {
    out = refs(c, a[3], "out");
    if (out.size() != in.size())
      refuse("out has " + std::to_string(out.size()) + " tensors; expected " + std::to_string(in.size()));
  }
  const at::Tensor *workspace = optional_tensor(a[6], "workspace");
  void *const ws = c.scratch(workspace, stream, [&](uint64_t *need) { return entry.norm_workspace_bytes(n, need); });
  const at::Tensor norm = c.make({});
  float *np = static_cast<float *>(norm.data_ptr());
  if (a[4] == Py_None) {
    c.done(entry.gradient_norm(c.ctx, in.data(), n, np, ws, stream));
  } else {
    const double limit = PyFloat_AsDouble(a[4]);
    if (PyErr_Occurred()) throw Failed();
    c.done(entry.clip_gradients(c.ctx, in.data(), a[3] != Py_None ? out.data() : nullptr, n, limit, np, ws, stream));
    PyObject *list = a[a[3] != Py_None ? 3 : 2];
    for (Py_ssize_t i = 0; i < static_cast<Py_ssize_t>(n); ++i) written(THPVariable_Unpack(PyList_GET_ITEM(list, i)));
  }
  return wrap(norm);
}

// bind({name: address}, RangeError, check)
PyObject *bind(PyObject *const *a) {
  const struct { const char *name; void *slot; } names[] = {
      {"af2_dense_saved_bytes", &entry.dense_saved_bytes},
      {"af2_dense_workspace_bytes", &entry.dense_workspace_bytes},
      {"af2_dense", &entry.dense},
      {"af2_dense_backward", &entry.dense_backward},
      {"af2_gated_transition_saved_bytes", &entry.gated_saved_bytes},
      {"af2_gated_transition_workspace_bytes", &entry.gated_workspace_bytes},
      {"af2_gated_transition", &entry.gated},
      {"af2_gated_transition_backward", &entry.gated_backward},
      {"af2_gradient_norm_workspace_bytes", &entry.norm_workspace_bytes},
      {"af2_gradient_norm", &entry.gradient_norm},
      {"af2_clip_gradients", &entry.clip_gradients}};
  for (const auto &n : names) {
    PyObject *o = PyDict_GetItemString(a[0], n.name);
    if (!o) {
      PyErr_SetString(PyExc_KeyError, n.name);
      throw Failed();
    }
    *static_cast<void **>(n.slot) = PyLong_AsVoidPtr(o);
  }
  Py_INCREF(a[1]);
  Py_INCREF(a[2]);
  range_error = a[1];
  check_status = a[2];
  Py_RETURN_NONE;
}

// No C++ exception leaves the module.
template <PyObject *(*F)(PyObject *const *), Py_ssize_t N>
PyObject *entry_point(PyObject *, PyObject *const *args, Py_ssize_t n) {
  if (n != N) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Failed &) {
    return nullptr;
  } catch (const c10::OutOfMemoryError &e) {
    PyErr_SetString(PyExc_MemoryError, e.what_without_backtrace());
    return nullptr;
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

#define ENTRY(name, count) {#name, reinterpret_cast<PyCFunction>(entry_point<name, count>), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {ENTRY(bind, 3),  ENTRY(dense, 11),          ENTRY(dense_backward, 12), ENTRY(gated, 10),
                         ENTRY(gated_backward, 10), ENTRY(gradients, 7), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors(void) { return PyModule_Create(&module); }
