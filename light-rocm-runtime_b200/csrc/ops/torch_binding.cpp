// lrrt_b200's paged-cache operators on torch tensors: the checks of the
// tensors, the outputs' allocation and the calls of include/lrrt_ops.h, as a
// Python extension module (an operator's small problems take less time on the
// GPU than Python takes to look at ten tensors). lrrt_b200/ops.py documents
// the operators and holds the context.
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "lrrt_ops.h"

#include <array>
#include <cstdint>
#include <optional>
#include <sstream>
#include <string>

namespace {

// Raised as ValueError: arguments that do not fit. Nothing was enqueued.
struct Refusal {
  std::string text;
};
// A Python exception is set already.
struct Raised {};

template <typename... Parts> [[noreturn]] void refuse(const Parts &...parts) {
  std::ostringstream text;
  (text << ... << parts);
  throw Refusal{text.str()};
}

PyObject *g_fail = nullptr; // Python's fail(status, operation): raises LrrtError

// What the calls need of an Ops object.
struct Ops {
  lro_context_t *context = nullptr;
  c10::DeviceIndex device = 0;
  c10::StreamId stream = 0;
};

constexpr const char *kOpsCapsule = "lrrt_b200.ops";

const Ops &ops_of(PyObject *capsule) {
  auto *ops = static_cast<Ops *>(PyCapsule_GetPointer(capsule, kOpsCapsule));
  if (ops == nullptr) {
    throw Raised{};
  }
  if (ops->context == nullptr) {
    refuse("these operators are closed");
  }
  if (c10::cuda::getCurrentCUDAStream(ops->device).id() != ops->stream) {
    refuse("the current stream is not the stream of these operators");
  }
  return *ops;
}

void check(lr_status_t status, const char *operation) {
  if (status != LR_SUCCESS) {
    Py_XDECREF(PyObject_CallFunction(g_fail, "is", static_cast<int>(status), operation));
    throw Raised{};
  }
}

// One call of the library. It enqueues and returns, and the interpreter's lock is
// kept meanwhile: a context serves one thread at a time. The library makes its device
// current; the caller's is put back.
template <typename Arguments>
void call_library(lr_status_t (*function)(lro_context_t *, const Arguments *), const Ops &ops,
                  const Arguments &arguments, const char *operation) {
  const c10::cuda::CUDAGuard guard(ops.device);
  check(function(ops.context, &arguments), operation);
}

// ---- tensors ------------------------------------------------------------------

const at::Tensor &tensor_of(PyObject *object, const char *name) {
  if (!THPVariable_Check(object)) {
    refuse(name, " is not a tensor");
  }
  return THPVariable_Unpack(object);
}

// A tensor on the operators' device with contiguous last dimension. The operators
// have no backward pass: a graph would end at them without a word.
void check(const Ops &ops, const at::Tensor &t, const char *name, int64_t dims,
           at::ScalarType type) {
  if (!t.is_cuda() || t.get_device() != ops.device) {
    refuse(name, " is on ", t.device().str(), ", not on cuda:", static_cast<int>(ops.device));
  }
  if (t.scalar_type() != type) {
    refuse(name, " is ", t.scalar_type(), ", not ", type);
  }
  if (t.requires_grad() && at::GradMode::is_enabled()) {
    refuse(name, " requires gradients, which these operators do not have: detach it, or call them "
                 "under torch.no_grad()");
  }
  if (t.dim() != dims) {
    refuse(name, " has ", t.dim(), " dimensions, not ", dims);
  }
  if (t.size(dims - 1) > 1 && t.stride(dims - 1) != 1) {
    refuse(name, " is not contiguous in its last dimension");
  }
}

template <typename T = void>
T *vector_of(const Ops &ops, PyObject *object, const char *name, int64_t count,
             at::ScalarType type, bool optional = false) {
  if (optional && object == Py_None) {
    return nullptr;
  }
  const at::Tensor &t = tensor_of(object, name);
  check(ops, t, name, 1, type);
  if (t.numel() != count) {
    refuse(name, " has ", t.numel(), " elements, not ", count);
  }
  return static_cast<T *>(t.data_ptr());
}

uint32_t count_of(int64_t value, const char *name) {
  if (value < 0 || value > 0x7fffffff) {
    refuse(name, " is out of range: ", value);
  }
  return static_cast<uint32_t>(value);
}

lro_rows_t rows_of(const Ops &ops, const at::Tensor &t, const char *name,
                   std::array<int64_t, 3> shape, at::ScalarType type) {
  check(ops, t, name, 3, type);
  if (t.size(0) != shape[0] || t.size(1) != shape[1] || t.size(2) != shape[2]) {
    refuse(name, " has the shape ", t.sizes(), ", not [", shape[0], ", ", shape[1], ", ", shape[2],
           "]");
  }
  return {t.data_ptr(), t.stride(0), t.stride(1)};
}

// Where an output may be the input as it is, but not lie partly in it.
void check_apart(const at::Tensor &out, const char *name, const at::Tensor &in,
                 const char *in_name) {
  if (at::get_overlap_status(out, in) == at::MemOverlapStatus::Partial) {
    refuse(name, " lies partly in ", in_name);
  }
}

uint32_t type_of(const at::Tensor &t, const char *what) {
  switch (t.scalar_type()) {
  case at::kFloat:
    return LRO_F32;
  case at::kBFloat16:
    return LRO_BF16;
  case at::kHalf:
    return LRO_F16;
  default:
    refuse(what, " of ", t.scalar_type());
  }
}

// One layer's pages, [pages, page_size, kv_heads, head_dim].
lro_cache_t cache_of(const Ops &ops, PyObject *keys_object, PyObject *values_object,
                     at::ScalarType &type) {
  const at::Tensor &keys = tensor_of(keys_object, "keys");
  const at::Tensor &values = tensor_of(values_object, "values");
  const uint32_t code = type_of(keys, "a cache");
  type = keys.scalar_type();
  check(ops, keys, "keys", 4, type);
  check(ops, values, "values", 4, type);
  if (keys.sizes() != values.sizes()) {
    refuse("keys and values differ in shape");
  }
  return {keys.data_ptr(),   values.data_ptr(), keys.stride(0),
          keys.stride(1),    keys.stride(2),    values.stride(0),
          values.stride(1),  values.stride(2),  code,
          count_of(keys.size(0), "pages"),      count_of(keys.size(1), "page_size"),
          count_of(keys.size(2), "kv_heads"),   count_of(keys.size(3), "head_dim")};
}

lro_table_t table_of(const Ops &ops, const at::Tensor &t) {
  check(ops, t, "table", 2, at::kInt);
  return {static_cast<const int32_t *>(t.data_ptr()), t.stride(0),
          count_of(t.size(0), "the table's rows"), count_of(t.size(1), "the table's columns")};
}

// All layers' pages, [layers, pages, page_size, kv_heads, head_dim], each page
// contiguous, token by token or head by head.
lro_pool_t pool_of(const Ops &ops, PyObject *keys_object, PyObject *values_object) {
  const at::Tensor &keys = tensor_of(keys_object, "keys");
  const at::Tensor &values = tensor_of(values_object, "values");
  type_of(keys, "a cache");
  check(ops, keys, "keys", 5, keys.scalar_type());
  check(ops, values, "values", 5, keys.scalar_type());
  if (keys.sizes() != values.sizes() || keys.strides() != values.strides()) {
    refuse("keys and values differ in shape or strides");
  }
  const int64_t size = keys.size(2), heads = keys.size(3), dim = keys.size(4);
  const int64_t token = keys.stride(2), head = keys.stride(3);
  const int64_t bytes = static_cast<int64_t>(keys.element_size());
  int64_t segments = 1, row = heads * dim;
  if (!((token == row || size == 1) && (head == dim || heads == 1))) {
    if (!((token == dim || size == 1) && head == size * dim)) {
      refuse("pages must be contiguous, token by token or head by head");
    }
    segments = heads;
    row = dim;
  }
  return {keys.data_ptr(),
          values.data_ptr(),
          keys.stride(0) * bytes,
          keys.stride(1) * bytes,
          count_of(keys.size(0), "layers"),
          count_of(keys.size(1), "pages"),
          count_of(size, "page_size"),
          count_of(segments, "kv_heads"),
          count_of(row * bytes, "a page's row"),
          0};
}

at::Tensor empty(const Ops &ops, at::IntArrayRef shape, at::ScalarType type) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(at::kCUDA, ops.device));
}

int64_t integer_of(PyObject *object) {
  const int64_t value = PyLong_AsLongLong(object);
  if (value == -1 && PyErr_Occurred() != nullptr) {
    throw Raised{};
  }
  return value;
}
float number_of(PyObject *object) {
  const double value = PyFloat_AsDouble(object);
  if (value == -1.0 && PyErr_Occurred() != nullptr) {
    throw Raised{};
  }
  return static_cast<float>(value);
}

PyObject *wrap(at::Tensor t) {
  PyObject *object = THPVariable_Wrap(std::move(t));
  if (object == nullptr) {
    throw Raised{};
  }
  return object;
}
template <typename... Tensors> PyObject *tuple_of(Tensors... tensors) {
  PyObject *tuple = PyTuple_New(sizeof...(tensors));
  if (tuple == nullptr) {
    throw Raised{};
  }
  try {
    Py_ssize_t at = 0;
    (PyTuple_SET_ITEM(tuple, at++, wrap(std::move(tensors))), ...);
  } catch (...) {
    Py_DECREF(tuple);
    throw;
  }
  return tuple;
}

// ---- operators (arguments as lrrt_b200/ops.py passes them) -----------------------

PyObject *rope_append(const Ops &ops, PyObject *const *a) {
  at::ScalarType type;
  lro_rope_append_t call{};
  call.cache = cache_of(ops, a[4], a[5], type);
  const at::Tensor &q = tensor_of(a[1], "q");
  check(ops, q, "q", 3, type);
  const int64_t tokens = q.size(0), heads = q.size(1), dim = call.cache.head_dim;
  const int64_t kv_heads = call.cache.kv_heads;
  if (q.size(2) != dim) {
    refuse("q has a head_dim of ", q.size(2), ", the cache of ", dim);
  }
  call.q = {q.data_ptr(), q.stride(0), q.stride(1)};
  call.k = rows_of(ops, tensor_of(a[2], "k"), "k", {tokens, kv_heads, dim}, type);
  call.v = rows_of(ops, tensor_of(a[3], "v"), "v", {tokens, kv_heads, dim}, type);
  call.table = table_of(ops, tensor_of(a[6], "table"));
  call.sequences = vector_of<int32_t>(ops, a[7], "sequences", tokens, at::kInt, true);
  call.positions = vector_of<int32_t>(ops, a[8], "positions", tokens, at::kInt);
  if (a[9] != Py_None) {
    const at::Tensor &cos = tensor_of(a[9], "cos"), &sin = tensor_of(a[10], "sin");
    check(ops, cos, "cos", 2, at::kFloat);
    check(ops, sin, "sin", 2, at::kFloat);
    if (cos.sizes() != sin.sizes() || !cos.is_contiguous() || !sin.is_contiguous()) {
      refuse("cos and sin must be contiguous and of one shape");
    }
    call.cos_table = static_cast<const float *>(cos.data_ptr());
    call.sin_table = static_cast<const float *>(sin.data_ptr());
    call.table_positions = count_of(cos.size(0), "the tables' positions");
    call.rotary_dim = count_of(2 * cos.size(1), "rotary_dim");
  }
  call.interleaved = integer_of(a[11]) != 0 ? 1u : 0u;
  call.tokens = count_of(tokens, "tokens");
  call.heads = count_of(heads, "heads");
  at::Tensor out = a[12] != Py_None ? tensor_of(a[12], "out")
                                    : empty(ops, {tokens, heads, dim}, type);
  call.q_out = rows_of(ops, out, "out", {tokens, heads, dim}, type);
  if (a[12] != Py_None) {
    check_apart(out, "out", q, "q");
    check_apart(out, "out", tensor_of(a[2], "k"), "k");
    check_apart(out, "out", tensor_of(a[3], "v"), "v");
  }
  call_library(lro_rope_append, ops, call, "lro_rope_append");
  return wrap(std::move(out));
}

PyObject *paged_attention(const Ops &ops, PyObject *const *a) {
  at::ScalarType type;
  lro_paged_attention_t call{};
  call.cache = cache_of(ops, a[2], a[3], type);
  const at::Tensor &q = tensor_of(a[1], "q");
  check(ops, q, "q", 3, type);
  const int64_t rows = q.size(0), heads = q.size(1), dim = call.cache.head_dim;
  if (q.size(2) != dim) {
    refuse("q has a head_dim of ", q.size(2), ", the cache of ", dim);
  }
  call.q = {q.data_ptr(), q.stride(0), q.stride(1)};
  call.table = table_of(ops, tensor_of(a[4], "table"));
  if (call.table.rows != rows) {
    refuse("the table has ", call.table.rows, " rows, not ", rows);
  }
  call.lengths = vector_of<int32_t>(ops, a[5], "lengths", rows, at::kInt);
  call.scale = a[6] == Py_None ? 1.0f / std::sqrt(static_cast<float>(dim)) : number_of(a[6]);
  call.softcap = number_of(a[7]);
  call.slopes = vector_of<float>(ops, a[8], "slopes", heads, at::kFloat, true);
  const int64_t window = integer_of(a[9]);
  call.window = count_of(window, "window");
  call.heads = count_of(heads, "heads");
  at::Tensor out = a[10] != Py_None ? tensor_of(a[10], "out")
                                    : empty(ops, {rows, heads, dim}, type);
  call.out = rows_of(ops, out, "out", {rows, heads, dim}, type);
  if (a[10] != Py_None) {
    check_apart(out, "out", q, "q");
  }
  at::Tensor lse = empty(ops, {rows, heads}, at::kFloat);
  call.lse = static_cast<float *>(lse.data_ptr());
  call_library(lro_paged_attention, ops, call, "lro_paged_attention");
  return tuple_of(std::move(out), std::move(lse));
}

at::Tensor table_out_of(const Ops &ops, PyObject *object, int64_t rows, int64_t columns) {
  if (object == Py_None) {
    return empty(ops, {rows, columns}, at::kInt);
  }
  const at::Tensor &t = tensor_of(object, "table_out");
  check(ops, t, "table_out", 2, at::kInt);
  if (t.size(0) != rows || t.size(1) != columns) {
    refuse("table_out has the shape ", t.sizes(), ", not [", rows, ", ", columns, "]");
  }
  return t;
}

PyObject *fork_pages(const Ops &ops, PyObject *const *a) {
  lro_pages_fork_t call{};
  call.pool = pool_of(ops, a[1], a[2]);
  call.table = table_of(ops, tensor_of(a[3], "table"));
  call.lengths = vector_of<int32_t>(ops, a[4], "lengths", call.table.rows, at::kInt);
  const at::Tensor &parents = tensor_of(a[5], "parents");
  call.rows_out = count_of(parents.numel(), "parents");
  call.parents = vector_of<int32_t>(ops, a[5], "parents", parents.numel(), at::kInt);
  call.room = count_of(integer_of(a[6]), "room");
  call.held = vector_of<uint8_t>(ops, a[7], "held", call.pool.page_count, at::kByte, true);
  at::Tensor table = table_out_of(ops, a[8], call.rows_out, call.table.columns);
  at::Tensor lengths = empty(ops, {parents.numel()}, at::kInt);
  at::Tensor status = empty(ops, {2}, at::kInt);
  call.table_out = static_cast<int32_t *>(table.data_ptr());
  call.table_out_row_stride = table.stride(0);
  call.lengths_out = static_cast<int32_t *>(lengths.data_ptr());
  call.status = static_cast<int32_t *>(status.data_ptr());
  call_library(lro_pages_fork, ops, call, "lro_pages_fork");
  return tuple_of(std::move(table), std::move(lengths), std::move(status));
}

PyObject *compact_pages(const Ops &ops, PyObject *const *a) {
  lro_pages_compact_t call{};
  call.pool = pool_of(ops, a[1], a[2]);
  call.table = table_of(ops, tensor_of(a[3], "table"));
  call.held = vector_of<uint8_t>(ops, a[4], "held", call.pool.page_count, at::kByte, true);
  at::Tensor table = table_out_of(ops, a[5], call.table.rows, call.table.columns);
  at::Tensor status = empty(ops, {2}, at::kInt);
  call.table_out = static_cast<int32_t *>(table.data_ptr());
  call.table_out_row_stride = table.stride(0);
  call.status = static_cast<int32_t *>(status.data_ptr());
  call_library(lro_pages_compact, ops, call, "lro_pages_compact");
  return tuple_of(std::move(table), std::move(status));
}

PyObject *copy_pages(const Ops &ops, PyObject *const *a) {
  lro_pages_copy_t call{};
  call.pool = pool_of(ops, a[1], a[2]);
  const int64_t count = tensor_of(a[3], "sources").numel();
  call.sources = vector_of<int32_t>(ops, a[3], "sources", count, at::kInt);
  call.targets = vector_of<int32_t>(ops, a[4], "targets", count, at::kInt);
  call.count = count_of(count, "sources");
  call_library(lro_pages_copy, ops, call, "lro_pages_copy");
  Py_RETURN_NONE;
}

PyObject *beam_select(const Ops &ops, PyObject *const *a) {
  lro_beam_select_t call{};
  const at::Tensor &logits = tensor_of(a[1], "logits");
  call.type = type_of(logits, "logits");
  check(ops, logits, "logits", 3, logits.scalar_type());
  const int64_t groups = logits.size(0), beams = logits.size(1);
  if (groups > 1 && beams > 1 && logits.stride(0) != beams * logits.stride(1)) {
    refuse("the rows of logits must be evenly spaced");
  }
  const auto beams_of = [&](PyObject *object, const char *name, at::ScalarType type) -> void * {
    const at::Tensor &t = tensor_of(object, name);
    check(ops, t, name, 2, type);
    if (t.size(0) != groups || t.size(1) != beams || !t.is_contiguous()) {
      refuse(name, " must be contiguous, of shape [", groups, ", ", beams, "]");
    }
    return t.data_ptr();
  };
  call.logits = logits.data_ptr();
  call.logits_row_stride = beams > 1 ? logits.stride(1) : logits.stride(0);
  call.scores = static_cast<const float *>(beams_of(a[2], "scores", at::kFloat));
  call.count = count_of(integer_of(a[3]), "count");
  call.finished = a[4] == Py_None
                      ? nullptr
                      : static_cast<const uint8_t *>(beams_of(a[4], "finished", at::kByte));
  const int64_t end_token = integer_of(a[5]);
  call.end_token = end_token < 0 ? -1 : static_cast<int32_t>(count_of(end_token, "end_token"));
  call.groups = count_of(groups, "groups");
  call.beams = count_of(beams, "beams");
  call.vocab = count_of(logits.size(2), "vocab");
  const int64_t count = call.count;
  at::Tensor scores = empty(ops, {groups, count}, at::kFloat);
  at::Tensor parents = empty(ops, {groups, count}, at::kInt);
  at::Tensor tokens = empty(ops, {groups, count}, at::kInt);
  at::Tensor finished = empty(ops, {groups, count}, at::kByte);
  call.scores_out = static_cast<float *>(scores.data_ptr());
  call.parents_out = static_cast<int32_t *>(parents.data_ptr());
  call.tokens_out = static_cast<int32_t *>(tokens.data_ptr());
  call.finished_out = static_cast<uint8_t *>(finished.data_ptr());
  call_library(lro_beam_select, ops, call, "lro_beam_select");
  return tuple_of(std::move(scores), std::move(parents), std::move(tokens), std::move(finished));
}

// ---- the module ------------------------------------------------------------------

template <PyObject *(*Operator)(const Ops &, PyObject *const *), int Arguments>
PyObject *entry(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
  if (count != Arguments) {
    PyErr_Format(PyExc_TypeError, "%d arguments, not %zd", Arguments, count);
    return nullptr;
  }
  try {
    return Operator(ops_of(arguments[0]), arguments);
  } catch (const Refusal &refusal) {
    PyErr_SetString(PyExc_ValueError, refusal.text.c_str());
  } catch (const Raised &) {
  } catch (const std::exception &error) {
    PyErr_SetString(PyExc_RuntimeError, error.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown failure");
  }
  return nullptr;
}

// open(context, device, fail): what the operators' calls take first. The
// current stream is the one that they belong to.
PyObject *open_ops(PyObject *, PyObject *arguments) {
  unsigned long long context = 0;
  int device = 0;
  PyObject *fail = nullptr;
  if (!PyArg_ParseTuple(arguments, "KiO", &context, &device, &fail)) {
    return nullptr;
  }
  try {
    auto *ops = new Ops{reinterpret_cast<lro_context_t *>(context),
                        static_cast<c10::DeviceIndex>(device),
                        c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).id()};
    Py_INCREF(fail);
    Py_XSETREF(g_fail, fail);
    PyObject *capsule = PyCapsule_New(ops, kOpsCapsule, [](PyObject *object) {
      delete static_cast<Ops *>(PyCapsule_GetPointer(object, kOpsCapsule));
    });
    if (capsule == nullptr) {
      delete ops;
    }
    return capsule;
  } catch (const std::exception &error) {
    PyErr_SetString(PyExc_RuntimeError, error.what());
    return nullptr;
  }
}

// reserve(ops, workspace_bytes, counters), on whatever stream.
PyObject *reserve_ops(PyObject *, PyObject *arguments) {
  PyObject *capsule = nullptr;
  unsigned long long bytes = 0, counters = 0;
  if (!PyArg_ParseTuple(arguments, "OKK", &capsule, &bytes, &counters)) {
    return nullptr;
  }
  const auto *ops = static_cast<const Ops *>(PyCapsule_GetPointer(capsule, kOpsCapsule));
  if (ops == nullptr) {
    return nullptr;
  }
  if (ops->context == nullptr) {
    PyErr_SetString(PyExc_ValueError, "these operators are closed");
    return nullptr;
  }
  try {
    const c10::cuda::CUDAGuard guard(ops->device);
    check(lro_context_reserve(ops->context, bytes), "lro_context_reserve");
    check(lro_context_reserve_counters(ops->context, counters), "lro_context_reserve_counters");
  } catch (const Raised &) {
    return nullptr;
  }
  Py_RETURN_NONE;
}

// close(ops): its context is about to be destroyed.
PyObject *close_ops(PyObject *, PyObject *capsule) {
  auto *ops = static_cast<Ops *>(PyCapsule_GetPointer(capsule, kOpsCapsule));
  if (ops == nullptr) {
    return nullptr;
  }
  ops->context = nullptr;
  Py_RETURN_NONE;
}

#define LRRT_ENTRY(name, arguments)                                                               \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<name, arguments>)),    \
   METH_FASTCALL, nullptr}

PyMethodDef g_methods[] = {{"open", open_ops, METH_VARARGS, nullptr},
                           {"reserve", reserve_ops, METH_VARARGS, nullptr},
                           {"close", close_ops, METH_O, nullptr},
                           LRRT_ENTRY(rope_append, 13),
                           LRRT_ENTRY(paged_attention, 11),
                           LRRT_ENTRY(fork_pages, 9),
                           LRRT_ENTRY(compact_pages, 6),
                           LRRT_ENTRY(copy_pages, 5),
                           LRRT_ENTRY(beam_select, 6),
                           {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "lrrt_ops_torch", nullptr, -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit_lrrt_ops_torch(void) { return PyModule_Create(&g_module); }
