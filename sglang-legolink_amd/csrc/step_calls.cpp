// The calls of a model's step (rotate_heads, append_rotated_kv_inplace,
// paged_attention) from their tensors: checks, outputs and the library's entry in
// one native call.
//
// A decode step makes these calls once per layer on a few rows, where the GPU
// takes 4 us; the checks and the argument block take Python 15 to 25 us a call,
// here 1 to 2 us.
//
// Each function returns None where a check of the Python operator does not hold,
// with nothing allocated or launched: the caller then runs the Python checks,
// which name the reason (or take the call: only plain tensors on the current
// device, and outputs that are new or the input itself, are taken here).  A
// non-zero status of the library's entry comes back as an int.  Whatever fails once
// the entry was called is raised: the call must not be made again.  With entry 0
// the checks run alone, on tensors of any device, and True comes back.
//
// The module names the torch version and the block sizes that it was built for:
// the caller uses it only where they are its own.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <cstdint>
#include <cstring>

#include "legolink_kv.h"

namespace {

// A strided tensor that needs no gradient and has no forward-mode tangent (which
// no_grad does not switch off).
const at::Tensor *plain(PyObject *object) {
  if (object == nullptr || !THPVariable_CheckExact(object)) return nullptr;
  const at::Tensor &t = THPVariable_Unpack(object);
  if (t.layout() != at::kStrided || (t.requires_grad() && c10::GradMode::is_enabled()) || t.is_conj() || t.is_neg())
    return nullptr;
  if (t._fw_grad(/*level=*/0).defined()) return nullptr;
  return &t;
}

int64_t half_code(at::ScalarType type) {
  return type == at::kHalf ? LL_DTYPE_FLOAT16 : type == at::kBFloat16 ? LL_DTYPE_BFLOAT16 : -1;
}
int64_t float_code(at::ScalarType type) { return type == at::kFloat ? LL_DTYPE_FLOAT32 : half_code(type); }
int64_t index_code(at::ScalarType type) {
  return type == at::kInt ? LL_DTYPE_INT32 : type == at::kLong ? LL_DTYPE_INT64 : -1;
}

struct Span {
  uintptr_t begin, end;
};
Span span_of(const at::Tensor &t) {
  const auto begin = reinterpret_cast<uintptr_t>(t.data_ptr());
  int64_t reach = 0;
  for (int64_t i = 0; i < t.dim(); ++i) reach += (t.size(i) - 1) * t.stride(i);
  return {begin, begin + static_cast<uintptr_t>((reach + 1) * t.element_size())};
}

// Whether two sets of rows [tokens, heads, dim] share bytes: exact for dense heads
// of one token stride, else where their spans meet.
bool overlap(const at::Tensor &a, const at::Tensor &b) {
  if (a.numel() == 0 || b.numel() == 0) return false;
  const Span x = span_of(a), y = span_of(b);
  if (x.end <= y.begin || y.end <= x.begin) return false;
  const auto dense = [](const at::Tensor &t) {
    return t.dim() == 3 && t.stride(2) == 1 && (t.size(1) == 1 || t.stride(1) == t.size(2));
  };
  if (!dense(a) || !dense(b) || a.stride(0) != b.stride(0)) return true;
  const int64_t stride = a.stride(0) * a.element_size();
  const int64_t wide = a.size(1) * a.size(2) * a.element_size(), other = b.size(1) * b.size(2) * b.element_size();
  if (stride < std::max(wide, other)) return true;
  int64_t offset = (static_cast<int64_t>(y.begin) - static_cast<int64_t>(x.begin)) % stride;
  if (offset < 0) offset += stride;
  return offset < wide || stride - offset < other;
}

bool rows_ok(const at::Tensor *t, int64_t tokens, const at::Tensor &query) {
  return t != nullptr && t->dim() == 3 && t->size(0) == tokens && t->size(1) >= 1 && t->size(2) >= 1 &&
         t->scalar_type() == query.scalar_type() && t->device() == query.device() &&
         (t->size(2) == 1 || t->stride(2) == 1);
}

bool vector_ok(const at::Tensor *t, int64_t count, at::Device device) {
  return t != nullptr && t->dim() == 1 && t->numel() == count && t->device() == device && t->is_contiguous();
}

// Rows that do not overlap each other, as an output must not.
bool apart(const at::Tensor &t) {
  const int64_t tokens = t.size(0), heads = t.size(1), dim = t.size(2), token = t.stride(0), head = t.stride(1);
  return ((heads == 1 || head >= dim) && (tokens == 1 || token >= (heads - 1) * head + dim)) ||
         ((tokens == 1 || token >= dim) && (heads == 1 || head >= (tokens - 1) * token + dim));
}

bool integer(PyObject *object, int64_t *out) {
  if (!PyLong_CheckExact(object)) return false;
  *out = PyLong_AsLongLong(object);
  return !PyErr_Occurred();
}
bool number(PyObject *object, double *out) {
  if (!PyFloat_CheckExact(object) && !PyLong_CheckExact(object)) return false;
  *out = PyFloat_AsDouble(object);
  return !PyErr_Occurred();
}

// Where a call goes: the library's entry (0: checks alone), the stream, the
// current device.
struct Target {
  int64_t entry = 0, stream = 0, device = 0;
  bool read(PyObject *const *a) { return integer(a[0], &entry) && integer(a[1], &stream) && integer(a[2], &device); }
  // (Tensors in host memory have the index -1, which is no current device's.)
  bool takes(const at::Tensor &query) const { return entry == 0 || query.device().index() == device; }

  // The entry's status.  The call's result is made before it: behind it nothing is
  // left that could fail.
  template <typename Args>
  int call(const Args *args, bool *launched) const {
    typedef int (*Entry)(const Args *, ll_stream_t);
    *launched = true;
    return reinterpret_cast<Entry>(entry)(args, reinterpret_cast<ll_stream_t>(stream));
  }
};

// An owned reference.
struct Object {
  PyObject *held;
  explicit Object(PyObject *object) : held(object) {}
  Object(const Object &) = delete;
  ~Object() { Py_XDECREF(held); }
  PyObject *release() {
    PyObject *object = held;
    held = nullptr;
    return object;
  }
};

PyObject *none() { Py_RETURN_NONE; }

// The tensors of a call that are not its rows: read, but for the counter.
struct Beside {
  std::array<const at::Tensor *, 4> read{};  // positions, table, norm weights (or null)
  const at::Tensor *skipped = nullptr;

  bool meets(const at::Tensor &written) const {
    for (const at::Tensor *other : read)
      if (other != nullptr && overlap(written, *other)) return true;
    return skipped != nullptr && overlap(written, *skipped);
  }
  bool counter_apart(std::initializer_list<const at::Tensor *> rows) const {
    if (skipped == nullptr) return true;
    for (const at::Tensor *other : read)
      if (other != nullptr && overlap(*skipped, *other)) return false;
    for (const at::Tensor *other : rows)
      if (overlap(*skipped, *other)) return false;
    return true;
  }
};

// What rotate_heads and append_rotated_kv_inplace have in common: query, key,
// positions, cos_sin_cache, rotary_dim, neox, query norm, key norm, eps, skipped.
bool read_rotary(PyObject *const *a, ll_head_rotary_args *args, const at::Tensor **query_out,
                 const at::Tensor **key_out, Beside *beside) {
  const at::Tensor *query = plain(a[0]), *key = plain(a[1]), *positions = plain(a[2]), *table = plain(a[3]);
  if (query == nullptr || query->dim() != 3) return false;
  const at::Device device = query->device();
  const int64_t tokens = query->size(0);
  args->dtype = half_code(query->scalar_type());
  if (args->dtype < 0 || !rows_ok(query, tokens, *query) || !rows_ok(key, tokens, *query)) return false;
  const int64_t dim = query->size(2);
  int64_t rotary = 0;
  if (key->size(2) != dim || dim > 256 || !integer(a[4], &rotary) || rotary < 2 || rotary % 2 != 0 || rotary > dim)
    return false;
  if (a[5] != Py_True && a[5] != Py_False) return false;
  if (!vector_ok(positions, tokens, device)) return false;
  args->positions_dtype = index_code(positions->scalar_type());
  if (args->positions_dtype < 0) return false;
  if (table == nullptr || table->dim() != 2 || table->size(1) < rotary || table->device() != device ||
      table->stride(1) != 1)
    return false;
  args->cos_sin_dtype = float_code(table->scalar_type());
  if (args->cos_sin_dtype < 0) return false;
  const void **weights[2] = {&args->query_norm_weight, &args->key_norm_weight};
  args->norm_weight_dtype = 0;
  for (int i = 0; i < 2; ++i) {
    *weights[i] = nullptr;
    if (a[6 + i] == Py_None) continue;
    const at::Tensor *weight = plain(a[6 + i]);
    if (!vector_ok(weight, dim, device)) return false;
    const int64_t code = float_code(weight->scalar_type());
    if (code < 0 || (args->norm_weight_dtype != 0 && args->norm_weight_dtype != code)) return false;
    args->norm_weight_dtype = code;
    *weights[i] = weight->data_ptr();
    beside->read[2 + i] = weight;
  }
  beside->read[0] = positions;
  beside->read[1] = table;
  if (!number(a[8], &args->norm_eps) || !(args->norm_eps >= 0.0)) return false;
  args->skipped_rows = nullptr;
  if (a[9] != Py_None) {
    const at::Tensor *skipped = plain(a[9]);
    if (skipped == nullptr || skipped->scalar_type() != at::kLong || skipped->numel() != 1 ||
        skipped->device() != device)
      return false;
    args->skipped_rows = static_cast<int64_t *>(skipped->data_ptr());
    beside->skipped = skipped;
  }
  args->struct_size = sizeof(ll_head_rotary_args);
  args->num_tokens = tokens;
  args->num_q_heads = query->size(1);
  args->num_kv_heads = key->size(1);
  args->head_dim = dim;
  args->query = query->data_ptr();
  args->query_token_stride = query->stride(0);
  args->query_head_stride = query->stride(1);
  args->key = key->data_ptr();
  args->key_token_stride = key->stride(0);
  args->key_head_stride = key->stride(1);
  args->positions = positions->data_ptr();
  args->cos_sin_cache = table->data_ptr();
  args->cos_sin_rows = table->size(0);
  args->cos_sin_cols = table->size(1);
  args->cos_sin_stride_row = table->stride(0);
  args->rotary_dim = rotary;
  args->is_neox_style = a[5] == Py_True;
  *query_out = query;
  *key_out = key;
  return true;
}

// An output that is its own input (the same Python object): its rows must lie
// apart, and not meet the call's other tensors.  The others go by their role: one
// that is the same object as the output is read by other waves while it is written.
bool in_place(const at::Tensor &rows, std::initializer_list<const at::Tensor *> others, const Beside &beside) {
  if (!apart(rows) || beside.meets(rows)) return false;
  for (const at::Tensor *other : others)
    if (overlap(rows, *other)) return false;
  return true;
}

at::Tensor empty_like_rows(const at::Tensor &rows) { return at::empty(rows.sizes(), rows.options()); }

void set_output(const at::Tensor &t, void **base, int64_t *token, int64_t *head) {
  *base = t.data_ptr();
  *token = t.stride(0);
  *head = t.stride(1);
}

// (entry, stream, device, query, key, positions, table, rotary_dim, neox, query
// norm, key norm, eps, skipped, query_output, key_output) -> (query, key)
PyObject *rotate_heads(PyObject *const *a, Py_ssize_t n, bool *launched) {
  Target target;
  ll_head_rotary_args args;
  memset(&args, 0, sizeof(args));
  const at::Tensor *query, *key;
  Beside beside;
  if (n != 15 || !target.read(a) || !read_rotary(a + 3, &args, &query, &key, &beside) || !target.takes(*query) ||
      !beside.counter_apart({query, key}))
    return none();
  const bool query_in_place = a[13] != Py_None, key_in_place = a[14] != Py_None;
  if (query_in_place && (a[13] != a[3] || !in_place(*query, {key}, beside))) return none();
  if (key_in_place && (a[14] != a[4] || !in_place(*key, {query}, beside))) return none();
  if (target.entry == 0) Py_RETURN_TRUE;
  const at::Tensor query_output = query_in_place ? *query : empty_like_rows(*query);
  const at::Tensor key_output = key_in_place ? *key : empty_like_rows(*key);
  set_output(query_output, &args.query_output, &args.query_output_token_stride, &args.query_output_head_stride);
  set_output(key_output, &args.key_output, &args.key_output_token_stride, &args.key_output_head_stride);
  Object first(THPVariable_Wrap(query_output)), second(THPVariable_Wrap(key_output));
  if (first.held == nullptr || second.held == nullptr) return nullptr;
  Object both(PyTuple_Pack(2, first.held, second.held));
  if (both.held == nullptr) return nullptr;
  const int status = target.call(&args, launched);
  return status != LL_OK ? PyLong_FromLong(status) : both.release();
}

// (entry, stream, device, query, key, positions, table, rotary_dim, neox, query
// norm, key norm, eps, skipped, query_output, value, key_buffer, value_buffer,
// slots) -> query
PyObject *append(PyObject *const *a, Py_ssize_t n, bool *launched) {
  Target target;
  ll_head_rotary_args args;
  memset(&args, 0, sizeof(args));
  const at::Tensor *query, *key;
  Beside beside;
  if (n != 18 || !target.read(a) || !read_rotary(a + 3, &args, &query, &key, &beside) || !target.takes(*query))
    return none();
  const at::Tensor *value = plain(a[14]), *keys = plain(a[15]), *values = plain(a[16]), *slots = plain(a[17]);
  if (args.num_tokens == 0 || !rows_ok(value, args.num_tokens, *query) || value->size(1) != key->size(1) ||
      value->size(2) > 256 || !vector_ok(slots, args.num_tokens, query->device()) ||
      !beside.counter_apart({query, key, value, slots}))
    return none();
  args.destination_slots_dtype = index_code(slots->scalar_type());
  if (args.destination_slots_dtype < 0) return none();
  const at::Tensor *buffers[2] = {keys, values}, *rows[2] = {key, value};
  for (int i = 0; i < 2; ++i) {
    const at::Tensor *buffer = buffers[i];
    if (buffer == nullptr || buffer->dim() != 3 || buffer->size(0) != keys->size(0) ||
        buffer->size(1) != rows[i]->size(1) || buffer->size(2) != rows[i]->size(2) ||
        buffer->scalar_type() != query->scalar_type() || buffer->device() != query->device() ||
        !buffer->is_contiguous() || overlap(*buffer, *query) || overlap(*buffer, *key) || overlap(*buffer, *value) ||
        overlap(*buffer, *slots) || beside.meets(*buffer))
      return none();
  }
  if (overlap(*keys, *values)) return none();
  const bool query_in_place = a[13] != Py_None;
  if (query_in_place && (a[13] != a[3] || !in_place(*query, {key, value, keys, values, slots}, beside))) return none();
  if (target.entry == 0) Py_RETURN_TRUE;
  const at::Tensor query_output = query_in_place ? *query : empty_like_rows(*query);
  set_output(query_output, &args.query_output, &args.query_output_token_stride, &args.query_output_head_stride);
  args.value = value->data_ptr();
  args.value_token_stride = value->stride(0);
  args.value_head_stride = value->stride(1);
  args.value_head_dim = value->size(2);
  args.key_buffer = keys->data_ptr();
  args.value_buffer = values->data_ptr();
  args.num_slots = keys->size(0);
  args.destination_slots = slots->data_ptr();
  Object result(THPVariable_Wrap(query_output));
  if (result.held == nullptr) return nullptr;
  const int status = target.call(&args, launched);
  return status != LL_OK ? PyLong_FromLong(status) : result.release();
}

typedef int64_t (*WorkspaceEntry)(const ll_paged_attention_args *);

// (entry, stream, device, workspace entry, query, key_buffer, value_buffer,
// page_table, kv_lengths, page_size, query_starts, scale) -> output
PyObject *paged_attention(PyObject *const *a, Py_ssize_t n, bool *launched) {
  Target target;
  int64_t workspace_entry = 0, page_size = 0;
  if (n != 12 || !target.read(a) || !integer(a[3], &workspace_entry)) return none();
  const at::Tensor *query = plain(a[4]), *keys = plain(a[5]), *values = plain(a[6]), *pages = plain(a[7]),
                   *lengths = plain(a[8]);
  if (query == nullptr || keys == nullptr || values == nullptr || pages == nullptr || !target.takes(*query))
    return none();
  ll_paged_attention_args args;
  memset(&args, 0, sizeof(args));
  const at::Device device = query->device();
  args.kv_dtype = half_code(query->scalar_type());
  if (args.kv_dtype < 0 || query->dim() != 3 || keys->dim() != 3 || values->sizes() != keys->sizes()) return none();
  const int64_t queries = query->size(0), q_heads = query->size(1), dim = query->size(2), kv_heads = keys->size(1);
  if (keys->size(2) != dim || (dim != 64 && dim != 128 && dim != 256) || kv_heads < 1 || q_heads < 1 ||
      q_heads % kv_heads != 0)
    return none();
  for (const at::Tensor *buffer : {keys, values})
    if (buffer->scalar_type() != query->scalar_type() || buffer->device() != device || !buffer->is_contiguous() ||
        reinterpret_cast<uintptr_t>(buffer->data_ptr()) % 16 != 0)
      return none();
  if (pages->dim() != 2 || pages->scalar_type() != at::kInt || pages->device() != device ||
      (pages->size(1) > 1 && pages->stride(1) != 1))
    return none();
  const int64_t requests = pages->size(0);
  if (!integer(a[9], &page_size) || page_size < 1 || !vector_ok(lengths, requests, device)) return none();
  args.kv_lengths_dtype = index_code(lengths->scalar_type());
  if (args.kv_lengths_dtype < 0) return none();
  if (a[10] != Py_None) {
    const at::Tensor *starts = plain(a[10]);
    if (!vector_ok(starts, requests + 1, device)) return none();
    args.query_starts = starts->data_ptr();
    args.query_starts_dtype = index_code(starts->scalar_type());
    if (args.query_starts_dtype < 0) return none();
  } else if (queries != requests) {
    return none();
  }
  if (a[11] == Py_None) args.softmax_scale = 1.0 / std::sqrt(static_cast<double>(dim));
  else if (!number(a[11], &args.softmax_scale)) return none();
  if (!(args.softmax_scale >= 1e-37 && args.softmax_scale < 1e30)) return none();
  if (query->stride(2) != 1 || query->stride(0) % 8 != 0 || query->stride(1) % 8 != 0 ||
      reinterpret_cast<uintptr_t>(query->data_ptr()) % 16 != 0)
    return none();
  if (target.entry == 0) Py_RETURN_TRUE;
  args.struct_size = sizeof(args);
  args.query = query->data_ptr();
  args.query_token_stride = query->stride(0);
  args.query_head_stride = query->stride(1);
  args.num_queries = queries;
  args.key_buffer = keys->data_ptr();
  args.value_buffer = values->data_ptr();
  args.num_slots = keys->size(0);
  args.num_q_heads = q_heads;
  args.num_kv_heads = kv_heads;
  args.head_dim = dim;
  args.page_table = static_cast<const int32_t *>(pages->data_ptr());
  args.page_table_stride = pages->stride(0);
  args.page_table_columns = pages->size(1);
  args.page_size = page_size;
  args.kv_lengths = lengths->data_ptr();
  args.num_requests = requests;
  const at::Tensor output = at::empty({queries, q_heads, dim}, query->options());
  args.output = output.data_ptr();
  const int64_t needed = reinterpret_cast<WorkspaceEntry>(workspace_entry)(&args);
  if (needed < 0) return PyLong_FromLongLong(needed);
  at::Tensor workspace;
  if (needed > 0) {
    workspace = at::empty({needed}, query->options().dtype(at::kByte));
    args.workspace = workspace.data_ptr();
    args.workspace_bytes = needed;
  }
  Object result(THPVariable_Wrap(output));
  if (result.held == nullptr) return nullptr;
  const int status = target.call(&args, launched);
  return status != LL_OK ? PyLong_FromLong(status) : result.release();
}

// No C++ exception leaves a call.  What fails before the library's entry is called,
// an allocation say, is left to the Python path, which meets it again; from there
// on it is raised.
typedef PyObject *Call(PyObject *const *, Py_ssize_t, bool *);

template <Call *kCall>
PyObject *guarded(PyObject *, PyObject *const *arguments, Py_ssize_t count) {
  PyObject *result = nullptr;
  bool launched = false;
  try {
    result = kCall(arguments, count, &launched);
  } catch (...) {
    result = nullptr;
  }
  if (result != nullptr && !PyErr_Occurred()) return result;
  Py_XDECREF(result);
  if (!launched) {
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "a step call failed behind its launch");
  return nullptr;
}

template <Call *kCall>
PyCFunction entry() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<kCall>));
}

PyMethodDef methods[] = {
    {"rotate_heads", entry<rotate_heads>(), METH_FASTCALL, "rotate_heads in one call, or None"},
    {"append", entry<append>(), METH_FASTCALL, "append_rotated_kv_inplace in one call, or None"},
    {"paged_attention", entry<paged_attention>(), METH_FASTCALL, "paged_attention in one call, or None"},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_step_calls", "A step's calls from their tensors.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__step_calls(void) {
  PyObject *created = PyModule_Create(&module);
  if (created == nullptr) return nullptr;
  if (PyModule_AddStringConstant(created, "TORCH_VERSION", TORCH_VERSION) != 0 ||
      PyModule_AddIntConstant(created, "HEAD_ROTARY_ARGS_SIZE", sizeof(ll_head_rotary_args)) != 0 ||
      PyModule_AddIntConstant(created, "PAGED_ATTENTION_ARGS_SIZE", sizeof(ll_paged_attention_args)) != 0) {
    Py_DECREF(created);
    return nullptr;
  }
  return created;
}
