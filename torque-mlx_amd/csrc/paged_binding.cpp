// paged_binding.cpp -- the Python operators of the paged 8-bit KV cache, as a
// CPython module over the C ABI: it checks tensors, allocates results and
// workspaces from torch's allocator and launches on the current stream.
//
// Single-token calls are bound by the host: the same checks in Python with a
// ctypes call took 17 us for an attention (9 us on the GPU) and 20 for an append
// (5 us).  Arguments come by position; torque_hip/paged.py has the signatures.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <cmath>

#include "torque_hip.h"

namespace {

// The library's entry points, from the library that the package has opened.
decltype(&tq_paged_append) g_append;
decltype(&tq_paged_dequantize) g_dequantize;
decltype(&tq_paged_attention) g_attention;
decltype(&tq_paged_attention_workspace_bytes) g_workspace;
PyObject* g_check;  // raises what a negative status stands for

using at::Tensor;

std::string shape_text(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + ")";
}

const Tensor& tensor(PyObject* o, const char* name) {
  TORCH_CHECK_VALUE(THPVariable_Check(o), name, " must be a torch tensor");
  return THPVariable_Unpack(o);
}
const Tensor* tensor_or_none(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

int type_code(at::ScalarType t) {
  return t == at::kFloat ? TQ_F32 : t == at::kHalf ? TQ_F16 : t == at::kBFloat16 ? TQ_BF16 : -1;
}

struct Pool {
  const Tensor &key_pages, &value_pages, &key_scales, &value_scales;
  at::Device device;
  int pages, heads, size, dim;

  explicit Pool(PyObject* const* a)
      : key_pages(tensor(a[0], "key_pages")),
        value_pages(tensor(a[1], "value_pages")),
        key_scales(tensor(a[2], "key_scales")),
        value_scales(tensor(a[3], "value_scales")),
        device(key_pages.device()) {
    TORCH_CHECK_VALUE(key_pages.dim() == 4 && key_pages.scalar_type() == at::kChar,
                      "key_pages must be int8 [num_pages, kv_heads, page_size, head_dim]");
    const int64_t n = key_pages.size(0), h = key_pages.size(1), t = key_pages.size(2), d = key_pages.size(3);
    TORCH_CHECK_VALUE(std::max(std::max(n, h), std::max(t, d)) <= INT32_MAX, "key_pages has too many pages");
    TORCH_CHECK_VALUE(value_pages.scalar_type() == at::kChar && value_pages.sizes() == at::IntArrayRef({n, h, d, t}),
                      "value_pages must be int8 (", n, ", ", h, ", ", d, ", ", t, ") (transposed), got ", shape_text(value_pages));
    const std::pair<const char*, const Tensor*> scales[] = {{"key_scales", &key_scales}, {"value_scales", &value_scales}};
    for (const auto& [name, s] : scales)
      TORCH_CHECK_VALUE(s->scalar_type() == at::kFloat && s->sizes() == at::IntArrayRef({n, h}), name, " must be float32 (", n, ", ", h,
                        "), got ", shape_text(*s));
    const std::pair<const char*, const Tensor*> all[] = {
        {"key_pages", &key_pages}, {"value_pages", &value_pages}, {"key_scales", &key_scales}, {"value_scales", &value_scales}};
    for (const auto& [name, x] : all) {
      TORCH_CHECK_VALUE(x->device() == device && device.is_cuda(), name, " must be on the pool's HIP device");
      TORCH_CHECK_VALUE(x->is_contiguous(), name, " must be contiguous");
    }
    pages = static_cast<int>(n), heads = static_cast<int>(h), size = static_cast<int>(t), dim = static_cast<int>(d);
  }
  int8_t* keys() const { return static_cast<int8_t*>(key_pages.data_ptr()); }
  int8_t* values() const { return static_cast<int8_t*>(value_pages.data_ptr()); }
  float* kscales() const { return static_cast<float*>(key_scales.data_ptr()); }
  float* vscales() const { return static_cast<float*>(value_scales.data_ptr()); }
};

struct Batch {
  const Tensor &table, &lens;
  const Tensor* starts;
  int batch, width;
  int64_t stride;

  Batch(PyObject* const* a, const Pool& pool, int64_t tokens)
      : table(tensor(a[0], "page_table")), lens(tensor(a[1], "context_lens")), starts(tensor_or_none(a[2], "token_starts")) {
    TORCH_CHECK_VALUE(table.dim() == 2 && table.scalar_type() == at::kInt, "page_table must be int32 [batch, max_pages]");
    const int64_t b = table.size(0), w = table.size(1);
    TORCH_CHECK_VALUE(b <= INT32_MAX && w <= INT32_MAX, "page_table is too large");
    TORCH_CHECK_VALUE((w <= 1 || table.stride(1) == 1) && (b <= 1 || table.stride(0) >= w),
                      "page_table rows must be contiguous and must not overlap");
    TORCH_CHECK_VALUE(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == b && lens.is_contiguous(),
                      "context_lens must be contiguous int32 (", b, ",), got ", shape_text(lens));
    if (starts == nullptr) {
      TORCH_CHECK_VALUE(tokens == b, "without token_starts there is one token per sequence: ", tokens, " tokens, ", b, " sequences");
    } else {
      TORCH_CHECK_VALUE(starts->scalar_type() == at::kInt && starts->dim() == 1 && starts->size(0) == b + 1 && starts->is_contiguous(),
                        "token_starts must be contiguous int32 (", b + 1, ",), got ", shape_text(*starts));
    }
    const std::pair<const char*, const Tensor*> all[] = {{"page_table", &table}, {"context_lens", &lens}, {"token_starts", starts}};
    for (const auto& [name, x] : all) TORCH_CHECK_VALUE(x == nullptr || x->device() == pool.device, name, " must be on the pool's device");
    batch = static_cast<int>(b), width = static_cast<int>(w), stride = std::max(b > 1 ? table.stride(0) : w, w);
  }
  const int32_t* pages() const { return static_cast<const int32_t*>(table.data_ptr()); }
  const int32_t* lengths() const { return static_cast<const int32_t*>(lens.data_ptr()); }
  const int32_t* offsets() const { return starts == nullptr ? nullptr : static_cast<const int32_t*>(starts->data_ptr()); }
};

// [tokens, heads, head_dim] rows with unit stride along head_dim (tokens, heads: -1 for any).
Tensor rows(const Tensor& t, const char* name, const Pool& pool, int64_t tokens, int64_t heads) {
  TORCH_CHECK_VALUE(t.dim() == 3 && t.size(2) == pool.dim && (tokens < 0 || t.size(0) == tokens) && (heads < 0 || t.size(1) == heads),
                    name, " must have shape [", tokens < 0 ? "tokens" : std::to_string(tokens), ", ",
                    heads < 0 ? "heads" : std::to_string(heads), ", ", pool.dim, "], got ", shape_text(t));
  TORCH_CHECK_VALUE(type_code(t.scalar_type()) >= 0, name, " must be float32, float16 or bfloat16, got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.device() == pool.device, name, " must be on the pool's device");
  TORCH_CHECK_VALUE(!(t.requires_grad() && at::GradMode::is_enabled()), "the paged cache has no backward pass: ", name,
                    " wants a gradient (use torch.no_grad())");
  Tensor x = t.is_neg() ? t.resolve_neg() : t;
  return x.stride(2) == 1 ? x : x.contiguous();
}

void* stream_of(at::Device device) { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(device.index()).stream(); }

// Raises for a negative status.
bool fine(int status) {
  if (status >= 0) return true;
  PyObject* r = PyObject_CallFunction(g_check, "i", status);
  Py_XDECREF(r);
  return false;
}

void* data(const Tensor* t) { return t == nullptr ? nullptr : t->data_ptr(); }

// key, value, pool (4), batch (3), query, cos, sin, positions, pair_axes (bytes or None), tables_by_token,
// signs_left, signs_right, rotate_values -> the turned queries or None
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_VALUE(n == 18, "append takes 18 arguments");
  const Pool pool(a + 2);
  const Tensor key = rows(tensor(a[0], "key"), "key", pool, -1, pool.heads);
  const int64_t tokens = key.size(0);
  const Tensor value = rows(tensor(a[1], "value"), "value", pool, tokens, pool.heads);
  TORCH_CHECK_VALUE(key.scalar_type() == value.scalar_type(), "key and value must share a dtype, got ", key.scalar_type(), " and ",
                    value.scalar_type());
  const Batch batch(a + 6, pool, tokens);
  const c10::DeviceGuard guard(pool.device);
  Tensor query, query_out;
  if (a[9] != Py_None) {
    query = rows(tensor(a[9], "query"), "query", pool, tokens, -1);
    query_out = at::empty(query.sizes(), query.options());
  }
  const Tensor *cos_in = tensor_or_none(a[10], "cos"), *sin_in = tensor_or_none(a[11], "sin");
  const Tensor* positions_in = tensor_or_none(a[12], "positions");
  const bool by_token = PyObject_IsTrue(a[14]) == 1;
  TORCH_CHECK_VALUE((cos_in == nullptr) == (sin_in == nullptr), "cos and sin come together");
  Tensor cos, sin, positions;
  int64_t table_rows = 0;
  int rotary = 0, table_type = 0, axes = 1;
  if (cos_in != nullptr) {
    TORCH_CHECK_VALUE(cos_in->dim() == 2 && cos_in->sizes() == sin_in->sizes() && cos_in->scalar_type() == sin_in->scalar_type() &&
                          type_code(cos_in->scalar_type()) >= 0,
                      "cos and sin must be [rows, rotary_dim] of one floating dtype");
    TORCH_CHECK_VALUE(cos_in->device() == pool.device && sin_in->device() == pool.device, "cos and sin must be on the pool's device");
    TORCH_CHECK_VALUE(cos_in->size(1) <= pool.dim, "rotary_dim must be even and at most head_dim");
    const auto plain = [](const Tensor& t) {
      const Tensor x = t.is_neg() ? t.resolve_neg() : t;
      return x.size(1) <= 1 || x.stride(1) == 1 ? x : x.contiguous();
    };
    cos = plain(*cos_in), sin = plain(*sin_in);
    table_rows = cos.size(0), rotary = static_cast<int>(cos.size(1)), table_type = type_code(cos.scalar_type());
  } else {
    TORCH_CHECK_VALUE(positions_in == nullptr && a[13] == Py_None && !by_token, "positions, pair_axes and tables_by_token need cos and sin");
  }
  if (positions_in != nullptr) {
    TORCH_CHECK_VALUE((positions_in->scalar_type() == at::kInt || positions_in->scalar_type() == at::kLong) &&
                          positions_in->device() == pool.device,
                      "positions must be int32 or int64 on the pool's device");
    const int64_t dims = positions_in->dim();
    TORCH_CHECK_VALUE((dims == 1 || dims == 2) && positions_in->size(dims - 1) == tokens, "positions must be [", tokens, "] or [axes, ",
                      tokens, "], got ", shape_text(*positions_in));
    positions = tokens <= 1 || positions_in->stride(dims - 1) == 1 ? *positions_in : positions_in->contiguous();
    if (dims == 2) axes = static_cast<int>(std::min<int64_t>(positions.size(0), 1 << 20));
  }
  const uint8_t* pair_axes = nullptr;
  if (a[13] != Py_None) {
    TORCH_CHECK_VALUE(PyBytes_Check(a[13]), "pair_axes must be bytes");
    TORCH_CHECK_VALUE(PyBytes_GET_SIZE(a[13]) == rotary / 2, "pair_axes must name ", rotary / 2, " axes, got ", PyBytes_GET_SIZE(a[13]));
    pair_axes = reinterpret_cast<const uint8_t*>(PyBytes_AS_STRING(a[13]));
  }
  const Tensor *left = tensor_or_none(a[15], "signs_left"), *right = tensor_or_none(a[16], "signs_right");
  const std::pair<const char*, const Tensor*> signs[] = {{"signs_left", left}, {"signs_right", right}};
  for (const auto& [name, s] : signs)
    TORCH_CHECK_VALUE(s == nullptr || (s->scalar_type() == at::kFloat && s->dim() == 1 && s->size(0) == pool.dim &&
                                       s->device() == pool.device && s->is_contiguous() && !s->is_neg()),
                      name, " must be contiguous float32 [", pool.dim, "] on the pool's device");
  const int flags = (PyObject_IsTrue(a[17]) == 1 ? TQ_ROTATE_VALUES : 0) | (by_token ? TQ_TABLES_BY_TOKEN : 0);
  const bool q = query.defined();
  const int status = g_append(
      key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0), value.stride(1), type_code(key.scalar_type()),
      q ? query.data_ptr() : nullptr, q ? query.stride(0) : 0, q ? query.stride(1) : 0, q ? type_code(query.scalar_type()) : 0,
      q ? static_cast<int>(query.size(1)) : 0, q ? query_out.data_ptr() : nullptr, tokens, pool.heads, pool.dim, pool.keys(), pool.values(),
      pool.kscales(), pool.vscales(), pool.pages, pool.size, batch.pages(), batch.stride, batch.width, batch.lengths(), batch.offsets(),
      batch.batch, cos.defined() ? cos.data_ptr() : nullptr, cos.defined() ? cos.stride(0) : 0, sin.defined() ? sin.data_ptr() : nullptr,
      sin.defined() ? sin.stride(0) : 0, table_type, table_rows, rotary, positions.defined() ? positions.data_ptr() : nullptr,
      positions.defined() && positions.scalar_type() == at::kLong, positions.defined() && positions.dim() == 2 ? positions.stride(0) : 0, axes,
      pair_axes, static_cast<const float*>(data(left)), static_cast<const float*>(data(right)), flags,
      static_cast<hipStream_t>(stream_of(pool.device)));
  if (!fine(status)) return nullptr;
  if (!q) Py_RETURN_NONE;
  return THPVariable_Wrap(query_out);
  END_HANDLE_TH_ERRORS
}

// page_ids, pool (4), dtype -> (keys, values)
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_VALUE(n == 6, "dequantize takes 6 arguments");
  const Pool pool(a + 1);
  const Tensor& ids = tensor(a[0], "page_ids");
  TORCH_CHECK_VALUE(ids.scalar_type() == at::kInt && ids.dim() == 1 && ids.device() == pool.device && ids.is_contiguous(),
                    "page_ids must be contiguous int32 [count] on the pool's device");
  TORCH_CHECK_VALUE(THPDtype_Check(a[5]), "dtype must be a torch dtype");
  const at::ScalarType type = reinterpret_cast<THPDtype*>(a[5])->scalar_type;
  TORCH_CHECK_VALUE(type_code(type) >= 0, "dtype must be float32, float16 or bfloat16, got ", type);
  const c10::DeviceGuard guard(pool.device);
  const std::array<int64_t, 4> shape{ids.size(0), pool.heads, pool.size, pool.dim};
  const auto options = pool.key_pages.options().dtype(type);
  const Tensor keys = at::empty(shape, options), values = at::empty(shape, options);
  const int status = g_dequantize(static_cast<const int32_t*>(ids.data_ptr()), ids.size(0), pool.keys(), pool.values(), pool.kscales(),
                                  pool.vscales(), pool.pages, pool.size, pool.heads, pool.dim, keys.data_ptr(), values.data_ptr(),
                                  type_code(type), static_cast<hipStream_t>(stream_of(pool.device)));
  if (!fine(status)) return nullptr;
  return Py_BuildValue("(NN)", THPVariable_Wrap(keys), THPVariable_Wrap(values));
  END_HANDLE_TH_ERRORS
}

// query, pool (4), batch (3), max_tokens (0: unknown), scale (None: head_dim ** -0.5), out -> out
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  TORCH_CHECK_VALUE(n == 11, "attention takes 11 arguments");
  const Pool pool(a + 1);
  const Tensor query = rows(tensor(a[0], "query"), "query", pool, -1, -1);
  const int64_t tokens = query.size(0), heads = query.size(1);
  TORCH_CHECK_VALUE(heads <= INT32_MAX, "query has too many heads");
  const Batch batch(a + 5, pool, tokens);
  const long long most = PyLong_AsLongLong(a[8]);
  double scale = 1.0 / std::sqrt(static_cast<double>(pool.dim));
  if (a[9] != Py_None) scale = PyFloat_AsDouble(a[9]);
  if (PyErr_Occurred()) return nullptr;
  const c10::DeviceGuard guard(pool.device);
  Tensor out;
  if (a[10] == Py_None) {
    out = batch.starts == nullptr ? at::empty(query.sizes(), query.options()) : at::zeros(query.sizes(), query.options());
  } else {
    out = tensor(a[10], "out");
    TORCH_CHECK_VALUE(out.sizes() == query.sizes() && out.scalar_type() == query.scalar_type() && out.device() == pool.device,
                      "out must be ", query.scalar_type(), " ", shape_text(query), " on the pool's device");
    TORCH_CHECK_VALUE(out.stride(2) == 1 && !out.is_neg(), "out must have unit stride along head_dim");
    TORCH_CHECK_VALUE(!(out.requires_grad() && at::GradMode::is_enabled()),
                      "the paged cache has no backward pass: out wants a gradient (use torch.no_grad())");
    TORCH_CHECK_VALUE(!out.storage().is_alias_of(query.storage()), "out must not share memory with query");
    TORCH_CHECK_VALUE(at::has_internal_overlap(out) != at::MemOverlap::Yes, "out must not overlap itself");
  }
  const size_t bytes = g_workspace(tokens, batch.batch, batch.starts != nullptr, static_cast<int>(heads), pool.heads, pool.dim, batch.width,
                                   pool.size, most, 0);
  // A tensor of the call's own, from the stream's pool or the graph's: calls on other streams and other graphs' replays have theirs.
  Tensor workspace;
  if (bytes > 0) workspace = at::empty({static_cast<int64_t>(bytes)}, pool.key_pages.options());
  const int status = g_attention(query.data_ptr(), query.stride(0), query.stride(1), type_code(query.scalar_type()), tokens,
                                 static_cast<int>(heads), pool.heads, pool.dim, pool.keys(), pool.values(), pool.kscales(), pool.vscales(),
                                 pool.pages, pool.size, batch.pages(), batch.stride, batch.width, batch.lengths(), batch.offsets(),
                                 batch.batch, most, static_cast<float>(scale), bytes > 0 ? workspace.data_ptr() : nullptr, bytes,
                                 out.data_ptr(), out.stride(0), out.stride(1), static_cast<hipStream_t>(stream_of(pool.device)));
  if (!fine(status)) return nullptr;
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// Addresses of the library's entry points and the callable that raises for a status.
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long append_at, dequantize_at, attention_at, workspace_at;
  PyObject* check;
  if (!PyArg_ParseTuple(args, "KKKKO", &append_at, &dequantize_at, &attention_at, &workspace_at, &check)) return nullptr;
  g_append = reinterpret_cast<decltype(g_append)>(append_at);
  g_dequantize = reinterpret_cast<decltype(g_dequantize)>(dequantize_at);
  g_attention = reinterpret_cast<decltype(g_attention)>(attention_at);
  g_workspace = reinterpret_cast<decltype(g_workspace)>(workspace_at);
  Py_INCREF(check);
  g_check = check;
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(append)), METH_FASTCALL, nullptr},
    {"dequantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(dequantize)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(attention)), METH_FASTCALL, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_paged", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged(void) { return PyModule_Create(&g_module); }
