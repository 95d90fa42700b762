// Python bindings of the operators whose calls are short beside a Python
// layer's checks: argument checks, output allocation and the C call in one
// step.  (A wrapper that checks ten tensors attribute by attribute and calls
// through ctypes takes 15 to 30 us; a decode step's kernels take 5 to 10.)
//
// The module holds no state but, per GPU, the address of the error word that
// the Python side owns.  Refusals become the Python exceptions that the
// package's documentation names; no C++ exception leaves a function.
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <initializer_list>
#include <string>

#include "iris_b200.h"

namespace {

using at::Tensor;

struct Refusal {
  PyObject* type;
  std::string text;
};
struct Raised {};  // a Python exception is set already

[[noreturn]] void refuse(PyObject* type, std::string text) { throw Refusal{type, std::move(text)}; }
void require(bool ok, PyObject* type, const char* text) {
  if (!ok) refuse(type, text);
}

const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string(name) + " must be a torch.Tensor");
  return THPVariable_Unpack(o);
}
const Tensor* optional_tensor(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}
int32_t integer32(PyObject* o, const char* name) {
  const int64_t v = integer(o);
  if (v < INT32_MIN || v > INT32_MAX) refuse(PyExc_ValueError, std::string(name) + " is out of range");
  return static_cast<int32_t>(v);
}

const char* type_name(at::ScalarType t) {
  switch (t) {
    case at::kByte: return "torch.uint8";
    case at::kChar: return "torch.int8";
    case at::kInt: return "torch.int32";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kFloat: return "torch.float32";
    default: return "another type";
  }
}

std::string shape_text(at::IntArrayRef s) {
  std::string out = "(";
  for (size_t i = 0; i < s.size(); ++i) out += (i ? ", " : "") + std::to_string(s[i]);
  return out + (s.size() == 1 ? ",)" : ")");
}

// Shape, type, device and contiguity of one argument.
void check(const char* name, const Tensor& t, at::IntArrayRef shape, at::ScalarType type, c10::Device device) {
  if (t.sizes() != shape) refuse(PyExc_ValueError, std::string(name) + " must have shape " + shape_text(shape));
  if (t.scalar_type() != type) refuse(PyExc_TypeError, std::string(name) + " must use " + type_name(type));
  if (t.device() != device) refuse(PyExc_ValueError, std::string(name) + " must be on " + device.str());
  if (!t.is_contiguous()) refuse(PyExc_ValueError, std::string(name) + " must be contiguous");
}

int32_t dtype_code(const char* name, at::ScalarType t) {
  if (t == at::kHalf) return IRIS_DTYPE_FP16;
  if (t == at::kBFloat16) return IRIS_DTYPE_BF16;
  refuse(PyExc_TypeError, std::string(name) + " must use FP16(torch.float16) or BF16(torch.bfloat16)");
}

// Rows [B, width] of int32 that may be apart.
struct Table {
  const int32_t* data;
  int64_t stride;
  int32_t width;
};
Table block_table(const Tensor& t, int64_t batch, c10::Device device) {
  require(t.dim() == 2 && t.size(0) == batch, PyExc_ValueError,
          "block_table must have shape [B, max_pages_per_sequence]");
  require(t.scalar_type() == at::kInt, PyExc_TypeError, "block_table must use torch.int32");
  if (t.device() != device) refuse(PyExc_ValueError, "block_table must be on " + device.str());
  require(batch == 0 || t.size(1) > 0, PyExc_ValueError, "block_table must have at least one column");
  require(t.size(1) <= 1 || t.stride(1) == 1, PyExc_ValueError, "block_table rows must be contiguous");
  require(t.size(1) <= INT32_MAX, PyExc_ValueError, "block_table has too many columns");
  return {static_cast<const int32_t*>(t.const_data_ptr()), t.stride(0), static_cast<int32_t>(t.size(1))};
}

// ------------------------------------------------------------------ devices
constexpr int kMaxDevices = 64;
PyObject* g_prepare = nullptr;  // prepare(index) -> address of the GPU's error word; raises if it cannot run the kernels
int32_t* g_words[kMaxDevices] = {};

c10::Device device_of(const char* name, const Tensor& t) {
  if (!t.is_cuda()) {
    require(c10::cuda::device_count() > 0, PyExc_RuntimeError, "Iris fused kernels require CUDA");
    refuse(PyExc_ValueError, std::string(name) + " must be a CUDA tensor");
  }
  return t.device();
}

int32_t* error_word(c10::Device device) {
  const int index = device.index();
  require(index >= 0 && index < kMaxDevices, PyExc_RuntimeError, "unexpected CUDA device index");
  if (g_words[index] == nullptr) {
    require(g_prepare != nullptr, PyExc_RuntimeError, "iris_kernel bindings are not set up");
    PyObject* got = PyObject_CallFunction(g_prepare, "i", index);
    if (got == nullptr) throw Raised{};
    void* word = PyLong_AsVoidPtr(got);
    Py_DECREF(got);
    if (word == nullptr) throw Raised{};
    g_words[index] = static_cast<int32_t*>(word);
  }
  return g_words[index];
}

// One C call on the device's current stream, without the interpreter lock (a
// launch may wait for room in the stream's queue).
template <typename F>
void launch(const char* what, c10::Device device, F&& call) {
  int32_t* word = error_word(device);
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != device.index()) guard.set_device(device);
  void* stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
  int status;
  Py_BEGIN_ALLOW_THREADS;
  status = call(word, stream);
  Py_END_ALLOW_THREADS;
  if (status != IRIS_OK) {
    std::string text = std::string(what) + " failed: " + iris_b200_status_string(status);
    if (status == IRIS_ECUDA) text += std::string(" ") + iris_b200_last_cuda_error();
    refuse(PyExc_RuntimeError, text);
  }
}

// (Straight from the CUDA allocator: the dispatcher's way there takes as long again.)
Tensor empty(at::IntArrayRef shape, at::ScalarType type, c10::Device device) {
  return at::Tensor(at::detail::empty_cuda(shape, type, device, std::nullopt));
}
Tensor workspace(size_t bytes, c10::Device device) {
  return empty({static_cast<int64_t>(bytes)}, at::kByte, device);
}

const void* ptr(const Tensor& t) { return t.const_data_ptr(); }
const int32_t* ints(const Tensor& t) { return static_cast<const int32_t*>(t.const_data_ptr()); }
const int32_t* ints(const Tensor* t) { return t == nullptr ? nullptr : ints(*t); }
void* out(const Tensor& t) { return t.data_ptr(); }

// The four tensors of an INT4 cache.
struct Cache {
  int64_t num_pages, page_size, heads, dim;
};
Cache cache_shape(const Tensor& k_data) {
  require(k_data.dim() == 4, PyExc_ValueError, "k_data/v_data must be rank-4 tensors");
  return {k_data.size(0), k_data.size(1), k_data.size(2), 2 * k_data.size(3)};
}
void check_cache(const Cache& c, const Tensor& kd, const Tensor& vd, const Tensor& ks, const Tensor& vs,
                 c10::Device device) {
  const int64_t data[] = {c.num_pages, c.page_size, c.heads, c.dim / 2};
  const int64_t scale[] = {c.num_pages, c.page_size, c.heads, c.dim / 32};
  check("k_data", kd, data, at::kByte, device);
  check("v_data", vd, data, at::kByte, device);
  check("k_scale", ks, scale, at::kHalf, device);
  check("v_scale", vs, scale, at::kHalf, device);
}

// ---------------------------------------------------------------- operators
struct Rows {
  const void* data;
  int64_t stride;
};
// [T, H, D] rows whose tokens may be apart (a slice of a fused projection).
Rows token_rows(const char* name, const Tensor& t, at::IntArrayRef shape, at::ScalarType type, c10::Device device) {
  if (t.sizes() != shape) refuse(PyExc_ValueError, std::string(name) + " must have shape " + shape_text(shape));
  if (t.scalar_type() != type) refuse(PyExc_TypeError, std::string(name) + " must use " + type_name(type));
  if (t.device() != device) refuse(PyExc_ValueError, std::string(name) + " must be on " + device.str());
  if (shape[0] == 0) return {nullptr, 0};
  if (t.stride(2) != 1 || (shape[1] > 1 && t.stride(1) != shape[2]) || (shape[0] > 1 && t.stride(0) % 8 != 0))
    refuse(PyExc_ValueError,
           std::string(name) + " must have contiguous heads and dims, and a token stride that is a multiple of 8");
  if (reinterpret_cast<uintptr_t>(ptr(t)) % 16 != 0)
    refuse(PyExc_ValueError, std::string(name) + " must start on a 16-byte boundary");
  return {ptr(t), shape[0] > 1 ? t.stride(0) : 0};
}

// A given output, contiguous, must not share memory with what the kernel reads
// after it has begun to write, or with what else it writes.
struct Named {
  const char* name;
  const Tensor* tensor;  // NULL: not given
};
void check_apart(const char* name, const Tensor& out, std::initializer_list<Named> others) {
  if (out.numel() == 0) return;
  const char* a = static_cast<const char*>(out.const_data_ptr());
  const char* end = a + out.numel() * out.element_size();
  for (const Named& other : others) {
    if (other.tensor == nullptr || other.tensor->numel() == 0) continue;
    const Tensor& in = *other.tensor;
    int64_t last = 0;
    for (int64_t d = 0; d < in.dim(); ++d) last += (in.size(d) - 1) * in.stride(d);
    const char* b = static_cast<const char*>(in.const_data_ptr());
    if (a < b + (last + 1) * in.element_size() && b < end)
      refuse(PyExc_ValueError, std::string(name) + " must not overlap " + other.name);
  }
}

// (key, value, positions, slot_mapping, cos, sin, k_data, v_data, k_scale, v_scale, query, sections, rotary_dim,
//  interleaved, group_size, page_size, query_out, key_out) -> rotated query or None
PyObject* mrope_append(PyObject* const* a) {
  const Tensor &key = tensor(a[0], "key"), &value = tensor(a[1], "value"), &positions = tensor(a[2], "positions"),
               &slots = tensor(a[3], "slot_mapping"), &cos = tensor(a[4], "cos_cache"), &sin = tensor(a[5], "sin_cache"),
               &kd = tensor(a[6], "k_data"), &vd = tensor(a[7], "v_data"), &ks = tensor(a[8], "k_scale"),
               &vs = tensor(a[9], "v_scale");
  const Tensor *query = optional_tensor(a[10], "query"), *query_out = optional_tensor(a[16], "query_out"),
               *key_out = optional_tensor(a[17], "key_out");
  const c10::Device device = device_of("key", key);
  require(key.dim() == 3 && value.sizes() == key.sizes(), PyExc_ValueError,
          "key and value must have shape [T, Hkv, D]");
  const at::ScalarType type = key.scalar_type();
  const int32_t code = dtype_code("key", type);
  const int64_t tokens = key.size(0), heads = key.size(1), dim = key.size(2), rotary = integer(a[12]);
  const int64_t page_size = integer(a[15]);
  require(dim % 64 == 0 && dim >= 64 && dim <= 512, PyExc_NotImplementedError,
          "fused append requires head_dim divisible by 64, up to 512");
  require(integer(a[14]) == 32, PyExc_NotImplementedError, "fused append supports group_size=32");
  require(rotary % 16 == 0 && rotary >= 16 && rotary <= dim, PyExc_NotImplementedError,
          "fused append requires rotary_dim divisible by 16, up to head_dim");
  require(heads > 0, PyExc_ValueError, "key and value must have at least one head");
  require(page_size > 0 && page_size <= INT32_MAX, PyExc_ValueError, "page_size must be positive");
  int32_t sections[IRIS_MROPE_MAX_AXES];
  PyObject* seq = PySequence_Fast(a[11], "sections must be a sequence");
  if (seq == nullptr) throw Raised{};
  const Py_ssize_t axes = PySequence_Fast_GET_SIZE(seq);
  int64_t sum = 0;
  bool fits = axes >= 1 && axes <= IRIS_MROPE_MAX_AXES, negative = false;
  for (Py_ssize_t i = 0; fits && i < axes; ++i) {
    const long long n = PyLong_AsLongLong(PySequence_Fast_GET_ITEM(seq, i));
    if (n == -1 && PyErr_Occurred()) {
      Py_DECREF(seq);
      throw Raised{};
    }
    negative |= n < 0 || n > 256;
    sections[i] = static_cast<int32_t>(n);
    sum += n;
  }
  Py_DECREF(seq);
  require(fits, PyExc_ValueError, "sections must name 1 to 4 axes");
  if (negative || sum != rotary / 2)
    refuse(PyExc_ValueError,
           "sections must be non-negative and add up to rotary_dim // 2 = " + std::to_string(rotary / 2));
  const Rows k = token_rows("key", key, key.sizes(), type, device);
  const Rows v = token_rows("value", value, key.sizes(), type, device);
  if (positions.dim() != 2 || positions.size(0) != axes || positions.size(1) != tokens)
    refuse(PyExc_ValueError, "positions must have shape [" + std::to_string(axes) + ", T]");
  require(positions.scalar_type() == at::kInt, PyExc_TypeError, "positions must use torch.int32");
  if (positions.device() != device) refuse(PyExc_ValueError, "positions must be on " + device.str());
  require(tokens <= 1 || positions.stride(1) == 1, PyExc_ValueError, "positions of one axis must be contiguous");
  check("slot_mapping", slots, {tokens}, at::kInt, device);
  require(cos.dim() == 2, PyExc_ValueError, "cos_cache must have shape [max_position, rotary_dim // 2]");
  check("cos_cache", cos, {cos.size(0), rotary / 2}, type, device);
  check("sin_cache", sin, {cos.size(0), rotary / 2}, type, device);
  require(kd.dim() == 4, PyExc_ValueError, "k_data/v_data must be rank-4 tensors");
  const Cache cache = {kd.size(0), page_size, heads, dim};
  check_cache(cache, kd, vd, ks, vs, device);
  Rows q = {nullptr, 0};
  int64_t q_heads = 0;
  Tensor rotated;
  if (query != nullptr) {
    require(query->dim() == 3 && query->size(1) > 0, PyExc_ValueError, "query must have shape [T, Hq, D]");
    q_heads = query->size(1);
    const int64_t shape[] = {tokens, q_heads, dim};
    q = token_rows("query", *query, shape, type, device);
    if (query_out == nullptr) {
      rotated = empty(shape, type, device);
    } else {
      check("query_out", *query_out, shape, type, device);
      check_apart("query_out", *query_out,
                  {{"query", query}, {"key", &key}, {"value", &value}, {"positions", &positions},
                   {"slot_mapping", &slots}, {"cos_cache", &cos}, {"sin_cache", &sin}, {"k_data", &kd}, {"v_data", &vd},
                   {"k_scale", &ks}, {"v_scale", &vs}});
      rotated = *query_out;
    }
  } else {
    require(query_out == nullptr, PyExc_ValueError, "query_out needs a query");
  }
  if (key_out != nullptr) {
    check("key_out", *key_out, key.sizes(), type, device);
    check_apart("key_out", *key_out,
                {{"query_out", query_out}, {"query", query}, {"key", &key}, {"value", &value}, {"positions", &positions},
                 {"slot_mapping", &slots}, {"cos_cache", &cos}, {"sin_cache", &sin}, {"k_data", &kd}, {"v_data", &vd},
                 {"k_scale", &ks}, {"v_scale", &vs}});
  }
  require(heads <= INT32_MAX && q_heads <= INT32_MAX, PyExc_ValueError, "too many heads");
  if (tokens > 0) {
    Tensor ws;
    const size_t bytes =
        iris_b200_mrope_append_workspace_bytes(tokens, cache.num_pages, static_cast<int32_t>(page_size));
    if (bytes > 0) ws = workspace(bytes, device);
    const int interleaved = PyObject_IsTrue(a[13]);
    if (interleaved < 0) throw Raised{};
    launch("iris_b200_mrope_int4_paged_append", device, [&](int32_t* word, void* stream) {
      return iris_b200_mrope_int4_paged_append(
          k.data, k.stride, v.data, v.stride, q.data, q.stride, ints(positions), positions.stride(0), sections,
          static_cast<int32_t>(axes), interleaved, ints(slots), ptr(cos), ptr(sin), out(kd), out(vd), out(ks), out(vs),
          rotated.defined() ? out(rotated) : nullptr, key_out != nullptr ? out(*key_out) : nullptr, tokens,
          static_cast<int32_t>(q_heads), static_cast<int32_t>(heads), static_cast<int32_t>(dim),
          static_cast<int32_t>(rotary), cos.size(0), cache.num_pages, static_cast<int32_t>(page_size), code,
          ws.defined() ? out(ws) : nullptr, bytes, word, stream);
    });
  }
  if (query == nullptr) Py_RETURN_NONE;
  if (query_out != nullptr) {
    Py_INCREF(a[16]);
    return a[16];
  }
  return THPVariable_Wrap(std::move(rotated));
}

PyObject* pair(PyObject* x, PyObject* y) {
  if (x == nullptr || y == nullptr) {
    Py_XDECREF(x);
    Py_XDECREF(y);
    return nullptr;
  }
  PyObject* t = PyTuple_New(2);
  if (t == nullptr) {
    Py_DECREF(x);
    Py_DECREF(y);
    return nullptr;
  }
  PyTuple_SET_ITEM(t, 0, x);
  PyTuple_SET_ITEM(t, 1, y);
  return t;
}
// A given output as the object it came as, or a new one.
PyObject* given_or(PyObject* given, Tensor& made) {
  if (given != Py_None) {
    Py_INCREF(given);
    return given;
  }
  return THPVariable_Wrap(std::move(made));
}

// (k_data, v_data, k_scale, v_scale, block_table, cu_seqlens, key, value, num_tokens, first_token, is_bf16 (None:
//  neither), page_size, group_size) -> (key, value)
PyObject* gather(PyObject* const* a) {
  const Tensor &kd = tensor(a[0], "k_data"), &vd = tensor(a[1], "v_data"), &ks = tensor(a[2], "k_scale"),
               &vs = tensor(a[3], "v_scale"), &bt = tensor(a[4], "block_table"), &cu = tensor(a[5], "cu_seqlens");
  const Tensor *key = optional_tensor(a[6], "key"), *value = optional_tensor(a[7], "value"),
               *first = optional_tensor(a[9], "first_token");
  const c10::Device device = device_of("k_data", kd);
  require(integer(a[12]) == 32, PyExc_NotImplementedError, "gather supports group_size=32");
  const Cache c = cache_shape(kd);
  const int64_t page_size = integer(a[11]), tokens = integer(a[8]);
  require(c.page_size == page_size && page_size > 0 && c.heads > 0 && page_size <= INT32_MAX, PyExc_ValueError,
          "packed cache shape does not match page_size");
  require(c.dim % 32 == 0 && c.dim >= 32 && c.dim <= 512, PyExc_NotImplementedError,
          "gather requires head_dim divisible by 32, up to 512");
  check_cache(c, kd, vd, ks, vs, device);
  require(bt.dim() == 2, PyExc_ValueError, "block_table must have shape [B, max_pages_per_sequence]");
  const int64_t batch = bt.size(0);
  const Table table = block_table(bt, batch, device);
  check("cu_seqlens", cu, {batch + 1}, at::kInt, device);
  if (first != nullptr) check("first_token", *first, {batch}, at::kInt, device);
  require(tokens >= 0, PyExc_ValueError, "num_tokens must not be negative");
  at::ScalarType type;
  if (key != nullptr) {
    type = key->scalar_type();
  } else {
    require(a[10] != Py_None, PyExc_TypeError, "dtype must use FP16(torch.float16) or BF16(torch.bfloat16)");
    type = PyObject_IsTrue(a[10]) == 1 ? at::kBFloat16 : at::kHalf;
  }
  const int32_t code = dtype_code("key", type);
  const int64_t shape[] = {tokens, c.heads, c.dim};
  Tensor k, v;
  if (key == nullptr) {
    k = empty(shape, type, device);
  } else {
    check("key", *key, shape, type, device);
    check_apart("key", *key, {{"value", value}, {"k_data", &kd}, {"v_data", &vd}, {"k_scale", &ks}, {"v_scale", &vs},
                              {"block_table", &bt}, {"cu_seqlens", &cu}, {"first_token", first}});
    k = *key;
  }
  if (value == nullptr) {
    v = empty(shape, type, device);
  } else {
    check("value", *value, shape, type, device);
    check_apart("value", *value, {{"k_data", &kd}, {"v_data", &vd}, {"k_scale", &ks}, {"v_scale", &vs},
                                  {"block_table", &bt}, {"cu_seqlens", &cu}, {"first_token", first}});
    v = *value;
  }
  if (tokens > 0) {
    require(batch > 0, PyExc_ValueError, "num_tokens must be 0 without sequences");
    require(c.num_pages > 0, PyExc_IndexError, "block_table contains an invalid physical page id");
    require(batch <= INT32_MAX && c.heads <= INT32_MAX, PyExc_ValueError, "too many sequences or heads");
    launch("iris_b200_int4_paged_gather", device, [&](int32_t* word, void* stream) {
      return iris_b200_int4_paged_gather(ptr(kd), ptr(vd), ptr(ks), ptr(vs), table.data, table.stride, ints(cu),
                                         ints(first), out(k), out(v), tokens, static_cast<int32_t>(batch),
                                         static_cast<int32_t>(c.heads), static_cast<int32_t>(c.dim), c.num_pages,
                                         static_cast<int32_t>(page_size), table.width, code, word, stream);
    });
  }
  PyObject* first_out = given_or(a[6], k);
  return pair(first_out, given_or(a[7], v));
}

void sparse_shape(int64_t page_size, int64_t dim) {
  require(page_size == 16, PyExc_NotImplementedError, "sparse decode currently supports page_size=16");
  require(dim == 64 || dim == 128, PyExc_NotImplementedError, "sparse decode currently supports head_dim in {64, 128}");
}
int32_t sparse_query(const Tensor& query, int64_t heads) {
  require(query.dim() == 3, PyExc_ValueError, "query must have shape [B, Hq, D]");
  const int32_t code = dtype_code("query", query.scalar_type());
  require(query.is_contiguous(), PyExc_ValueError, "query must be contiguous");
  const int64_t hq = query.size(1);
  require(heads > 0 && hq > 0 && hq % heads == 0, PyExc_ValueError,
          "num_query_heads must be divisible by num_kv_heads");
  require(hq / heads <= 16, PyExc_NotImplementedError, "sparse decode supports at most 16 query heads per KV head");
  require(reinterpret_cast<uintptr_t>(ptr(query)) % 16 == 0, PyExc_ValueError,
          "query must start on a 16-byte boundary");
  require(query.size(0) <= INT32_MAX && hq <= INT32_MAX, PyExc_ValueError, "too many sequences or heads");
  return code;
}

// (k_data, k_scale, block_table, seq_lens, bounds, bounds_step, first_token, values, page_size, group_size) -> None
PyObject* page_bounds(PyObject* const* a) {
  const Tensor &kd = tensor(a[0], "k_data"), &ks = tensor(a[1], "k_scale"), &bt = tensor(a[2], "block_table"),
               &lens = tensor(a[3], "seq_lens"), &bounds = tensor(a[4], "bounds"), &step = tensor(a[5], "bounds_step");
  const Tensor *first = optional_tensor(a[6], "first_token"), *values = optional_tensor(a[7], "values");
  const c10::Device device = device_of("k_data", kd);
  require(integer(a[9]) == 32, PyExc_NotImplementedError, "sparse decode currently supports group_size=32");
  const Cache c = cache_shape(kd);
  const int64_t page_size = integer(a[8]);
  sparse_shape(page_size, c.dim);
  require(c.page_size == page_size && c.heads > 0, PyExc_ValueError, "packed cache shape does not match page_size");
  check("k_data", kd, kd.sizes(), at::kByte, device);
  check("k_scale", ks, {c.num_pages, page_size, c.heads, c.dim / 32}, at::kHalf, device);
  check("bounds", bounds, {c.num_pages, c.heads, 2, c.dim}, at::kChar, device);
  check("bounds_step", step, {c.num_pages, c.heads}, at::kFloat, device);
  if (values != nullptr) check("values", *values, {c.num_pages, c.heads, 2, c.dim}, at::kHalf, device);
  require(bt.dim() == 2, PyExc_ValueError, "block_table must have shape [B, max_pages_per_sequence]");
  const int64_t batch = bt.size(0);
  const Table table = block_table(bt, batch, device);
  check("seq_lens", lens, {batch}, at::kInt, device);
  if (first != nullptr) check("first_token", *first, {batch}, at::kInt, device);
  if (batch > 0) {
    require(c.num_pages > 0, PyExc_IndexError, "block_table contains an invalid physical page id");
    require(batch <= INT32_MAX && c.heads <= INT32_MAX, PyExc_ValueError, "too many sequences or heads");
    launch("iris_b200_int4_page_bounds", device, [&](int32_t* word, void* stream) {
      return iris_b200_int4_page_bounds(ptr(kd), ptr(ks), table.data, table.stride, ints(lens), ints(first),
                                        out(bounds), static_cast<float*>(out(step)),
                                        values != nullptr ? out(*values) : nullptr, static_cast<int32_t>(batch),
                                        static_cast<int32_t>(c.heads), static_cast<int32_t>(c.dim), c.num_pages,
                                        static_cast<int32_t>(page_size), table.width, word, stream);
    });
  }
  Py_RETURN_NONE;
}

// (query, bounds, bounds_step, block_table, seq_lens, page_list, page_count, max_pages, sink_pages, recent_pages,
//  page_size) -> (page_list, page_count)
PyObject* page_select(PyObject* const* a) {
  const Tensor &query = tensor(a[0], "query"), &bounds = tensor(a[1], "bounds"), &step = tensor(a[2], "bounds_step"),
               &bt = tensor(a[3], "block_table"), &lens = tensor(a[4], "seq_lens");
  const Tensor *list = optional_tensor(a[5], "page_list"), *count = optional_tensor(a[6], "page_count");
  const c10::Device device = device_of("query", query);
  require(bounds.dim() == 4 && bounds.size(2) == 2, PyExc_ValueError, "bounds must have shape [pages, Hkv, 2, D]");
  const int64_t pages = bounds.size(0), heads = bounds.size(1), dim = bounds.size(3);
  const int32_t code = sparse_query(query, heads);
  const int64_t page_size = integer(a[10]);
  sparse_shape(page_size, dim);
  const int64_t batch = query.size(0), hq = query.size(1);
  require(query.size(2) == dim, PyExc_ValueError, "bounds do not match the query's head_dim");
  const int64_t keep = integer(a[7]), sink = integer(a[8]), recent = integer(a[9]);
  require(keep > 0 && keep <= INT32_MAX && sink >= 0 && recent >= 0 && sink <= keep && recent <= keep - sink,
          PyExc_ValueError, "max_pages must be positive and hold sink_pages and recent_pages");
  check("bounds", bounds, bounds.sizes(), at::kChar, device);
  check("bounds_step", step, {pages, heads}, at::kFloat, device);
  const Table table = block_table(bt, batch, device);
  check("seq_lens", lens, {batch}, at::kInt, device);
  const int64_t shape[] = {batch, heads, keep};
  Tensor l, n;
  if (list == nullptr) {
    l = empty(shape, at::kInt, device);
  } else {
    check("page_list", *list, shape, at::kInt, device);
    check_apart("page_list", *list, {{"page_count", count}, {"query", &query}, {"bounds", &bounds}, {"bounds_step", &step},
                                     {"block_table", &bt}, {"seq_lens", &lens}});
    l = *list;
  }
  if (count == nullptr) {
    n = empty({batch, heads}, at::kInt, device);
  } else {
    check("page_count", *count, {batch, heads}, at::kInt, device);
    check_apart("page_count", *count, {{"query", &query}, {"bounds", &bounds}, {"bounds_step", &step},
                                       {"block_table", &bt}, {"seq_lens", &lens}});
    n = *count;
  }
  if (batch > 0) {
    require(pages > 0, PyExc_IndexError, "block_table contains an invalid physical page id");
    const size_t bytes = iris_b200_page_select_workspace_bytes(static_cast<int32_t>(batch),
                                                               static_cast<int32_t>(heads), table.width);
    const Tensor ws = workspace(bytes, device);
    launch("iris_b200_page_select", device, [&](int32_t* word, void* stream) {
      return iris_b200_page_select(ptr(query), ptr(bounds), static_cast<const float*>(ptr(step)), table.data,
                                   table.stride, ints(lens), static_cast<int32_t*>(out(l)),
                                   static_cast<int32_t*>(out(n)), static_cast<int32_t>(batch),
                                   static_cast<int32_t>(hq), static_cast<int32_t>(heads), static_cast<int32_t>(dim),
                                   pages, static_cast<int32_t>(page_size), table.width, static_cast<int32_t>(keep),
                                   static_cast<int32_t>(sink), static_cast<int32_t>(recent), code, out(ws), bytes, word,
                                   stream);
    });
  }
  PyObject* first_out = given_or(a[5], l);
  return pair(first_out, given_or(a[6], n));
}

// (query, k_data, v_data, k_scale, v_scale, block_table, seq_lens, page_list, page_count, output, page_size,
//  group_size, softmax_scale, return_lse) -> output or (output, lse)
PyObject* sparse_decode(PyObject* const* a) {
  const Tensor &query = tensor(a[0], "query"), &kd = tensor(a[1], "k_data"), &vd = tensor(a[2], "v_data"),
               &ks = tensor(a[3], "k_scale"), &vs = tensor(a[4], "v_scale"), &bt = tensor(a[5], "block_table"),
               &lens = tensor(a[6], "seq_lens"), &list = tensor(a[7], "page_list"), &count = tensor(a[8], "page_count");
  const Tensor* output = optional_tensor(a[9], "output");
  const c10::Device device = device_of("query", query);
  require(integer(a[11]) == 32, PyExc_NotImplementedError, "sparse decode currently supports group_size=32");
  const Cache c = cache_shape(kd);
  const int32_t code = sparse_query(query, c.heads);
  const int64_t page_size = integer(a[10]);
  sparse_shape(page_size, c.dim);
  const int64_t batch = query.size(0), hq = query.size(1);
  require(c.page_size == page_size && query.size(2) == c.dim, PyExc_ValueError,
          "packed cache shape does not match query/page_size");
  check_cache(c, kd, vd, ks, vs, device);
  const Table table = block_table(bt, batch, device);
  check("seq_lens", lens, {batch}, at::kInt, device);
  require(list.dim() == 3 && list.size(2) > 0 && list.size(2) <= INT32_MAX, PyExc_ValueError,
          "page_list must have shape [B, Hkv, max_pages], max_pages >= 1");
  const int32_t keep = static_cast<int32_t>(list.size(2));
  check("page_list", list, {batch, c.heads, keep}, at::kInt, device);
  check("page_count", count, {batch, c.heads}, at::kInt, device);
  Tensor o, lse;
  if (output == nullptr) {
    o = empty(query.sizes(), query.scalar_type(), device);
  } else {
    check("output", *output, query.sizes(), query.scalar_type(), device);
    // (in the query's own place it is: a row is read before it is written)
    const bool in_place = output->const_data_ptr() == query.const_data_ptr();
    check_apart("output", *output, {{"query", in_place ? nullptr : &query}, {"k_data", &kd}, {"v_data", &vd},
                                    {"k_scale", &ks}, {"v_scale", &vs}, {"block_table", &bt}, {"seq_lens", &lens},
                                    {"page_list", &list}, {"page_count", &count}});
    o = *output;
  }
  const int with_lse = PyObject_IsTrue(a[13]);
  if (with_lse < 0) throw Raised{};
  if (with_lse) lse = empty({batch, hq}, at::kFloat, device);
  if (batch > 0) {
    require(c.num_pages > 0, PyExc_IndexError, "block_table contains an invalid physical page id");
    double factor = a[12] == Py_None ? 0.0 : PyFloat_AsDouble(a[12]);
    if (factor == -1.0 && PyErr_Occurred()) throw Raised{};
    if (factor == 0.0) factor = c.dim == 64 ? 0.125 : 0.08838834764831845;  // dim ** -0.5
    const size_t bytes = iris_b200_sparse_decode_workspace_bytes(
        static_cast<int32_t>(batch), static_cast<int32_t>(hq), static_cast<int32_t>(c.heads),
        static_cast<int32_t>(c.dim), keep, device.index());
    const Tensor ws = workspace(bytes, device);
    launch("iris_b200_int4_sparse_paged_decode", device, [&](int32_t* word, void* stream) {
      return iris_b200_int4_sparse_paged_decode(
          ptr(query), ptr(kd), ptr(vd), ptr(ks), ptr(vs), table.data, table.stride, ints(lens), ints(list),
          ints(count), out(o), with_lse ? static_cast<float*>(out(lse)) : nullptr, static_cast<int32_t>(batch),
          static_cast<int32_t>(hq), static_cast<int32_t>(c.heads), static_cast<int32_t>(c.dim), c.num_pages,
          static_cast<int32_t>(page_size), table.width, keep, static_cast<float>(factor), code, out(ws), bytes, word,
          stream);
    });
  }
  PyObject* first_out = given_or(a[9], o);
  if (!with_lse) return first_out;
  return pair(first_out, THPVariable_Wrap(std::move(lse)));
}

// ------------------------------------------------- attention of new tokens
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return v;
}

// What attention of new tokens and its weights share: the query's rows, the sequences, what a row sees.
struct NewTokens {
  Rows query;
  Table table;
  int64_t tokens, hq, batch;
  int32_t code, window;
  float scale, cap;
  const Tensor *cu, *slopes, *prefix, *first;
};
NewTokens new_tokens(const Tensor& query, const Cache& c, const Tensor& bt, const Tensor& lens, PyObject* cu_arg,
                     PyObject* page_arg, PyObject* group_arg, PyObject* scale_arg, PyObject* cap_arg,
                     PyObject* slopes_arg, PyObject* window_arg, PyObject* prefix_arg, PyObject* first_arg,
                     c10::Device device) {
  NewTokens n;
  require(integer(group_arg) == 32, PyExc_NotImplementedError, "varlen attention currently supports group_size=32");
  require(integer(page_arg) == 16, PyExc_NotImplementedError, "varlen attention currently supports page_size=16");
  require(c.dim == 64 || c.dim == 128, PyExc_NotImplementedError,
          "varlen attention currently supports head_dim in {64, 128}");
  require(query.dim() == 3, PyExc_ValueError, "query must have shape [T, Hq, D]");
  n.code = dtype_code("query", query.scalar_type());
  n.tokens = query.size(0);
  n.hq = query.size(1);
  require(c.page_size == 16 && query.size(2) == c.dim, PyExc_ValueError,
          "packed cache shape does not match query/page_size");
  require(c.heads > 0 && n.hq > 0 && n.hq % c.heads == 0, PyExc_ValueError,
          "num_query_heads must be divisible by num_kv_heads");
  n.query = token_rows("query", query, query.sizes(), query.scalar_type(), device);
  if (n.tokens == 1) n.query.stride = n.hq * c.dim;
  require(bt.dim() == 2, PyExc_ValueError, "block_table must have shape [B, max_pages_per_sequence]");
  n.batch = bt.size(0);
  n.table = block_table(bt, n.batch, device);
  check("seq_lens", lens, {n.batch}, at::kInt, device);
  n.cu = optional_tensor(cu_arg, "cu_seqlens");
  if (n.cu != nullptr)
    check("cu_seqlens", *n.cu, {n.batch + 1}, at::kInt, device);
  else
    require(n.tokens == n.batch, PyExc_ValueError, "query needs one row a sequence, or cu_seqlens");
  n.slopes = optional_tensor(slopes_arg, "slopes");
  if (n.slopes != nullptr) check("slopes", *n.slopes, {n.hq}, at::kFloat, device);
  n.prefix = optional_tensor(prefix_arg, "prefix_lens");
  if (n.prefix != nullptr) check("prefix_lens", *n.prefix, {n.batch}, at::kInt, device);
  n.first = optional_tensor(first_arg, "first_visible");
  if (n.first != nullptr) check("first_visible", *n.first, {n.tokens}, at::kInt, device);
  n.window = integer32(window_arg, "window");
  require(n.window >= 0, PyExc_ValueError, "window must not be negative");
  double scale = scale_arg == Py_None ? 0.0 : number(scale_arg);
  if (scale == 0.0) scale = c.dim == 64 ? 0.125 : 0.08838834764831845;  // dim ** -0.5
  n.scale = static_cast<float>(scale);
  require(n.scale > 0.0f && n.scale <= 3.0e38f, PyExc_ValueError, "softmax_scale must be positive and finite");
  n.cap = static_cast<float>(number(cap_arg));
  require(n.cap >= 0.0f && n.cap <= 1.0e20f, PyExc_ValueError, "logit_cap must lie in [0, 1e20]");
  require(n.tokens <= INT32_MAX && n.hq <= INT32_MAX && n.batch <= INT32_MAX && c.heads <= INT32_MAX, PyExc_ValueError,
          "too many tokens, heads or sequences");
  if (n.tokens > 0) {
    require(n.batch > 0, PyExc_ValueError, "query must be empty without sequences");
    require(c.num_pages > 0, PyExc_IndexError, "block_table contains an invalid physical page id");
  }
  return n;
}
const float* floats(const Tensor* t) { return t == nullptr ? nullptr : static_cast<const float*>(t->const_data_ptr()); }

// (query, k_data, v_data, k_scale, v_scale, block_table, seq_lens, cu_seqlens, output, page_size, group_size,
//  softmax_scale, logit_cap, slopes, window, prefix_lens, first_visible, return_lse) -> output or (output, lse)
PyObject* varlen_attention(PyObject* const* a) {
  const Tensor &query = tensor(a[0], "query"), &kd = tensor(a[1], "k_data"), &vd = tensor(a[2], "v_data"),
               &ks = tensor(a[3], "k_scale"), &vs = tensor(a[4], "v_scale"), &bt = tensor(a[5], "block_table"),
               &lens = tensor(a[6], "seq_lens");
  const Tensor* output = optional_tensor(a[8], "output");
  const c10::Device device = device_of("query", query);
  const Cache c = cache_shape(kd);
  const NewTokens n = new_tokens(query, c, bt, lens, a[7], a[9], a[10], a[11], a[12], a[13], a[14], a[15], a[16], device);
  check_cache(c, kd, vd, ks, vs, device);
  Tensor o, lse;
  if (output == nullptr) {
    o = empty(query.sizes(), query.scalar_type(), device);
  } else {
    check("output", *output, query.sizes(), query.scalar_type(), device);
    // (in a dense query's own place it is: a row is read before it is written)
    const bool in_place = output->const_data_ptr() == query.const_data_ptr() && query.is_contiguous();
    check_apart("output", *output,
                {{"query", in_place ? nullptr : &query}, {"k_data", &kd}, {"v_data", &vd}, {"k_scale", &ks},
                 {"v_scale", &vs}, {"block_table", &bt}, {"seq_lens", &lens}, {"cu_seqlens", n.cu}, {"slopes", n.slopes},
                 {"prefix_lens", n.prefix}, {"first_visible", n.first}});
    require(reinterpret_cast<uintptr_t>(ptr(*output)) % 16 == 0, PyExc_ValueError,
            "output must start on a 16-byte boundary");
    o = *output;
  }
  const int with_lse = PyObject_IsTrue(a[17]);
  if (with_lse < 0) throw Raised{};
  if (with_lse) lse = empty({n.tokens, n.hq}, at::kFloat, device);
  if (n.tokens > 0) {
    const size_t bytes = iris_b200_varlen_attention_workspace_bytes(
        n.tokens, static_cast<int32_t>(n.batch), static_cast<int32_t>(n.hq), static_cast<int32_t>(c.heads),
        static_cast<int32_t>(c.dim), n.table.width, n.window, n.prefix != nullptr, n.cu != nullptr, device.index());
    Tensor ws;
    if (bytes > 0) ws = workspace(bytes, device);
    launch("iris_b200_int4_paged_varlen_attention", device, [&](int32_t* word, void* stream) {
      return iris_b200_int4_paged_varlen_attention(
          n.query.data, n.query.stride, ptr(kd), ptr(vd), ptr(ks), ptr(vs), n.table.data, n.table.stride, ints(lens),
          ints(n.cu), floats(n.slopes), ints(n.prefix), ints(n.first), out(o),
          with_lse ? static_cast<float*>(out(lse)) : nullptr, n.tokens, static_cast<int32_t>(n.batch),
          static_cast<int32_t>(n.hq), static_cast<int32_t>(c.heads), static_cast<int32_t>(c.dim), c.num_pages, 16,
          n.table.width, n.window, n.cap, n.scale, n.code, ws.defined() ? out(ws) : nullptr, bytes, word, stream);
    });
  }
  PyObject* first_out = given_or(a[8], o);
  if (!with_lse) return first_out;
  return pair(first_out, THPVariable_Wrap(std::move(lse)));
}

// (query, lse, k_data, k_scale, block_table, seq_lens, mass, cu_seqlens, first_token, decay, page_size, group_size,
//  softmax_scale, logit_cap, slopes, window, prefix_lens, first_visible) -> None
PyObject* attention_mass(PyObject* const* a) {
  const Tensor &query = tensor(a[0], "query"), &lse = tensor(a[1], "lse"), &kd = tensor(a[2], "k_data"),
               &ks = tensor(a[3], "k_scale"), &bt = tensor(a[4], "block_table"), &lens = tensor(a[5], "seq_lens"),
               &mass = tensor(a[6], "mass");
  const Tensor* first_token = optional_tensor(a[8], "first_token");
  const c10::Device device = device_of("query", query);
  const Cache c = cache_shape(kd);
  const NewTokens n =
      new_tokens(query, c, bt, lens, a[7], a[10], a[11], a[12], a[13], a[14], a[15], a[16], a[17], device);
  check("k_data", kd, {c.num_pages, 16, c.heads, c.dim / 2}, at::kByte, device);
  check("k_scale", ks, {c.num_pages, 16, c.heads, c.dim / 32}, at::kHalf, device);
  check("lse", lse, {n.tokens, n.hq}, at::kFloat, device);
  check("mass", mass, {c.num_pages, c.heads, 16}, at::kFloat, device);
  if (first_token != nullptr) check("first_token", *first_token, {n.batch}, at::kInt, device);
  check_apart("mass", mass, {{"query", &query}, {"lse", &lse}, {"k_data", &kd}, {"k_scale", &ks}, {"block_table", &bt},
                             {"seq_lens", &lens}, {"cu_seqlens", n.cu}, {"first_token", first_token},
                             {"slopes", n.slopes}, {"prefix_lens", n.prefix}, {"first_visible", n.first}});
  const double decay = number(a[9]);
  require(decay >= 0.0 && decay <= 1.0, PyExc_ValueError, "decay must lie in [0, 1]");
  if (n.batch > 0) {
    require(c.num_pages > 0, PyExc_IndexError, "block_table contains an invalid physical page id");
    launch("iris_b200_int4_paged_attention_mass", device, [&](int32_t* word, void* stream) {
      return iris_b200_int4_paged_attention_mass(
          n.query.data, n.query.stride, floats(&lse), ptr(kd), ptr(ks), n.table.data, n.table.stride, ints(lens),
          ints(n.cu), floats(n.slopes), ints(n.prefix), ints(n.first), ints(first_token), static_cast<float*>(out(mass)),
          n.tokens, static_cast<int32_t>(n.batch), static_cast<int32_t>(n.hq), static_cast<int32_t>(c.heads),
          static_cast<int32_t>(c.dim), c.num_pages, 16, n.table.width, n.window, n.cap, n.scale,
          static_cast<float>(decay), n.code, word, stream);
    });
  }
  Py_RETURN_NONE;
}

// (k_data, v_data, k_scale, v_scale, mass, block_table, seq_lens, new_lens, kept, budget, sink_tokens, recent_tokens,
//  page_size, group_size, return_kept) -> new_lens or (new_lens, kept)
PyObject* evict(PyObject* const* a) {
  const Tensor &kd = tensor(a[0], "k_data"), &vd = tensor(a[1], "v_data"), &ks = tensor(a[2], "k_scale"),
               &vs = tensor(a[3], "v_scale"), &mass = tensor(a[4], "mass"), &bt = tensor(a[5], "block_table"),
               &lens = tensor(a[6], "seq_lens");
  const Tensor *new_lens = optional_tensor(a[7], "new_lens"), *kept = optional_tensor(a[8], "kept");
  const c10::Device device = device_of("k_data", kd);
  require(integer(a[13]) == 32, PyExc_NotImplementedError, "eviction currently supports group_size=32");
  require(integer(a[12]) == 16, PyExc_NotImplementedError, "eviction currently supports page_size=16");
  const Cache c = cache_shape(kd);
  require(c.dim == 64 || c.dim == 128, PyExc_NotImplementedError, "eviction currently supports head_dim in {64, 128}");
  require(c.page_size == 16 && c.heads > 0 && c.heads <= INT32_MAX, PyExc_ValueError,
          "packed cache shape does not match page_size");
  check_cache(c, kd, vd, ks, vs, device);
  check("mass", mass, {c.num_pages, c.heads, 16}, at::kFloat, device);
  require(reinterpret_cast<uintptr_t>(ptr(mass)) % 16 == 0, PyExc_ValueError, "mass must start on a 16-byte boundary");
  require(bt.dim() == 2, PyExc_ValueError, "block_table must have shape [B, max_pages_per_sequence]");
  const int64_t batch = bt.size(0);
  const Table table = block_table(bt, batch, device);
  check("seq_lens", lens, {batch}, at::kInt, device);
  const int32_t budget = integer32(a[9], "budget"), sink = integer32(a[10], "sink_tokens"),
                recent = integer32(a[11], "recent_tokens");
  require(budget > 0 && sink >= 0 && recent >= 0 && sink <= budget && recent <= budget - sink, PyExc_ValueError,
          "budget must be positive and hold sink_tokens and recent_tokens");
  const int with_kept = PyObject_IsTrue(a[14]);
  if (with_kept < 0) throw Raised{};
  const std::initializer_list<Named> data = {{"k_data", &kd}, {"v_data", &vd}, {"k_scale", &ks}, {"v_scale", &vs},
                                             {"block_table", &bt}, {"seq_lens", &lens}};
  check_apart("mass", mass, data);
  Tensor l, k;
  if (new_lens == nullptr) {
    l = empty({batch}, at::kInt, device);
  } else {
    check("new_lens", *new_lens, {batch}, at::kInt, device);
    check_apart("new_lens", *new_lens, data);
    check_apart("new_lens", *new_lens, {{"mass", &mass}, {"kept", kept}});
    l = *new_lens;
  }
  if (kept != nullptr) {
    check("kept", *kept, {batch, c.heads, budget}, at::kInt, device);
    check_apart("kept", *kept, data);
    check_apart("kept", *kept, {{"mass", &mass}});
    k = *kept;
  } else if (with_kept) {
    k = empty({batch, c.heads, budget}, at::kInt, device);
  }
  if (batch > 0) {
    require(c.num_pages > 0, PyExc_IndexError, "block_table contains an invalid physical page id");
    require(batch <= INT32_MAX, PyExc_ValueError, "too many sequences");
    const size_t bytes = budget >= static_cast<int64_t>(table.width) * 16
                             ? 0
                             : iris_b200_evict_workspace_bytes(static_cast<int32_t>(batch), static_cast<int32_t>(c.heads),
                                                               budget, recent);
    Tensor ws;
    if (bytes > 0) ws = workspace(bytes, device);
    launch("iris_b200_int4_paged_evict", device, [&](int32_t* word, void* stream) {
      return iris_b200_int4_paged_evict(out(kd), out(vd), out(ks), out(vs), static_cast<float*>(out(mass)), table.data,
                                        table.stride, ints(lens), static_cast<int32_t*>(out(l)),
                                        k.defined() ? static_cast<int32_t*>(out(k)) : nullptr,
                                        static_cast<int32_t>(batch), static_cast<int32_t>(c.heads),
                                        static_cast<int32_t>(c.dim), c.num_pages, 16, table.width, budget, sink, recent,
                                        ws.defined() ? out(ws) : nullptr, bytes, word, stream);
    });
  }
  PyObject* first_out = given_or(a[7], l);
  if (!k.defined()) return first_out;
  return pair(first_out, given_or(a[8], k));
}

// ------------------------------------------------------------------- module
template <PyObject* (*kFn)(PyObject* const*), int kArgs>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kArgs) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    return kFn(args);
  } catch (const Refusal& r) {
    PyErr_SetString(r.type, r.text.c_str());
  } catch (const Raised&) {
  } catch (const std::exception& e) {  // out of memory, among others, as torch words it
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "iris_kernel: unexpected C++ exception");
  }
  return nullptr;
}

PyObject* set_up(PyObject*, PyObject* fn) {
  Py_INCREF(fn);
  Py_XSETREF(g_prepare, fn);
  Py_RETURN_NONE;
}

template <PyObject* (*kFn)(PyObject* const*), int kArgs>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<kFn, kArgs>)), METH_FASTCALL, nullptr};
}

PyMethodDef g_methods[] = {
    {"set_up", set_up, METH_O, nullptr},
    method<mrope_append, 18>("mrope_append"),
    method<gather, 13>("gather"),
    method<page_bounds, 10>("page_bounds"),
    method<page_select, 11>("page_select"),
    method<sparse_decode, 14>("sparse_decode"),
    method<varlen_attention, 18>("varlen_attention"),
    method<attention_mass, 18>("attention_mass"),
    method<evict, 15>("evict"),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_ops", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops() { return PyModule_Create(&g_module); }
