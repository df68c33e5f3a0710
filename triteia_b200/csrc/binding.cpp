// Python binding of the operators between a layer's projections (norm with rotation, paged cache, paged attention).
// Their smallest calls run for a few microseconds on the device; checking the tensors and marshalling some thirty
// arguments from Python took 10 to 15 (one decode token through paged_attention: 15.8 us a call, 4 of them on the GPU).
// Here the same checks and the call of the C ABI take about 2.  Everything else of the library is bound with ctypes.
//
// Every check comes before the one for a CUDA device, so that a refusal does not need one.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <math.h>
#include <stdarg.h>
#include <stdio.h>

#include "../../include/triteia_b200.h"

namespace {

struct Refused {};      // a Python error is set

[[noreturn]] __attribute__((format(printf, 1, 2))) void refuse(const char* fmt, ...) {
  char text[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(text, sizeof text, fmt, ap);
  va_end(ap);
  PyErr_SetString(PyExc_RuntimeError, text);
  throw Refused();
}

void check_status(int status, const char* what, const char* shapes) {
  if (status == TRB_OK) return;
  if (status == TRB_ERR_PROB_SHAPE || status == TRB_ERR_KERN_SHAPE) refuse("No suitable kernel. %s", shapes);
  refuse("%s: %s (status %d)", what, trb_status_string(status), status);
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s must be a tensor", name);
    throw Refused();
  }
  return THPVariable_Unpack(o);
}

// nullptr for None.
const at::Tensor* maybe(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }

long long integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused();
  return v;
}

double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refused();
  return v;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Refused();
  return v != 0;
}

int tag_of(at::ScalarType t) {
  if (t == at::kHalf) return TRB_F16;
  if (t == at::kBFloat16) return TRB_BF16;
  refuse("No suitable kernel. dtype=%s", c10::toString(t));
}

int small(int64_t v, const char* name) {
  if (v > 0x7fffffff) refuse("%s of %lld is too large", name, (long long)v);
  return (int)v;
}

const void* ptr(const at::Tensor& t) { return t.const_data_ptr(); }
const void* ptr(const at::Tensor* t) { return t ? t->const_data_ptr() : nullptr; }
void* out_ptr(const at::Tensor& t) { return t.mutable_data_ptr(); }

int cuda_index(const at::Tensor& t) {
  if (!t.is_cuda()) refuse("triteia_b200: tensors must live on a CUDA device (there is no CPU path)");
  return t.get_device();
}

void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }

// A new tensor, past the dispatcher (half a microsecond a tensor).
at::Tensor fresh_tensor(at::IntArrayRef sizes, at::ScalarType type, const at::Device& device) {
  return at::Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));
}

bool last_contiguous(const at::Tensor& t) { return t.stride(-1) == 1 || t.size(-1) <= 1; }

void check_vector(const at::Tensor& t, const char* name, at::ScalarType type, int64_t n, const at::Device& device) {
  if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != n || !t.is_contiguous() || t.device() != device)
    refuse("%s must be a contiguous one-dimensional %s tensor of %lld entries on %s", name, c10::toString(type), (long long)n,
           device.str().c_str());
}

// A cache that holds `type`, or e4m3 with exponents.
struct Cache {
  const at::Tensor &key, &value;
  const at::Tensor *key_exp, *value_exp;
  int64_t pages, page, token, head, e_page = 0, e_token = 0, e_head = 0;
  int page_size, heads, size;

  Cache(const at::Tensor& k, const at::Tensor& v, const at::Tensor* ke, const at::Tensor* ve, at::ScalarType type, const at::Device& device)
      : key(k), value(v), key_exp(ke), value_exp(ve) {
    if (k.dim() != 4 || k.sizes() != v.sizes() || k.strides() != v.strides())
      refuse("key_cache and value_cache must be [pages, page_size, kv_heads, head_size] with the same strides");
    pages = k.size(0);
    page_size = small(k.size(1), "page size");
    heads = small(k.size(2), "number of heads");
    size = small(k.size(3), "head size");
    if (page_size == 0 || heads == 0 || !last_contiguous(k)) refuse("a cache needs a page size, heads and a contiguous last dimension");
    if ((ke == nullptr) != (ve == nullptr)) refuse("key_exponents and value_exponents go together");
    const at::ScalarType want = ke ? at::kFloat8_e4m3fn : type;
    if (k.scalar_type() != want || v.scalar_type() != want)
      refuse("the cache holds %s and %s: %s is needed %s exponents", c10::toString(k.scalar_type()), c10::toString(v.scalar_type()),
             c10::toString(want), ke ? "with" : "without");
    if (k.device() != device || v.device() != device) refuse("the cache must be on %s", device.str().c_str());
    page = k.stride(0), token = k.stride(1), head = k.stride(2);
    if (!ke) return;
    for (const at::Tensor* e : {ke, ve})
      if (e->scalar_type() != at::kByte || e->sizes() != k.sizes().slice(0, 3) || e->strides() != ke->strides() || e->device() != device)
        refuse("exponents must be uint8 [pages, page_size, kv_heads] on the cache's device, both with the same strides");
    e_page = ke->stride(0), e_token = ke->stride(1), e_head = ke->stride(2);
  }
};

#define TRB_TRY try {
#define TRB_CATCH                                              \
  }                                                            \
  catch (const Refused&) {                                     \
    return nullptr;                                            \
  }                                                            \
  catch (const std::exception& e) {                            \
    PyErr_SetString(PyExc_RuntimeError, e.what());             \
    return nullptr;                                            \
  }
#define TRB_COUNT(n)                                                                 \
  if (nargs != n) {                                                                  \
    PyErr_Format(PyExc_TypeError, "%d arguments are needed, %zd given", n, nargs);   \
    return nullptr;                                                                  \
  }

// cache_write(key, value, key_cache, value_cache, slots, key_exponents, value_exponents)
PyObject* cache_write(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  TRB_COUNT(7)
  TRB_TRY
  const at::Tensor &key = tensor(args[0], "key"), &value = tensor(args[1], "value"), &slots = tensor(args[4], "slots");
  if (key.dim() != 3 || key.sizes() != value.sizes() || key.scalar_type() != value.scalar_type() || key.device() != value.device())
    refuse("key and value must be [tokens, kv_heads, head_size] of one dtype on one device");
  if (!last_contiguous(key) || !last_contiguous(value)) refuse("key and value need a contiguous last dimension");
  const at::Device device = key.device();
  const Cache c(tensor(args[2], "key_cache"), tensor(args[3], "value_cache"), maybe(args[5], "key_exponents"),
                maybe(args[6], "value_exponents"), key.scalar_type(), device);
  const int T = small(key.size(0), "number of tokens");
  if (key.size(1) != c.heads || key.size(2) != c.size)
    refuse("key of shape [%d, %lld, %lld]: the cache needs [%d, %d, %d]", T, (long long)key.size(1), (long long)key.size(2), T, c.heads, c.size);
  check_vector(slots, "slots", at::kLong, T, device);
  const int tag = tag_of(key.scalar_type()), dev = cuda_index(key);
  const int status = trb_cache_write(ptr(key), ptr(value), ptr(slots), out_ptr(c.key), out_ptr(c.value), const_cast<void*>(ptr(c.key_exp)),
                                     const_cast<void*>(ptr(c.value_exp)), T, c.heads, c.size, c.page_size, c.pages, key.stride(0),
                                     key.stride(1), value.stride(0), value.stride(1), c.page, c.token, c.head, c.e_page, c.e_token,
                                     c.e_head, tag, dev, stream_of(dev));
  check_status(status, "cache_write", "head_size is a multiple of 8 up to 256 and heads begin on 16-byte boundaries");
  Py_RETURN_NONE;
  TRB_CATCH
}

// cache_read(key_cache, value_cache, slots, key_exponents, value_exponents, dtype or None)
PyObject* cache_read(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  TRB_COUNT(6)
  TRB_TRY
  const at::Tensor &kc = tensor(args[0], "key_cache"), &slots = tensor(args[2], "slots");
  if (args[5] != Py_None && !THPDtype_Check(args[5])) refuse("dtype must be a torch.dtype");
  const at::ScalarType type = args[5] == Py_None ? kc.scalar_type() : (at::ScalarType)reinterpret_cast<THPDtype*>(args[5])->scalar_type;
  const int tag = tag_of(type);
  const at::Device device = kc.device();
  const Cache c(kc, tensor(args[1], "value_cache"), maybe(args[3], "key_exponents"), maybe(args[4], "value_exponents"), type, device);
  check_vector(slots, "slots", at::kLong, slots.numel(), device);
  const int T = small(slots.numel(), "number of tokens");
  const int dev = cuda_index(kc);
  at::Tensor key = fresh_tensor({T, c.heads, c.size}, type, device), value = fresh_tensor({T, c.heads, c.size}, type, device);
  const int status = trb_cache_read(ptr(c.key), ptr(c.value), ptr(c.key_exp), ptr(c.value_exp), ptr(slots), out_ptr(key), out_ptr(value), T,
                                    c.heads, c.size, c.page_size, c.pages, c.page, c.token, c.head, c.e_page, c.e_token, c.e_head, tag, dev,
                                    stream_of(dev));
  check_status(status, "cache_read", "head_size is a multiple of 8 up to 256 and heads begin on 16-byte boundaries");
  PyObject* k = THPVariable_Wrap(std::move(key));
  PyObject* v = k ? THPVariable_Wrap(std::move(value)) : nullptr;
  PyObject* both = v ? PyTuple_Pack(2, k, v) : nullptr;
  Py_XDECREF(k);
  Py_XDECREF(v);
  return both;
  TRB_CATCH
}

// paged_attention(query, key_cache, value_cache, page_table, lengths, query_starts, scale, causal, window, key_exponents,
//                 value_exponents, out)
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  TRB_COUNT(12)
  TRB_TRY
  const at::Tensor &query = tensor(args[0], "query"), &table = tensor(args[3], "page_table"), &lengths = tensor(args[4], "lengths");
  const at::Tensor* starts = maybe(args[5], "query_starts");
  if (query.dim() != 3 || !last_contiguous(query)) refuse("query must be [tokens, heads, head_size] with a contiguous last dimension");
  const int T = small(query.size(0), "number of tokens"), heads = small(query.size(1), "number of heads"), size = small(query.size(2), "head size");
  const at::Device device = query.device();
  const Cache c(tensor(args[1], "key_cache"), tensor(args[2], "value_cache"), maybe(args[9], "key_exponents"),
                maybe(args[10], "value_exponents"), query.scalar_type(), device);
  if (c.size != size || heads == 0 || heads % c.heads != 0)
    refuse("query heads %d x %d do not go with key heads %d x %d", heads, size, c.heads, c.size);
  if (table.dim() != 2 || table.scalar_type() != at::kInt || table.device() != device || !last_contiguous(table))
    refuse("page_table must be int32 [sequences, pages] with contiguous rows on %s", device.str().c_str());
  const int B = small(table.size(0), "number of sequences");
  check_vector(lengths, "lengths", at::kInt, B, device);
  if (starts) check_vector(*starts, "query_starts", at::kInt, (int64_t)B + 1, device);
  else if (T != B) refuse("%d tokens for %d sequences: query_starts is needed", T, B);
  const double scale = args[6] == Py_None ? 1.0 / sqrt((double)size) : real(args[6]);
  if (size > 0 && !(fabs(scale) <= 2e38)) refuse("scale must be a finite number that 32 bits hold");
  const bool causal = truth(args[7]);
  const long long window = args[8] == Py_None ? 0 : integer(args[8]);
  if (args[8] != Py_None && (window <= 0 || !causal)) refuse("a window is a positive number of tokens and needs causal=True");
  at::Tensor fresh;
  const at::Tensor* out = maybe(args[11], "out");
  if (out && (out->sizes() != query.sizes() || out->scalar_type() != query.scalar_type() || out->device() != device || !last_contiguous(*out)))
    refuse("out must have the shape, dtype and device of query and a contiguous last dimension");
  const int tag = tag_of(query.scalar_type()), dev = cuda_index(query);
  if (!out) {
    fresh = fresh_tensor({T, heads, size}, query.scalar_type(), device);
    out = &fresh;
  }
  const int width = small(table.size(1), "page table's width");
  // A buffer of each call's own: calls on different streams, and graphs that are replayed side by side, share nothing.
  at::Tensor workspace;
  const size_t bytes = trb_paged_attention_cache_workspace_bytes(T, B, heads, c.heads, size, c.page_size, c.pages, width, c.page, c.token,
                                                                 c.head, starts == nullptr, c.key_exp != nullptr, dev);
  if (bytes > 0) workspace = fresh_tensor({(int64_t)bytes}, at::kByte, device);
  // Rows of a new tensor that belong to no sequence are zeros, not what lay in the memory before.
  const int status = trb_paged_attention_clear(
      ptr(query), ptr(c.key), ptr(c.value), ptr(c.key_exp), ptr(c.value_exp), ptr(table), ptr(lengths), ptr(starts), out_ptr(*out), T, B,
      heads, c.heads, size, c.page_size, c.pages, table.stride(0), width, query.stride(0),
      query.stride(1), out->stride(0), out->stride(1), c.page, c.token, c.head, c.e_page, c.e_token, c.e_head, (float)scale, causal,
      (int)(window > 0x7fffffff ? 0x7fffffff : window), tag,
      bytes > 0 ? out_ptr(workspace) : nullptr, bytes, dev, stream_of(dev), fresh.defined() && starts);
  check_status(status, "paged_attention", "heads of 64 or 128 that begin on 16-byte boundaries are needed");
  if (!fresh.defined()) return Py_NewRef(args[11]);
  return THPVariable_Wrap(std::move(fresh));
  TRB_CATCH
}

// Rows of a [..., heads * size] tensor.
struct Rows {
  const void* data = nullptr;
  int64_t rows = 0, stride = 0, cols = 0;
  Rows() = default;
  Rows(const at::Tensor& t, const char* name, int size, const at::Tensor& like) {
    if (t.device() != like.device() || t.scalar_type() != like.scalar_type())
      refuse("%s must have the device and dtype of query (%s, %s)", name, like.device().str().c_str(), c10::toString(like.scalar_type()));
    const bool flat = t.dim() == 2 || (t.dim() >= 1 && t.is_contiguous());
    if (!flat || !last_contiguous(t) || size <= 0 || t.size(-1) % size != 0)
      refuse("%s must be [tokens, heads * %d] with contiguous rows", name, size);
    cols = t.size(-1);
    rows = t.dim() == 2 ? t.size(0) : cols ? t.numel() / cols : 0;
    stride = t.dim() == 2 ? t.stride(0) : cols;
    data = t.const_data_ptr();
  }
};

// qk_norm_rotary(positions, query, key, head_size, cos_sin_cache, is_neox, query_weight, key_weight, eps, query_out, key_out)
PyObject* qk_norm_rotary(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  TRB_COUNT(11)
  TRB_TRY
  const at::Tensor &positions = tensor(args[0], "positions"), &query = tensor(args[1], "query"), &table = tensor(args[4], "cos_sin_cache");
  const at::Tensor *key = maybe(args[2], "key"), *qo = maybe(args[9], "query_out"), *ko = maybe(args[10], "key_out");
  const int size = small(integer(args[3]), "head size");
  const Rows q(query, "query", size, query), q_out = qo ? Rows(*qo, "query_out", size, query) : q;
  const Rows k = key ? Rows(*key, "key", size, query) : Rows(), k_out = ko && key ? Rows(*ko, "key_out", size, query) : k;
  if (key && (k.rows != q.rows || k_out.rows != q.rows || k_out.cols != k.cols))
    refuse("key and key_out must have one row per row of query and the same heads");
  if (q_out.rows != q.rows || q_out.cols != q.cols || positions.numel() != q.rows)
    refuse("positions and query_out must have one entry and one row per row of query");
  if (positions.scalar_type() != at::kLong || !positions.is_contiguous()) refuse("positions must be a contiguous int64 tensor");
  const bool wide = table.scalar_type() == at::kFloat;
  if (table.dim() != 2 || !table.is_contiguous() || (!wide && table.scalar_type() != query.scalar_type()))
    refuse("cos_sin_cache must be a contiguous [max_position, rot_dim] tensor of query's dtype or float32");
  const at::Tensor* weights[2] = {maybe(args[6], "query_weight"), maybe(args[7], "key_weight")};
  for (const at::Tensor* w : weights)
    if (w && (w->scalar_type() != query.scalar_type() || w->numel() != size || !w->is_contiguous() || w->device() != query.device()))
      refuse("query_weight and key_weight must be contiguous [%d] tensors of query's dtype and device", size);
  if (positions.device() != query.device() || table.device() != query.device())
    refuse("positions and cos_sin_cache must be on the device of query");
  const float eps = args[8] == Py_None ? 0.f : (float)real(args[8]);
  if (!(eps >= 0.f)) refuse("eps must not be negative (None: no norm)");
  const int tag = tag_of(query.scalar_type()), dev = cuda_index(query);
  const int status = trb_qk_norm_rotary(
      ptr(positions), q.data, const_cast<void*>(q_out.data), k.data, const_cast<void*>(k_out.data), ptr(weights[0]), ptr(weights[1]),
      ptr(table), wide, table.size(0), small(q.rows, "number of tokens"), small(table.size(1), "rot_dim"), q.stride, q_out.stride, k.stride,
      k_out.stride, (int)(q.cols / size), (int)(k.cols / size), size, args[8] == Py_None ? -1.f : eps, truth(args[5]), tag, dev, stream_of(dev));
  check_status(status, "qk_norm_rotary_embedding",
               "head_size is a multiple of 8 up to 256, rot_dim even and at most head_size, rows begin on 16-byte boundaries");
  Py_RETURN_NONE;
  TRB_CATCH
}

#define TRB_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {TRB_METHOD(cache_write), TRB_METHOD(cache_read), TRB_METHOD(paged_attention), TRB_METHOD(qk_norm_rotary),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", TRB_BINDING_TAG) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
